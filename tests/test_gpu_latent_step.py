"""The latent cache and its pages as a server uses them: reservations, appends, attention, forks, frees and compactions in turn, captured and replayed, on streams of their own."""
import pytest
import torch

import int_flashattention_amd as M
from latent_reference import attend, normalised
from paged_reference import rotate
from test_gpu_latent_attention import bound, freqs_of, queries

pytestmark = pytest.mark.gpu
DEV = "cuda"
DC, DR, PAGE = 256, 64, 32


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Server:
    """Layers of latent caches that share a table, and what has been appended to each sequence as plain rows."""

    def __init__(self, Z, pages, width, layers=2, dtype=torch.bfloat16, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.Z, self.dtype, self.g = Z, dtype, g
        self.caches = [torch.randint(-128, 128, (pages, PAGE, DC + DR), generator=g, dtype=torch.int8).to(DEV) for _ in range(layers)]
        self.scales = [torch.rand((pages, PAGE, 2), generator=g).to(DEV) for _ in range(layers)]
        self.refs, self.table, self.lens = ints(*[0] * pages), torch.full((Z, width), -1, dtype=torch.int32, device=DEV), ints(*[0] * Z)
        self.weights = [(1 + 0.2 * torch.randn(DC, generator=g)).to(dtype).to(DEV) for _ in range(layers)]
        self.freqs = freqs_of(DR // 2).to(DEV)
        self.rows = [[[] for _ in range(Z)] for _ in range(layers)]

    def pools(self):
        return [t for pair in zip(self.caches, self.scales) for t in pair]

    def books(self):
        return [self.refs, self.table, self.lens, *self.pools()]

    def new(self, n):
        return [((torch.randn((self.Z, n, DC), generator=self.g) * 3).to(self.dtype).to(DEV), torch.randn((self.Z, n, DR), generator=self.g).to(self.dtype).to(DEV)) for _ in self.caches]

    def step(self, new, fresh):
        granted = M.paged_reserve(self.pools(), self.refs, self.table, self.lens, fresh, PAGE)
        for (c, k), cache, scale, w in zip(new, self.caches, self.scales, self.weights):
            M.paged_latent_append(cache, scale, c, k, self.table, self.lens, self.freqs, seqlens_new=granted, norm_weight=w)
        self.lens += granted
        return granted

    def attend(self, layer, q, **kw):
        return M.attention_paged_latent_int8(*q, self.caches[layer], self.scales[layer], self.table, self.lens, True, 0.1, freqs=self.freqs, **kw)

    # ---- the same on lists
    def note(self, new, granted):
        for layer, (c, k) in enumerate(new):
            for z, m in enumerate(granted.tolist()):
                self.rows[layer][z] = self.rows[layer][z] + [(c[z, i].cpu(), k[z, i].cpu()) for i in range(m)]

    def check(self, dtype=torch.bfloat16, N=2):
        """Every token of every sequence is in the cache, to half a step of its scales, and attention is that over what the cache holds."""
        lens, table = self.lens.tolist(), self.table.cpu()
        named = table[(table >= 0)]
        assert torch.equal(torch.bincount(named.flatten(), minlength=self.refs.numel()).int(), self.refs.cpu())
        for layer, rows in enumerate(self.rows):
            cache, scale, w = self.caches[layer].cpu(), self.scales[layer].cpu(), self.weights[layer].cpu()
            for z, n in enumerate(lens):
                assert n == len(rows[z])
                if n == 0:
                    continue
                at = torch.arange(n)
                page, r = table[z, at // PAGE].long(), at % PAGE
                c = normalised(torch.stack([a for a, _ in rows[z]]), w, 1e-6)
                k = rotate(torch.stack([b for _, b in rows[z]]).double()[None, None], at[None], self.freqs.cpu())[0, 0]
                for part, x in ((slice(0, DC), c), (slice(DC, DC + DR), k)):
                    s = scale[page, r, int(part.start > 0)].double()[:, None]
                    # (the rounding to int8 is half a step, the scale and the arithmetic before it are fp32: 2^-18 of 127 steps at most)
                    assert ((cache[page, r, part].double() * s - x).abs() <= s * (0.5 + 127 * 2.0 ** -18)).all()
            q = queries(self.g, self.Z, 5, N, DC, DR, dtype)
            out, lse = (t.cpu() for t in self.attend(layer, [t.to(DEV) for t in q], return_lse=True))
            want, want_lse, mean_v, size, step = attend(*q, cache, scale, table, lens, True, 0.1, rope=dict(freqs=self.freqs.cpu()))
            assert ((out.double() - want).abs() <= bound(want, mean_v, size, step, dtype)).all() and torch.equal(lse.isinf(), want_lse.isinf())


def test_a_server_runs():
    s = Server(9, 60, 7)
    prompts = ints(70, 33, 0, 128, 64, 1, 0, 31, 97)
    new = s.new(128)
    granted = s.step(new, prompts)
    assert torch.equal(granted, prompts)
    s.note(new, granted)
    s.check()
    # two continuations of sequences 0 and 3 each: their last pages are copied when they part, but for the last holder's
    M.paged_fork(s.refs, s.table, s.lens, ints(0, 3), ints(2, 6))
    for rows in s.rows:
        rows[2], rows[6] = rows[0], rows[3]
    s.check()
    free_before = int((s.refs == 0).sum())
    for step in range(4):
        new = s.new(2)
        fresh = ints(*[1 + (z + step) % 2 for z in range(9)])
        granted = s.step(new, fresh)
        assert torch.equal(granted, fresh)
        s.note(new, granted)
        s.check(torch.float16 if step % 2 else torch.bfloat16)
    assert int((s.refs == 0).sum()) < free_before
    # drafts that were not taken: back to fewer tokens, and on from there; a sequence ends; the pool is packed
    M.paged_free(s.refs, s.table, s.lens, ints(0, 4, 3, 4), PAGE, ints(65, 60, 0, 64))
    for rows in s.rows:
        rows[0], rows[4], rows[3] = rows[0][:65], rows[4][:60], []
    s.check()
    used = int((s.refs > 0).sum())
    where = M.paged_compact(s.pools(), s.refs, s.table)
    assert int(where.max()) == used - 1 and int((s.refs[used:] != 0).sum()) == 0
    s.check()
    new = s.new(40)
    granted = s.step(new, ints(*[40] * 9))
    s.note(new, granted)
    s.check()


def test_a_server_runs_out_of_pages():
    """Tokens that find no page are neither appended nor seen."""
    s = Server(5, 6, 8)
    for n in (40, 40, 40):
        new = s.new(n)
        granted = s.step(new, ints(*[n] * 5))
        s.note(new, granted)
        s.check()
    # (six pages of 32: two each for the first three, 40 tokens in them, and then what the second page holds, 64)
    assert s.lens.tolist() == [64, 64, 64, 0, 0] and int((s.refs == 0).sum()) == 0


def _captured(f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    return graph


@pytest.mark.parametrize("H,width", [(4, 6), (40, 6), (40, 800)])
def test_a_captured_step_replays_like_eager_ones(H, width):
    """Reservation, appends, lengths and attention captured once, replayed over new tokens with forks, frees and eager work in between; eager steps on a second server give the same bits."""
    a, b = Server(6, 80, width), Server(6, 80, width)
    start = [t.clone() for t in a.books()]
    q = [torch.zeros((6, H, 1, d), dtype=torch.bfloat16, device=DEV) for d in (DC, DR)]
    new, fresh = [tuple(torch.zeros_like(t) for t in pair) for pair in a.new(3)], ints(*[0] * 6)

    def step(s):
        granted = s.step(new, fresh)
        return [granted, *(s.attend(layer, q) for layer in range(2))]

    graph = _captured(lambda: step(a))
    for t, x in zip(a.books(), start):
        t.copy_(x)
    with torch.cuda.graph(graph):
        out = step(a)
    g = torch.Generator().manual_seed(11)
    for i in range(8):
        for t in [*q, *(t for pair in new for t in pair)]:
            t.copy_(torch.randn(t.shape, generator=g))
        fresh.copy_(torch.randint(0, 4, (6,), generator=g))
        for s in (a, b):
            if i % 3 == 1:
                M.paged_fork(s.refs, s.table, s.lens, ints(0, 1), ints(5, 4))
            if i == 4:
                M.paged_free(s.refs, s.table, s.lens, ints(2, 3), PAGE, ints(0, 2))
            if i == 6:
                M.paged_compact(s.pools(), s.refs, s.table)
        graph.replay()
        torch.cuda.synchronize()
        want = step(b)
        for x, y in zip([*out, *a.books()], [*want, *b.books()]):
            assert torch.equal(x, y), i
        torch.randn((512, 512), device=DEV).sum().item()
    assert int(a.lens.max()) > 8


def test_two_graphs_of_one_memory_pool():
    """Attention of two lengths and the expanded form captured into graphs that share their memory, workspaces too, replayed in turn."""
    servers = [Server(3, 200, 60, layers=1, seed=i) for i in range(2)]
    for s, n in zip(servers, (1800, 70)):
        s.step(s.new(n), ints(n, n // 2, 1))
    g = torch.Generator().manual_seed(4)
    qs = [[torch.randn((3, H, N, d), generator=g).half().to(DEV) for d in (DC, DR)] for H, N in ((16, 1), (20, 4))]
    x = [torch.randn((1, h, 200, d), generator=g).half().to(DEV) for h, d in ((4, 128), (4, 64), (4, 128), (1, 64), (4, 128))]
    work = [lambda: [servers[0].attend(0, qs[0]), servers[0].attend(0, [-t for t in qs[0]])], lambda: [servers[1].attend(0, qs[1]), M.attention_latent(*x, True, 0.1)]]
    graphs, outs = [], []
    for f in work:
        graph = _captured(f)
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(f())
        graphs.append(graph)
    for step in range(4):
        for graph, out, f, q in zip(graphs, outs, work, qs):
            q[0].copy_(torch.randn(q[0].shape, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            for got, want in zip(out, f()):
                assert torch.equal(got, want)


def test_two_streams_at_once():
    """Two servers' steps on streams of their own, many at a time, equal to the same ones in order."""
    servers = [Server(4, 120, 24, seed=i % 2) for i in range(4)]
    prompts = [s.new(600) for s in servers[:2]]
    for i, s in enumerate(servers):
        s.step(prompts[i % 2], 600)
    g = torch.Generator().manual_seed(8)
    steps = [([torch.randn((4, 12, 1, d), generator=g).bfloat16().to(DEV) for d in (DC, DR)], servers[0].new(1)) for _ in range(6)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for q, new in steps:
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                servers[i].step(new, 1)
                got[i].append(servers[i].attend(i, q))
    torch.cuda.synchronize()
    for i in range(2):
        for (q, new), o in zip(steps, got[i]):
            servers[2 + i].step(new, 1)
            assert torch.equal(servers[2 + i].attend(i, q), o)
        assert all(torch.equal(x, y) for x, y in zip(servers[i].books(), servers[2 + i].books()))


@pytest.mark.parametrize("width", [40, 1000])
def test_calls_repeat_to_the_bit(width):
    s = Server(5, 200, width, layers=1)
    s.step(s.new(1200), ints(1200, 700, 3, 64, 999))
    for H, N in ((16, 1), (30, 1), (128, 1), (10, 6)):
        q = [t.to(DEV) for t in queries(s.g, 5, H, N, DC, DR, torch.bfloat16)]
        first = s.attend(0, q, return_lse=True)
        for _ in range(5):
            again = s.attend(0, q, return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_refusals():
    s = Server(2, 8, 4, layers=1)
    q, cache, scale = [torch.zeros((2, 4, 1, d), dtype=torch.float16, device=DEV) for d in (DC, DR)], s.caches[0], s.scales[0]
    c, k, w, f = (torch.zeros(n, dtype=torch.float16, device=DEV) for n in ((2, 1, DC), (2, 1, DR), (DC,), (1,)))
    f = s.freqs

    def attend_(q=q[0], r=q[1], cache=cache, scale=scale, table=s.table, lens=s.lens, **kw):
        return M.attention_paged_latent_int8(q, r, cache, scale, table, lens, True, 0.1, **kw)

    def append_(c=c, k=k, cache=cache, scale=scale, table=s.table, lens=s.lens, **kw):
        return M.paged_latent_append(cache, scale, c, k, table, lens, kw.pop("freqs", None), **kw)

    attend_(), append_()
    for call, first in ((attend_, "q"), (append_, "c")):
        second = dict(q="r", c="k")[first]
        x, y = dict(q=(q[0], q[1]), c=(c, k))[first]
        with pytest.raises(TypeError):
            call(**{first: x.float()})
        with pytest.raises(TypeError):
            call(**{second: y.bfloat16()})
        with pytest.raises((ValueError, AssertionError)):
            call(**{second: y[:1]})
        with pytest.raises((ValueError, AssertionError, RuntimeError)):
            call(**{second: y.cpu()})
        for parts in ((x[..., :192], y), (x, y[..., :48])):
            with pytest.raises(AssertionError):
                call(**dict(zip((first, second), parts)))
        for kw in (dict(cache=cache.view(torch.uint8)), dict(cache=cache[:, :8]), dict(cache=cache[..., :256]), dict(cache=cache.cpu()), dict(cache=cache.transpose(1, 2).contiguous().transpose(1, 2)),
                   dict(cache=torch.zeros(8 * PAGE * (DC + DR) + 8, dtype=torch.int8, device=DEV)[8:].view(8, PAGE, DC + DR)), dict(scale=scale.half()), dict(scale=scale[:7]),
                   dict(scale=scale[..., :1]), dict(scale=scale.cpu()), dict(scale=scale.transpose(1, 2).contiguous().transpose(1, 2)), dict(table=s.table.long()), dict(table=s.table[:1]),
                   dict(table=s.table[:, :0]), dict(table=s.table[:, ::2]), dict(table=s.table.cpu()), dict(lens=s.lens.long()), dict(lens=s.lens[:1]), dict(lens=s.lens.cpu()),
                   dict(freqs=f.float()), dict(freqs=f[:12]), dict(freqs=torch.cat([f, f])), dict(freqs=f.cpu()), dict(freqs=f, magnitude=0.0)):
            with pytest.raises((ValueError, AssertionError)):
                call(**kw)
    with pytest.raises(ValueError):
        attend_(seqlens_q=s.lens[:1])
    for kw in (dict(norm_weight=w.float()), dict(norm_weight=w[:100]), dict(norm_weight=w.cpu()), dict(norm_weight=w, norm_eps=0.0), dict(norm_weight=w, norm_eps=float("nan")),
               dict(seqlens_new=s.lens[:1]), dict(seqlens_new=s.lens.long())):
        with pytest.raises(ValueError):
            append_(**kw)
    # nothing to do is no error
    assert attend_(q=q[0][:, :, :0], r=q[1][:, :, :0]).shape == (2, 4, 0, DC) and append_(c=c[:, :0], k=k[:, :0]) is None

    x = [torch.zeros((2, h, n, d), dtype=torch.float16, device=DEV) for h, n, d in ((4, 3, 128), (4, 3, 64), (4, 5, 128), (1, 5, 64), (4, 5, 128))]

    def expanded(i=None, t=None, **kw):
        return M.attention_latent(*(t if j == i else y for j, y in enumerate(x)), True, 0.1, **kw)

    expanded()
    for i, t in ((1, x[1].bfloat16()), (4, x[4].float())):
        with pytest.raises(TypeError):
            expanded(i, t)
    with pytest.raises(AssertionError):
        expanded(4, x[4][..., :64])
    for i, t in ((1, x[1][:, :2]), (2, x[2][:1]), (3, x[3].expand(-1, 4, -1, -1)), (3, x[3][:, :, :4]), (4, x[4][:, :, :4])):
        with pytest.raises(ValueError):
            expanded(i, t)
    for i in range(5):
        with pytest.raises((ValueError, RuntimeError)):
            expanded(i, x[i].cpu())
    for kw in (dict(seqlens_q=s.lens[:1]), dict(seqlens_k=s.lens.long()), dict(seqlens_k=s.lens.cpu())):
        with pytest.raises(ValueError):
            expanded(**kw)
    torch.cuda.synchronize()


def test_tables_and_pools_that_overlap_are_refused():
    """What is changed in place must be there once."""
    s = Server(3, 8, 4, layers=1)
    same = s.table[:1].expand(3, -1)
    wide = torch.zeros(3 + 3, dtype=torch.int32, device=DEV).as_strided((3, 4), (1, 1))
    pages = torch.zeros((1, 4), device=DEV).expand(8, -1)
    for table in (same, wide):
        for call in (lambda: M.paged_fork(s.refs, table, s.lens, ints(0), ints(1)), lambda: M.paged_free(s.refs, table, s.lens, ints(0), PAGE),
                     lambda: M.paged_reserve([], s.refs, table, s.lens, 1, PAGE), lambda: M.paged_compact([], s.refs, table)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: M.paged_copy([pages], ints(0), ints(1)), lambda: M.paged_reserve([pages], s.refs, s.table, s.lens, 1, PAGE), lambda: M.paged_compact([pages], s.refs, s.table)):
        with pytest.raises(ValueError):
            call()

"""Rotation, append and attention as a server calls them: prompts and steps over one pool of pages, captured steps, other streams, refusals."""
import pytest
import torch

import int_flashattention_amd as M
from paged_reference import attend, bound, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Pool:
    """Pages of one layer and the sequences in them."""

    def __init__(self, Z, Hkv, d, page, columns):
        self.kv = torch.zeros((Z * columns, 2, Hkv, page, d), dtype=torch.int8, device=DEV)
        self.sc = torch.zeros((Z * columns, 2, Hkv), device=DEV)
        g = torch.Generator().manual_seed(1)
        self.table = torch.randperm(Z * columns, generator=g).to(torch.int32).reshape(Z, columns).to(DEV)
        self.lens = torch.zeros((Z,), dtype=torch.int32, device=DEV)
        self.rope = dict(freqs=M.rotary_frequencies(d, device=DEV)[0])

    def append(self, k, v, fresh=None):
        M.paged_kvcache_append(self.kv[:, 0], self.sc[:, 0], self.kv[:, 1], self.sc[:, 1], k, v, self.table, self.lens, seqlens_new=fresh, **self.rope)
        self.lens += k.shape[2] if fresh is None else fresh

    def attend(self, q, fresh=None, rope=True):
        return M.attention_paged_int8(q, self.kv[:, 0], self.kv[:, 1], self.sc[:, 0], self.sc[:, 1], self.table, self.lens, True, q.shape[-1] ** -0.5,
                                      seqlens_q=fresh, **(self.rope if rope else {}))

    def want(self, q, fresh=None):
        cache = dict(k=self.kv[:, 0].cpu(), v=self.kv[:, 1].cpu(), ks=self.sc[:, 0].cpu(), vs=self.sc[:, 1].cpu())
        return attend(q.cpu(), cache, self.table.cpu(), self.lens.tolist(), True, q.shape[-1] ** -0.5, None if fresh is None else fresh.tolist(),
                      dict(freqs=self.rope["freqs"].cpu()))


def rows(g, Z, H, N, d, dtype):
    return torch.randn((Z, H, N, d), generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype,page,d", [(torch.float16, 16, 64), (torch.bfloat16, 64, 128)])
def test_prompts_then_steps(dtype, page, d):
    """Prompts of three lengths in one padded batch, a second chunk, then tokens one by one: each call's output is the attention over what the cache
    holds, and that is near the attention over the unquantised tokens."""
    Z, H, Hkv = 3, 8, 2
    g = torch.Generator().manual_seed(2)
    pool = Pool(Z, Hkv, d, page, -(-160 // page))
    keys, values = [], []                                       # per call: rows and how many of each sequence's count

    def call(N, fresh):
        q, k, v = rows(g, Z, H, N, d, dtype), rows(g, Z, Hkv, N, d, dtype), rows(g, Z, Hkv, N, d, dtype)
        pool.append(k, v, fresh)
        o = pool.attend(q, fresh)
        want, _, mean_v, size = pool.want(q, fresh)
        step = 2.0 ** -12 if dtype == torch.bfloat16 and H // Hkv * N > 64 else 0.0      # (many rows of bf16 queries: 11 bits)
        assert ((o.cpu().double() - want).abs() <= bound(want, mean_v, size, dtype, step)).all()
        counts = [N] * Z if fresh is None else fresh.tolist()
        keys.append((k.cpu(), counts)); values.append((v.cpu(), counts))
        # the rotation as a call of its own: its rounding to the queries' type is all the difference
        first = pool.lens - (N if fresh is None else fresh)
        alone = pool.attend(M.rotary(q, first, pool.rope["freqs"]), fresh, rope=False)
        eps = torch.finfo(dtype).eps
        assert ((alone.double() - o.double()).abs().cpu() <= 2 * bound(want, mean_v, size, dtype, step) + 2 * eps / 2 * size * mean_v).all()
        return q, o

    call(70, torch.tensor([70, 33, 1], dtype=torch.int32, device=DEV))
    call(40, torch.tensor([5, 40, 0], dtype=torch.int32, device=DEV))
    for _ in range(4):
        q, o = call(1, None)
    for z in range(Z):
        k = torch.cat([x[z, :, :n[z]] for x, n in keys], 1).double()
        v = torch.cat([x[z, :, :n[z]] for x, n in values], 1).double()
        n = k.shape[1]
        assert n == pool.lens[z].item()
        k = rotate(k[None], torch.arange(n)[None], pool.rope["freqs"].cpu())[0].repeat_interleave(H // Hkv, 0)
        qr = rotate(q[z:z + 1].cpu(), torch.tensor([[n - 1]]), pool.rope["freqs"].cpu())[0]
        w = torch.softmax((qr @ k.transpose(1, 2)) * d ** -0.5, -1)
        exact = (w @ v.repeat_interleave(H // Hkv, 0))[:, 0]
        # int8 with a scale per page: a step of 4 / 127 or so, half of it off at most in every value, averaging out
        assert (o[z, :, 0].cpu().double() - exact).abs().max() <= 0.08


def test_a_captured_step_replays_like_eager_ones():
    """A decoding step - append, lengths, attention - captured once and replayed over new tokens, with eager work in between; the eager steps on a
    second pool give the same bits."""
    Z, H, Hkv, d, page = 4, 8, 2, 128, 32
    g = torch.Generator().manual_seed(3)
    a, b = Pool(Z, Hkv, d, page, 8), Pool(Z, Hkv, d, page, 8)
    for pool in (a, b):
        pool.append(*(rows(torch.Generator().manual_seed(4 + i), Z, Hkv, 100, d, torch.float16) for i in range(2)))
    q, k, v = (torch.zeros((Z, h, 1, d), dtype=torch.float16, device=DEV) for h in (H, Hkv, Hkv))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.attend(q)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.append(k, v)
        out = a.attend(q)
    for step in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        b.append(k, v)
        want = b.attend(q)
        assert torch.equal(out, want) and torch.equal(a.kv, b.kv) and torch.equal(a.sc, b.sc) and torch.equal(a.lens, b.lens)
        torch.randn((512, 512), device=DEV).sum().item()


def test_two_graphs_of_one_memory_pool():
    """Attention steps of two lengths captured one after the other into graphs that share their memory, workspaces too, replayed in turn."""
    d, H, Hkv = 128, 16, 2
    g = torch.Generator().manual_seed(6)
    pools = [Pool(2, Hkv, d, 32, 70) for _ in range(2)]
    for pool, n in zip(pools, (2000, 130)):
        pool.append(*(rows(g, 2, Hkv, n, d, torch.float16) for _ in range(2)))
    qs = [rows(g, 2, H, n, d, torch.float16) for n in (1, 40)]                  # one kernel, the other
    for pool, q in zip(pools, qs):
        pool.attend(q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for pool, q in zip(pools, qs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append([pool.attend(q), pool.attend(-q)])
        graphs.append(graph)
    for step in range(4):
        for graph, pool, q, out in zip(graphs, pools, qs, outs):
            q.copy_(torch.randn(q.shape, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], pool.attend(q)) and torch.equal(out[1], pool.attend(-q))


def test_sequences_that_share_pages():
    """A prefix held once, named by both tables, and a page twice in one table."""
    d, H, Hkv = 64, 8, 2
    g = torch.Generator().manual_seed(7)
    pool = Pool(2, Hkv, d, 16, 12)
    pool.append(*(rows(g, 2, Hkv, 150, d, torch.float16) for _ in range(2)))
    q = rows(g, 2, H, 3, d, torch.float16)
    pool.table[1, :5] = pool.table[0, :5]
    pool.table[0, 7] = pool.table[0, 2]
    want, _, mean_v, size = pool.want(q)
    assert ((pool.attend(q).cpu().double() - want).abs() <= bound(want, mean_v, size, torch.float16)).all()


def test_two_streams_at_once():
    """Two requests' steps on streams of their own, many at a time, equal to the same ones in order."""
    d, H, Hkv = 64, 8, 8
    g = torch.Generator().manual_seed(5)
    pools = [Pool(2, Hkv, d, 16, 70) for _ in range(4)]
    prompt = [rows(g, 2, Hkv, 1000, d, torch.bfloat16) for _ in range(2)]
    steps = [[rows(g, 2, h, 1, d, torch.bfloat16) for h in (H, Hkv, Hkv)] for _ in range(6)]
    for pool in pools:
        pool.append(*prompt)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for q, k, v in steps:
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                pools[i].append(k, v)
                got[i].append(pools[i].attend(q))
    torch.cuda.synchronize()
    for i in range(2):
        for (q, k, v), o in zip(steps, got[i]):
            pools[2 + i].append(k, v)
            assert torch.equal(pools[2 + i].attend(q), o)


def test_refusals():
    pool = Pool(2, 2, 64, 16, 4)
    q, k = torch.zeros((2, 4, 1, 64), dtype=torch.float16, device=DEV), torch.zeros((2, 2, 1, 64), dtype=torch.float16, device=DEV)
    kc, vc, ks, vs, f = pool.kv[:, 0], pool.kv[:, 1], pool.sc[:, 0], pool.sc[:, 1], pool.rope["freqs"]

    def attend_(q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=pool.table, lens=pool.lens, **kw):
        return M.attention_paged_int8(q, kc, vc, ks, vs, table, lens, True, 0.125, **kw)

    def append_(k=k, v=k, kc=kc, vc=vc, ks=ks, vs=vs, table=pool.table, lens=pool.lens, f=None, **kw):
        return M.paged_kvcache_append(kc, ks, vc, vs, k, v, table, lens, f, **kw)

    attend_(), append_(), M.rotary(q, 0, f)
    with pytest.raises(TypeError):
        attend_(q=q.float())
    with pytest.raises(TypeError):
        append_(v=k.bfloat16())
    with pytest.raises(TypeError):
        M.rotary(q.float(), 0, f)
    with pytest.raises(AssertionError):
        attend_(q=torch.zeros((2, 4, 1, 128), dtype=torch.float16, device=DEV))
    with pytest.raises(RuntimeError):
        M.rotary(torch.zeros((1, 1, 1, 48), dtype=torch.float16, device=DEV), 0, f[:8])
    for call in (lambda **kw: attend_(**kw), lambda **kw: append_(**kw)):
        for kw in (dict(kc=kc.half()), dict(kc=kc[:, :, :8]), dict(vc=vc[:3]), dict(ks=ks.half()), dict(ks=ks[:, :1]), dict(table=pool.table.long()),
                   dict(table=pool.table[:1]), dict(table=pool.table[:, :0]), dict(table=pool.table[:, ::2]), dict(table=pool.table.cpu()), dict(lens=pool.lens.long()),
                   dict(lens=pool.lens[:1]), dict(lens=pool.lens.cpu()), dict(kc=kc.cpu()), dict(kc=kc.transpose(2, 3).contiguous().transpose(2, 3)),
                   dict(vs=vs.cpu())):
            with pytest.raises((ValueError, AssertionError)):
                call(**kw)
    for kw in (dict(freqs=f.float()), dict(freqs=f[:12]), dict(freqs=torch.cat([f, f])), dict(freqs=f.cpu()), dict(freqs=f, magnitude=0.0), dict(freqs=f[:, None]),
               dict(seqlens_q=pool.lens[:1]), dict(q=torch.zeros((2, 3, 1, 64), dtype=torch.float16, device=DEV))):
        with pytest.raises(ValueError):
            attend_(**kw)
    for positions in (torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros((2, 5), dtype=torch.int32, device=DEV),
                      torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            M.rotary(q, positions, f)
    # nothing to do is no error
    assert attend_(q=q[:, :, :0]).shape == (2, 4, 0, 64) and append_(k=k[:, :, :0], v=k[:, :, :0]) is None and M.rotary(q[:, :, :0], 0, f).shape == (2, 4, 0, 64)
    torch.cuda.synchronize()

"""Attention over a paged latent cache against its formula in float64."""
import math

import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import attend, make_pool
from paged_reference import make_table

pytestmark = pytest.mark.gpu


def bound(out, mean_v, size, step, dtype):
    """How far the kernel may be from the formula: half a step of the output's type; P rounded to 11 bits, at most 2^-11 of the mean of |v|, or to steps of 2^-35 of the
    row's largest, half of one for each token (which mean_v includes, as 2^11 times as much); scores off by dS move a weight by dS and their sum as much: dS is the
    error of the query's steps (`step`), and of the fp32 steps that scale and add a score, twelve roundings of at most the sum of |q k|, 2^-19 of it with the exponential's; the
    exponent's logarithm and the weights' reciprocal 2^-20 of a weight; sums over keys 2^-14."""
    return torch.finfo(dtype).eps / 2 * out.abs() + 1.05 * (2.0 ** -11 + 2.0 ** -14 + 2.0 ** -20 + 2.0 * (step + 2.0 ** -19 * size)) * mean_v + 2.0 ** -24


def freqs_of(pairs):
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)


def queries(g, Z, H, N, dc, dr, dtype, size=1.5):
    return (torch.randn((Z, H, N, dc), generator=g) * size * (64.0 / dc) ** 0.5).to(dtype), (torch.randn((Z, H, N, dr), generator=g) * size).to(dtype)


WIDE = {"on": False}


@pytest.fixture(autouse=True, params=[False, True], ids=["", "wide"])
def wide(request, monkeypatch):
    """Tables with room for few keys and for many, behind the same lengths: calls of more than 32 rows take tiles of 32 rows with the one and of 64 with the other."""
    monkeypatch.setitem(WIDE, "on", request.param)


def widened(table, q, page, lens):
    if not WIDE["on"] or max(lens) > table.shape[1] * page:      # (a length behind the table's end stays there)
        return table
    Z, H, N = q.shape[:3]
    more = 2100 * 64 // (Z * -(-H * N // 64) * page) + 1
    return torch.cat([table, torch.full((table.shape[0], more), -1, dtype=torch.int32)], 1)


def run(q, pool, table, lens, causal, sm=0.1, fresh=None, rope=None, **kw):
    table = widened(table, q[0], pool[0].shape[1], lens)
    i32 = dict(dtype=torch.int32, device="cuda")
    rope_kw = {} if rope is None else dict(freqs=rope["freqs"].cuda(), magnitude=rope.get("magnitude", 1.0), interleaved=rope.get("interleaved", False))
    return ifa.attention_paged_latent_int8(q[0].cuda(), q[1].cuda(), pool[0].cuda(), pool[1].cuda(), table.cuda(), torch.tensor(lens, **i32), causal, sm,
                                           seqlens_q=None if fresh is None else torch.tensor(fresh, **i32), return_lse=True, **rope_kw, **kw)


def check(q, pool, table, lens, causal, sm=0.1, fresh=None, rope=None):
    out, lse = (x.cpu() for x in run(q, pool, table, lens, causal, sm, fresh, rope))
    want, want_lse, mean_v, size, step = attend(*q, *pool, table, lens, causal, sm, fresh, rope)
    assert out.dtype == q[0].dtype and out.shape == q[0].shape
    d, b = (out.double() - want).abs(), bound(want, mean_v, size, step, out.dtype)
    # (what is past the output type's largest number rounds to infinity)
    past = (want.abs() + b > torch.finfo(out.dtype).max) & (out.double() == torch.sign(want) * math.inf)
    d[past] = 0.0
    assert (d <= b).all(), f"{(d / b).max():.3f} of the bound at {tuple(int(i) for i in (d / b).view(-1).argmax()[None])}"
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all()
    e = (lse.double() - want_lse)[~empty].abs()
    # (scores as above, in base 2, and the sum's own roundings)
    assert (e <= ((step + 2.0 ** -19 * size)[..., 0][~empty] * 1.5 + 2.0 ** -14 + 2.0 ** -22 * want_lse[~empty].abs())).all()
    return out, lse


def case(seed, Z, H, N, dc, dr, page, dtype, lens, causal, spread=0.5, sm=0.1, fresh=None, rope=None, extra=1, size=1.5):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(0, n) // page) for n in lens) + 3
    table = make_table(g, [max(0, n) for n in lens], page, pages, extra)
    check(queries(g, Z, H, N, dc, dr, dtype, size), make_pool(g, pages, page, dc, dr, spread), table, lens, causal, sm, fresh, rope)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dc,dr", [(128, 32), (128, 64), (256, 32), (256, 64), (512, 32), (512, 64)])
@pytest.mark.parametrize("H,N", [(1, 1), (16, 1), (20, 1), (33, 1), (128, 1), (16, 5)])
def test_shapes(dtype, dc, dr, H, N):
    """One tile of 16, 32 and 64 rows, several tiles, several tokens."""
    case(dc + dr + H, 3, H, N, dc, dr, 16, dtype, [77, 200, 5 if N == 5 else 1], N > 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dr,pairs", [(64, 32), (64, 24), (64, 8), (32, 16), (32, 8)])
@pytest.mark.parametrize("H,N", [(16, 1), (8, 12)])
def test_rotated_queries(dtype, interleaved, dr, pairs, H, N):
    case(pairs + H, 2, H, N, 256, dr, 32, dtype, [300, 41], N > 1, rope=dict(freqs=freqs_of(pairs), magnitude=1.125, interleaved=interleaved))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 129, 1000])
def test_lengths(page, n):
    case(n * page, 2, 16, 1, 512, 64, page, torch.bfloat16, [n, 3 * n], False)


@pytest.mark.parametrize("H,N", [(16, 1), (64, 1), (5, 9)])
def test_lengths_that_differ(H, N):
    """From no key to many; lengths below zero and behind the table's end; causal rows that see nothing."""
    case(H, 7, H, N, 512, 64, 16, torch.float16, [0, 1, 500, 3, -4, 64, 161], True, extra=0)
    g = torch.Generator().manual_seed(1)
    pool, table = make_pool(g, 9, 16, 256, 64), torch.tensor([[4, 7], [0, 3]], dtype=torch.int32)
    check(queries(g, 2, H, N, 256, 64, torch.bfloat16), pool, table, [1000, 20], False)


@pytest.mark.parametrize("H,N,fresh", [(16, 4, [4, 0, 1, 3]), (3, 50, [50, 7, 0, -2]), (16, 1, [1, 0, 5, 1])])
def test_new_tokens_that_differ(H, N, fresh):
    case(N, 4, H, N, 512, 64, 32, torch.bfloat16, [70, 300, 12, 100], True, fresh=fresh, rope=dict(freqs=freqs_of(32)))
    case(N, 4, H, N, 128, 32, 32, torch.float16, [70, 300, 12, 100], False, fresh=fresh)


def test_pages_that_are_none():
    g = torch.Generator().manual_seed(3)
    for H in (16, 64):
        table = make_table(g, [200, 90, 30], 16, 40)
        table[0, 3], table[0, 8], table[1, 0], table[2, :2] = -1, 40, 2 ** 31 - 1, -5
        check(queries(g, 3, H, 2, 512, 64, torch.float16), make_pool(g, 40, 16, 512, 64), table, [200, 90, 30], True)


def test_hidden_places_may_hold_anything():
    """Rows behind a sequence's end, and what the scales there hold, have no part in it."""
    g = torch.Generator().manual_seed(5)
    for H, N in ((16, 1), (64, 3)):
        pool, table, lens = make_pool(g, 12, 32, 512, 64), make_table(g, [70, 100], 32, 12), [70, 100]
        q = queries(g, 2, H, N, 512, 64, torch.bfloat16)
        want = run(q, pool, table, lens, N > 1)
        for z, n in enumerate(lens):
            p = int(table[z, n // 32])
            pool[0][p, n % 32:], pool[1][p, n % 32:] = -128, math.nan
        unused = [p for p in range(12) if p not in table.flatten().tolist()]
        pool[1][unused] = math.inf
        for a, b in zip(run(q, pool, table, lens, N > 1), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("spread", [0.0, 3.0, 20.0])
def test_scales_that_differ(H, spread):
    """Tokens whose scales are up to e^40 apart, keys small and large: scores stay of a size."""
    g = torch.Generator().manual_seed(int(spread) + H)
    cache, scale = make_pool(g, 30, 16, 512, 64, spread)
    check(queries(g, 2, H, 1, 512, 64, torch.float16, 1.0 if spread < 10 else 1e-4), (cache, scale), make_table(g, [250, 100], 16, 30), [250, 100], False,
          0.1 if spread < 10 else 1e-4)


@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -60, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("H", [4, 64])
def test_values_of_any_size(H, size):
    """Latent vectors of these sizes with queries that leave scores of about one, in bf16."""
    g = torch.Generator().manual_seed(7)
    cache, scale = make_pool(g, 20, 16, 512, 64, 1.0)
    scale[..., 0] = torch.clamp(scale[..., 0].double() * size, min=2.0 ** -100).float()
    q = queries(g, 1, H, 1, 512, 64, torch.bfloat16)
    q = (torch.clamp(q[0].double() / max(size, 2.0 ** -95), -2.0 ** 100, 2.0 ** 100).bfloat16(), q[1] * 0)
    check(q, (cache, scale), make_table(g, [150], 16, 20), [150], False)


def test_zero_rows_and_sinks():
    """Tokens of zeros (their scale the least there is) that take most of the weight, beside many that share the rest."""
    g = torch.Generator().manual_seed(11)
    for H in (16, 64):
        cache, scale = make_pool(g, 70, 64, 512, 64)
        table = make_table(g, [64 * 64], 64, 70)
        p = int(table[0, 0])
        cache[p, 0, :512], scale[p, 0, 0] = 0, 2.0 ** -100
        cache[p, 0, 512:], scale[p, 0, 1] = 127, 12.0 / 64 / 127
        q = queries(g, 1, H, 1, 512, 64, torch.bfloat16, 0.3)
        q[1][:] = 1.0
        check(q, (cache, scale), table, [64 * 64], False, 1.0)
        cache[:, :, :512], scale[..., 0] = 0, 2.0 ** -100
        check(q, (cache, scale), table, [64 * 64], False, 1.0)
        scale[..., 0] = 0.0
        out, lse = run(q, (cache, scale), table, [64 * 64], False, 1.0)
        assert (out == 0).all() and lse.isfinite().all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_queries_that_hold_no_number(bad):
    """Their rows are none, and no other row is touched; without a key they are zeros all the same."""
    g = torch.Generator().manual_seed(13)
    for H in (16, 64):
        pool, table = make_pool(g, 12, 16, 512, 64), make_table(g, [90, 40], 16, 12)
        q = queries(g, 2, H, 1, 512, 64, torch.float16)
        want, want_lse = run(q, pool, table, [90, 0], False)
        q[0][0, 3, 0, 7], q[1][0, 5, 0, 60], q[0][1, 2] = bad, bad, bad
        out, lse = run(q, pool, table, [90, 0], False)
        assert out[0, [3, 5]].isnan().all() and lse[0, [3, 5]].isnan().all() and (out[1] == 0).all() and (lse[1] == -math.inf).all()
        others = [h for h in range(H) if h not in (3, 5)]
        assert torch.equal(out[0, others], want[0, others]) and torch.equal(lse[0, others], want_lse[0, others])


@pytest.mark.parametrize("sm", [-0.1, 0.0, 30.0])
def test_scales_of_scores(sm):
    case(17, 2, 16, 1, 512, 64, 32, torch.float16, [200, 100], False, sm=sm, size=0.05 if sm > 1 else 1.5)
    case(17, 1, 64, 1, 256, 64, 32, torch.bfloat16, [200], False, sm=sm, size=0.05 if sm > 1 else 1.5)


def test_many_keys_and_pieces():
    """Long sequences of few rows, which many workgroups share; a batch of very different lengths beside them."""
    case(19, 1, 16, 1, 512, 64, 64, torch.bfloat16, [20000], False, extra=0)
    case(23, 1, 128, 1, 256, 32, 128, torch.float16, [9000], False, extra=0)
    case(29, 9, 16, 2, 128, 64, 16, torch.bfloat16, [5000, 1, 0, 700, 64, 2, 3000, 33, 9], True)


def test_many_tiles():
    """A chunk of a prompt: more row tiles than workgroups; a workgroup has several items, whole ones and parts."""
    case(31, 2, 40, 70, 128, 32, 32, torch.float16, [70, 300], True, rope=dict(freqs=freqs_of(16)))
    case(37, 1, 128, 130, 128, 64, 64, torch.bfloat16, [400], True)


def test_strides():
    g = torch.Generator().manual_seed(41)
    pool, table, lens = make_pool(g, 20, 16, 512, 64), make_table(g, [100, 150], 16, 20), [100, 150]
    wide = torch.randn((2, 3, 16, 512 + 64 + 16), generator=g).bfloat16()
    q = wide[..., :512].transpose(1, 2), wide[..., 528:].transpose(1, 2)
    want = run(tuple(x.contiguous() for x in q), pool, table, lens, True)
    rows = torch.zeros((20, 2, 16, 608), dtype=torch.int8)
    rows[:, 1, :, 16:592] = pool[0]
    table = widened(table, q[0], 16, lens)
    scales = torch.zeros((20, 16, 4))
    scales[..., 2:] = pool[1]
    i32 = dict(dtype=torch.int32, device="cuda")
    dev = wide.cuda()
    got = ifa.attention_paged_latent_int8(dev[..., :512].transpose(1, 2), dev[..., 528:].transpose(1, 2), rows.cuda()[:, 1, :, 16:592], scales.cuda()[..., 2:],
                                          torch.cat([table, table], 1).cuda()[:, :table.shape[1]], torch.tensor(lens, **i32), True, 0.1, return_lse=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    odd = torch.randn((2, 16, 1, 513), generator=g).bfloat16()[..., 1:]
    a = run((odd, q[1][:, :, :1]), pool, table, lens, False)
    b = run((odd.contiguous(), q[1][:, :, :1].contiguous()), pool, table, lens, False)
    assert torch.equal(a[0], b[0])


def test_cache_behind_4_gib():
    pages = (4 << 30) // (64 * 576) + 9
    cache = torch.zeros((pages, 64, 576), dtype=torch.int8, device="cuda")
    scale = torch.zeros((pages, 64, 2), device="cuda")
    g = torch.Generator().manual_seed(43)
    small = make_pool(g, 5, 64, 512, 64)
    for at in (2, pages - 6):
        cache[at:at + 5], scale[at:at + 5] = small[0].cuda(), small[1].cuda()
    table = torch.tensor([[2, 4, 3, 6, 5]], dtype=torch.int32)
    i32 = dict(dtype=torch.int32, device="cuda")
    for H in (16, 64):
        q = [x.cuda() for x in queries(g, 1, H, 1, 512, 64, torch.float16)]
        table = widened(table, q[0], 64, [300])
        outs = [ifa.attention_paged_latent_int8(*q, cache, scale, (table + off).cuda(), torch.tensor([300], **i32), False, 0.1) for off in (0, pages - 8)]
        assert torch.equal(*outs) and outs[0].abs().max() > 0

"""Attention over pages where the formula gives numbers and a step on the way to them could fail to: scores, queries and scales of values of any size
that their types hold."""
import math

import pytest
import torch

import int_flashattention_amd as M
from paged_reference import attend, bound, make_cache, make_table

pytestmark = pytest.mark.gpu
DEV = "cuda"


def call(q, kv, sc, table, lens, sm, causal=False, **kw):
    kv_d, sc_d = kv.to(DEV), sc.to(DEV)
    o, lse = M.attention_paged_int8(q.to(DEV), kv_d[:, 0], kv_d[:, 1], sc_d[:, 0], sc_d[:, 1], table.to(DEV),
                                    torch.tensor(lens, dtype=torch.int32, device=DEV), causal, sm, return_lse=True, **kw)
    torch.cuda.synchronize()
    return o.cpu(), lse.cpu()


def of_page(x, table, z, n):
    """Rows [H, n, d] of sequence z."""
    page = x.shape[2]
    return x[table[z, :(n + page - 1) // page].long()].transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n]


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("N,d", [(1, 64), (3, 128), (20, 256), (100, 64), (100, 128), (100, 256)])
@pytest.mark.parametrize("size", [16.0, 19.9, 20.1, 23.0, 24.3, 25.4, 25.8, 26.5, 27.5, 28.4, 30.0, 40.0, 100.0])
def test_scores_of_any_size(N, d, page, size):
    """Each query is a multiple of one key, whose score in base 2 is about 2^size and several times that of any other: the softmax is that key's, its value the
    output to half a step and P's rounding.  (The scores of the others are behind by more than a tenth of 2^size, which exceeds every rounding of a score, 2^-18 of
    it, and 30 from size 10 on.)"""
    g = torch.Generator().manual_seed(int(10 * size) + N + d)
    n = 4 * 64 + 7
    cache, kv, sc = make_cache(g, n // page + 3, 1, page, d)
    kv[:, 0] = torch.where(torch.rand(kv[:, 0].shape, generator=g) < 0.5, -1, 1).to(torch.int8) * torch.randint(60, 90, kv[:, 0].shape, generator=g, dtype=torch.int8)
    sc[:, 0] = 0.5
    table = make_table(g, [n], page, kv.shape[0])
    keys, values = of_page(cache["k"], table, 0, n)[0], of_page(cache["v"].float() * cache["vs"][..., None, None], table, 0, n)[0]
    winner = torch.randint(0, n, (N,), generator=g)
    q = keys[winner].float()[None, None].bfloat16()                              # (whole numbers to 90: exact)
    apart = keys.float() @ keys.float().T
    norm = apart.diagonal().clone()
    assert (apart - torch.diag(norm)).amax(0).div(norm.min()).max() < 0.85
    sm = 2.0 ** size * math.log(2.0) / (0.5 * norm.mean().item())
    o, lse = call(q, kv, sc, table, [n], sm)
    assert o.isfinite().all() and lse.isfinite().all()
    want = values[winner].double()
    assert ((o[0, 0].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * want.abs()).all()
    top = norm[winner].double() * 0.5 * sm / math.log(2.0)
    assert ((lse[0, 0].double() - top).abs() <= 2.0 ** -20 * top).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("size", [22.0, 23.0, 23.9, 24.6, 26.0, 27.3, 28.6])
@pytest.mark.parametrize("N", [1, 100])
def test_large_scores_that_grow_slowly(N, page, size):
    """Scores of about 2^size that grow by five in base 2 every 64 keys: a followed maximum may stay behind by as much, and the scales of values double with it."""
    g = torch.Generator().manual_seed(int(10 * size) + page)
    d, n = 64, 512
    cache, kv, sc = make_cache(g, n // page, 1, page, d)
    table = torch.arange(n // page, dtype=torch.int32)[None]
    kv[:, 0] = 0
    kv[:, 0, :, :, 0] = 127
    kv[:, 0, 0, :, 1] = (torch.arange(n).reshape(-1, page) // 64).to(torch.int8)
    sc[:, 0], sc[:, 1] = 1.0, 1.9 ** (torch.arange(n // page) * page // 64)[:, None]
    q = torch.zeros((1, 1, N, d), dtype=torch.float16)
    q[..., 0], q[..., 1] = 1.0, 127.0 * 5.0 / 2.0 ** size
    sm = 2.0 ** size / 127.0 * math.log(2.0)
    o, lse = call(q, kv, sc, table, [n], sm)
    assert o.isfinite().all() and lse.isfinite().all()
    want, want_lse, mean_v, extent = attend(q, cache, table, [n], False, sm)
    assert ((o.double() - want).abs() <= bound(want, mean_v, extent, q.dtype)).all()
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -12 + 2.0 ** -18 * extent[..., 0]).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("N,d", [(1, 64), (5, 128), (30, 256), (100, 64), (100, 128), (100, 256)])
@pytest.mark.parametrize("up", [90, 105, 110, 120])
@pytest.mark.parametrize("rot", [0, 64])
def test_queries_over_the_range_of_bf16(N, d, page, up, rot):
    """Queries times 2^up with the softmax's scale by 2^-up: powers of two, so the same bits."""
    g = torch.Generator().manual_seed(up + N)
    lens = [N + 90]
    cache, kv, sc = make_cache(g, 20, 2, page, d)
    table = make_table(g, lens, page, 20)
    q = torch.randn((1, 4, N, d), generator=g).bfloat16()
    kw = dict(freqs=M.rotary_frequencies(rot, device=DEV)[0]) if rot else {}
    o, lse = call(q, kv, sc, table, lens, d ** -0.5, True, **kw)
    far, far_lse = call((q.float() * 2.0 ** up).bfloat16(), kv, sc, table, lens, d ** -0.5 * 2.0 ** -up, True, **kw)
    assert o.isfinite().all() and torch.equal(far, o) and torch.equal(far_lse, lse)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("N,d", [(1, 64), (5, 128), (30, 256), (100, 64), (100, 128), (100, 256)])
@pytest.mark.parametrize("up", [80, 100, 118])
def test_values_over_the_range_of_bf16(N, d, page, up):
    """Values of up to 2^(up + 7), thousands of them in a row with like weights: sums of them fit fp32 for as long as their mean does."""
    g = torch.Generator().manual_seed(up)
    lens = [5000, N]
    pages = 2 * (5000 // page + 3)
    cache, kv, sc = make_cache(g, pages, 1, page, d)
    kv[:, 1] = kv[:, 1].abs()
    sc[:, 1] = 2.0 ** up
    table = make_table(g, lens, page, pages)
    q = (0.1 * torch.randn((2, 2, N, d), generator=g)).bfloat16()
    o, lse = call(q, kv, sc, table, lens, d ** -0.5, True)
    assert o.isfinite().all() and lse.isfinite().all()
    want, _, mean_v, extent = attend(q, cache, table, lens, True, d ** -0.5)
    assert ((o.double() - want).abs() <= bound(want, mean_v, extent, q.dtype)).all()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("N,d", [(1, 64), (5, 128), (100, 64), (100, 128), (100, 256)])
@pytest.mark.parametrize("up,order", [(60, 0), (60, 1), (90, 0), (90, 1), (115, 0), (115, 1)])
def test_pages_of_zeros_beside_large_values(N, d, page, up, order):
    """Every other page holds zeros at the least scale that an append leaves, 2^-100; the others' scale is 2^up."""
    g = torch.Generator().manual_seed(up + page)
    lens = [700]
    pages = 700 // page + 3
    cache, kv, sc = make_cache(g, pages, 1, page, d)
    table = make_table(g, lens, page, pages)
    sc[:, 1] = 2.0 ** up
    zeros = table[0, order::2].long()
    kv[zeros, 1], sc[zeros, 1] = 0, 2.0 ** -100
    q = (0.5 * torch.randn((1, 2, N, d), generator=g)).bfloat16()
    o, lse = call(q, kv, sc, table, lens, d ** -0.5)
    assert o.isfinite().all() and lse.isfinite().all()
    want, want_lse, mean_v, extent = attend(q, cache, table, lens, False, d ** -0.5)
    assert ((o.double() - want).abs() <= bound(want, mean_v, extent, q.dtype)).all()
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -12 + 2.0 ** -18 * extent[..., 0]).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("N", [1, 70])
@pytest.mark.parametrize("scale,first", [(2.0 ** -5, 1.0), (2.0 ** -9.9, 1.0), (2.0 ** 9, 1.0), (2.0 ** -3, 2.0 ** 9.9), (2.0 ** -3, 2.0 ** 3.9)])
def test_many_keys_of_small_weight(N, page, scale, first):
    """32768 keys that each weigh 2^-14.6 of the first one, and together more than it: their weights keep 11 bits whatever the scale of the values, or one
    of another page.  512 sequences of the same pages, so that no workgroup has only part of one.  (All weights are the same, so a rounding coarser than that does not average out; in steps of 2^-24 a weight of
    2^(8 - 9.9 - 14.6033) is 180.6.)"""
    g = torch.Generator().manual_seed(3)
    Z, d, n = 512, 64, 1 << 15
    cache, kv, sc = make_cache(g, n // page, 1, page, d)
    table = torch.arange(n // page, dtype=torch.int32)[None]
    kv[:, 0] = 0
    kv[0, 0, 0, 0, 0] = 100
    kv[:, 1] = torch.randint(100, 127, (1, 1, 1, d), generator=g, dtype=torch.int8)
    kv[0, 1] = 0
    sc[:, 0], sc[:, 1] = 1.0, scale
    sc[0, 1] = scale * first                                 # (of the first key's page, whose values are zeros)
    q = torch.zeros((1, 1, N, d), dtype=torch.float16)
    q[..., 0] = 1.0
    sm = 14.6033 / 100.0 * math.log(2.0)
    o, _ = call(q.expand(Z, 1, N, d), kv, sc, table.expand(Z, -1), [n] * Z, sm)
    want, _, mean_v, extent = attend(q, cache, table, [n], False, sm)
    assert ((o.double() - want).abs() <= bound(want, mean_v, extent, q.dtype)).all()

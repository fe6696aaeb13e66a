"""Attention over a paged latent cache where the scales of a row's tokens are far apart: tokens of zeros (their scale is the least there is) beside large ones, first and last, few and many."""
import math

import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import attend, make_pool
from paged_reference import make_table
from test_gpu_latent_attention import bound, queries

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -100


def check(q, pool, table, lens, sm=1.0, rotary_alone=False):
    """rotary_alone: the latent queries are zeros, whose steps are exact.  Tolerances: as where scales are alike, and of the logarithms of scales (within 2^8, half a step of fp32 is
    2^-17 there): the logarithm itself, a score and it added, their differences from the row's frame and the logarithm taken out again, at most nine such roundings in the weights
    of values and of the sum, times ln 2: less than 2^-14 of a weight."""
    i32 = dict(dtype=torch.int32, device="cuda")
    out, lse = (x.cpu() for x in ifa.attention_paged_latent_int8(q[0].cuda(), q[1].cuda(), pool[0].cuda(), pool[1].cuda(), table.cuda(), torch.tensor(lens, **i32), False, sm, return_lse=True))
    want, want_lse, mean_v, size, step = attend(*q, *pool, table, lens, False, sm)
    if rotary_alone:
        size, step = attend(*q, pool[0], pool[1] * torch.tensor([0.0, 1.0]), table, lens, False, sm)[3:]
    d, b = (out.double() - want).abs(), bound(want, mean_v, size, step, out.dtype) + 2.0 ** -14 * mean_v
    assert (d <= b).all(), f"{(d / b).max():.3f} of the bound"
    b = (step + 2.0 ** -19 * size)[..., 0] * 1.5 + 2.0 ** -13 + 2.0 ** -22 * want_lse.abs()
    assert b.max() < 2.0 ** -4                 # (the sum of weights is known to 4 % at the least: more than that missing shows)
    assert ((lse.double() - want_lse).abs() <= b).all()


def pool_of(g, pages, page, size):
    cache, scale = make_pool(g, pages, page, 512, 64, 0.5)
    return cache, (scale.double() * size).float()


def zero(pool, table, page, tokens):
    for i in tokens:
        p, r = int(table[0, i // page]), i % page
        pool[0][p, r, :512], pool[1][p, r, 0] = 0, LEAST


@pytest.mark.parametrize("size", [2.0 ** 6, 2.0 ** 15, 2.0 ** 30, 2.0 ** 60, 2.0 ** 95])
@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("n,where", [(200, [0]), (200, [199]), (200, [70]), (200, list(range(64))), (200, list(range(100, 200))), (200, list(range(1, 200))), (2, [0]), (2, [1]),
                                     (9000, list(range(0, 4500))), (9000, [8999]), (9000, [0])])
def test_tokens_of_zeros_beside_large_ones(n, where, H, size):
    """Scores of one size: a token of zeros has the weight of any other."""
    g, page = torch.Generator().manual_seed(n + len(where)), 32
    pages = -(-n // page) + 2
    pool, table = pool_of(g, pages, page, size), make_table(g, [n], page, pages)
    zero(pool, table, page, where)
    q = [(x / size).bfloat16() for x in queries(g, 1, H, 1, 512, 64, torch.bfloat16)]
    check(q, pool, table, [n], 0.3)


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 95])
@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("at", [0, 1500, 2999])
def test_a_sink_of_zeros(at, H, size):
    """One token of zeros with nearly all of the weight."""
    g, page, n = torch.Generator().manual_seed(at), 64, 3000
    pool, table = pool_of(g, 50, page, size), make_table(g, [n], page, 50)
    zero(pool, table, page, [at])
    p, r = int(table[0, at // page]), at % page
    pool[0][p, r, 512:], pool[1][p, r, 1] = 127, size * 12.0 / 64 / 127
    q = queries(g, 1, H, 1, 512, 64, torch.bfloat16, 0.3)
    check(((q[0] / size).bfloat16(), torch.ones_like(q[1]) / size), pool, table, [n], 1.0)


@pytest.mark.parametrize("H", [1, 20, 64])
@pytest.mark.parametrize("seed", range(4))
def test_scales_of_all_sizes(seed, H):
    """Scales from 2^-100 to 2^110, in any order; scores come of the rotary parts alone."""
    g, page, n = torch.Generator().manual_seed(seed), 16, 300 if seed < 3 else 7000
    pages = -(-n // page) + 1
    cache, scale = make_pool(g, pages, page, 256, 32, 0.5)
    scale[..., 0] = torch.exp2(torch.rand(scale.shape[:2], generator=g).double() * 210 - 100).float()
    table = make_table(g, [n], page, pages)
    q = queries(g, 1, H, 1, 256, 32, torch.bfloat16, 1.0)
    check((q[0] * 0, q[1]), (cache, scale), table, [n], 0.4, rotary_alone=True)


@pytest.mark.parametrize("H", [16, 64])
def test_very_many_tokens_of_zeros(H):
    """2^22 of them on one page (a table may name it as often as it likes): their weights' sum has a place in fp32, in every piece and all together; and a value beside them."""
    page, columns = 256, 1 << 14
    cache, scale = torch.zeros((2, page, 160), dtype=torch.int8), torch.full((2, page, 2), LEAST)
    cache[0, :, 128:], scale[..., 1] = 1, 1.0
    cache[1, :, :128], scale[1, :, 0] = 100, 2.0 ** 20
    q_latent, q_rope = torch.zeros((1, H, 1, 128), dtype=torch.bfloat16), torch.full((1, H, 1, 32), 2.0, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    for large in (None, 0, columns - 1):
        table = torch.zeros((1, columns), **i32)
        if large is not None:
            table[0, large] = 1                # (256 values of 100 * 2^20, with scores of 0)
        out, lse = ifa.attention_paged_latent_int8(q_latent.cuda(), q_rope.cuda(), cache.cuda(), scale.cuda(), table, torch.tensor([page * columns], **i32), False, 0.25, return_lse=True)
        zeros, others = page * (columns - (large is not None)) * math.exp(16.0), page * (large is not None)
        # (queries of powers of two, exact scores; the sum's roundings: a lane's terms in each of its pieces and the joins, 2^-24 for each of at most 2^10 in a row)
        assert (lse.double() - math.log2(zeros + others)).abs().max() <= 2.0 ** -13
        want = others / (zeros + others) * 100 * 2.0 ** 20
        assert (out.double() - want).abs().max() <= want * (2.0 ** -8 + 2.0 ** -10)

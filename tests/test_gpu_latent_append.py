"""The append to a latent cache against its formula in float64.

A value's place between two int8 numbers is known to the rounding of its fp32 steps alone: q is right if it is within half a step, and a little, of the exact quotient."""
import math

import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import append, make_pool
from paged_reference import make_table

pytestmark = pytest.mark.gpu


def check(cache, scale, before, values, scales, new, dc):
    """Of the fp32 steps: a norm sums up to 512 squares in a tree (2^-24 for each of its nine levels and of a lane's eight, half of it through the root) and rounds five times more;
    a turn rounds three times beside its angle's 2^-22 (sine and cosine).  2^-20 of the part's largest value covers either, which is 127 * 2^-20 of a step."""
    cache, scale = cache.cpu(), scale.cpu()
    assert torch.equal(cache[~new], before[0][~new]) and torch.equal(scale[~new], before[1][~new])
    assert (scale.double() / scales - 1).abs()[new].max() <= 2.0 ** -20
    for part, cols in ((0, slice(0, dc)), (1, slice(dc, None))):
        q, x = cache[..., cols][new].double(), values[..., cols][new]
        s = scales[..., part][new][:, None]
        want = torch.nan_to_num(x / s, nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127)
        assert (q - want).abs().max() <= 0.5 + 127 * 2.0 ** -19


def case(g, Z, N, dc, dr, page, dtype, lens, fresh=None, rope=None, interleaved=False, norm=False, extra=0, change=None, hole=False):
    top = max(max(0, n) for n in lens) + N
    pages = Z * (top // page + 2) + 3
    table = make_table(g, [max(0, n) + N for n in lens], page, pages, extra)
    if hole:
        table[0, max(0, lens[0]) // page] = -1
    cache, scale = make_pool(g, pages, page, dc, dr)
    c, k = torch.randn((Z, N, dc), generator=g).mul(3).to(dtype), torch.randn((Z, N, dr), generator=g).to(dtype)
    if change:
        change(c, k)
    weight = (1 + 0.3 * torch.randn((dc,), generator=g)).to(dtype) if norm else None
    freqs = None if rope is None else 10000.0 ** (-torch.arange(rope, dtype=torch.float64) / rope)
    magnitude = 1.0 if rope is None else 1.25
    want = append(cache, scale, c, k, table, lens, fresh, None if rope is None else dict(freqs=freqs, magnitude=magnitude, interleaved=interleaved), weight, 1e-5)
    dev = cache.cuda(), scale.cuda()
    ifa.paged_latent_append(*dev, c.cuda(), k.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), None if rope is None else freqs.cuda(),
                            interleaved=interleaved, magnitude=magnitude, seqlens_new=None if fresh is None else torch.tensor(fresh, dtype=torch.int32, device="cuda"),
                            norm_weight=None if weight is None else weight.cuda(), norm_eps=1e-5)
    check(*dev, (cache, scale), *want, dc)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dc,dr", [(128, 32), (128, 64), (256, 32), (256, 64), (512, 32), (512, 64)])
@pytest.mark.parametrize("norm,rope,interleaved", [(False, None, False), (True, 0, False), (True, 0, True), (False, 8, False), (True, 16, True)])
def test_append(dtype, dc, dr, norm, rope, interleaved):
    """rope 0: all of the rotary part; 8 and 16 pairs: a part of it."""
    g = torch.Generator().manual_seed(dc + dr + 7 * norm + (rope or 0))
    case(g, 3, 37, dc, dr, 16, dtype, [0, 100, 31], rope=None if rope is None else rope or dr // 2, interleaved=interleaved, norm=norm)


@pytest.mark.parametrize("N", [1, 2, 5])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_few_tokens(N, page):
    g = torch.Generator().manual_seed(N * page)
    case(g, 5, N, 512, 64, page, torch.bfloat16, [0, page - 1, page, 3 * page + 5, 777], rope=32, norm=True)


def test_lengths_that_differ_and_rows_that_have_no_place():
    """Fewer rows than the batch holds, none, more than there are; lengths below zero; columns behind the table and pages that are none."""
    g = torch.Generator().manual_seed(2)
    case(g, 6, 20, 512, 64, 16, torch.float16, [-5, 0, 40, 16, 3, 90], fresh=[20, 0, 7, -2, 500, 1], rope=32)
    case(g, 2, 40, 256, 32, 16, torch.bfloat16, [10, 33], hole=True, norm=True)
    cache, scale = make_pool(g, 4, 16, 512, 64)
    dev, table = (cache.cuda(), scale.cuda()), torch.tensor([[2, 1], [0, 9]], dtype=torch.int32)
    c, k = torch.randn((2, 30, 512), generator=g).half(), torch.randn((2, 30, 64), generator=g).half()
    lens = [17, 2 ** 31 - 5]
    want = append(cache, scale, c, k, table, lens)
    ifa.paged_latent_append(*dev, c.cuda(), k.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    check(*dev, (cache, scale), *want, 512)


def test_far_positions():
    """Angles of positions that fp32 does not hold."""
    g = torch.Generator().manual_seed(4)
    page, n = 256, 2 ** 24 + 3
    cache, scale = make_pool(g, 2, page, 128, 64)
    table = torch.full((1, n // page + 1), -1, dtype=torch.int32)
    table[0, -1] = 1
    c, k = torch.randn((1, 9, 128), generator=g).half(), torch.randn((1, 9, 64), generator=g).half()
    freqs = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    want = append(cache, scale, c, k, table, [n], rope=dict(freqs=freqs))
    dev = cache.cuda(), scale.cuda()
    ifa.paged_latent_append(*dev, c.cuda(), k.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), freqs.cuda())
    check(*dev, (cache, scale), *want, 128)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -130, 2.0 ** -70, 2.0 ** 60, 2.0 ** 126])
def test_rows_of_any_size(norm, size):
    """bf16's whole range: squares of these leave fp32's, their norm does not."""
    g = torch.Generator().manual_seed(6)

    def change(c, k):
        c[0, 1] = (torch.randn(512, generator=g).clamp(-1.9, 1.9) * size).to(c.dtype)
        c[0, 2, 5] = size
        k[0, 1] = (torch.randn(64, generator=g).clamp(-1.9, 1.9) * size).to(k.dtype)
    case(g, 1, 4, 512, 64, 16, torch.bfloat16, [3], norm=norm, change=change)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(bad):
    """They do not count for their part's scale and touch no other token; through a norm a row that holds one becomes zeros."""
    g = torch.Generator().manual_seed(8)

    def change(c, k):
        c[0, 1, 7] = bad
        k[1, 0, 3] = bad
        k[1, 2] = bad
        c[1, 1] = bad
    case(g, 2, 5, 512, 64, 16, torch.bfloat16, [3, 14], change=change)
    cache, scale = (x.cuda() for x in make_pool(g, 2, 16, 512, 64))
    c, k = torch.randn((1, 3, 512), generator=g).bfloat16().cuda(), torch.randn((1, 3, 64), generator=g).bfloat16().cuda()
    c[0, 1, 7] = bad
    ifa.paged_latent_append(cache, scale, c, k, torch.tensor([[1]], dtype=torch.int32, device="cuda"), torch.tensor([0], dtype=torch.int32, device="cuda"),
                            norm_weight=torch.ones(512, dtype=torch.bfloat16, device="cuda"))
    assert (cache[1, 1, :512] == 0).all() and scale[1, 1, 0] == 2.0 ** -100
    assert cache[1, 0, :512].abs().max() == 127 and cache[1, 2, :512].abs().max() == 127


def test_strides():
    """New rows that are slices of a projection, pages of a wider tensor, scales that lie apart, a table inside a wider one: the result is that of contiguous ones."""
    g = torch.Generator().manual_seed(10)
    wide = torch.randn((4, 9, 512 + 64 + 32), generator=g).bfloat16().cuda()
    c, k = wide[..., 16:528], wide[..., 528:592]
    pool = torch.zeros((7, 2, 16, 640), dtype=torch.int8, device="cuda")
    scales = torch.zeros((7, 16, 6), device="cuda")
    table = torch.full((4, 8), -1, dtype=torch.int32, device="cuda")
    table[:, 3] = torch.tensor([6, 0, 2, 3])
    lens = torch.tensor([0, 5, 7, 1], dtype=torch.int32, device="cuda")
    ifa.paged_latent_append(pool[:, 1, :, 32:608], scales[..., 2:4], c, k, table[:, 3:], lens)
    other = torch.zeros((7, 16, 576), dtype=torch.int8, device="cuda"), torch.zeros((7, 16, 2), device="cuda")
    ifa.paged_latent_append(*other, c.contiguous(), k.contiguous(), table[:, 3:].contiguous(), lens)
    assert torch.equal(pool[:, 1, :, 32:608], other[0]) and torch.equal(scales[..., 2:4], other[1])
    assert (pool[:, 0] == 0).all() and (pool[:, 1, :, :32] == 0).all() and (pool[:, 1, :, 608:] == 0).all() and (scales[..., :2] == 0).all() and (scales[..., 4:] == 0).all()
    # (rows that start off their 16 bytes are copied first)
    odd = wide[..., 3:515]
    ifa.paged_latent_append(pool[:, 0, :, :576], scales[..., 4:], odd, k, table[:, 3:], lens)
    ifa.paged_latent_append(*other, odd.contiguous(), k, table[:, 3:], lens)
    assert torch.equal(pool[:, 0, :, :576], other[0])


def test_pages_behind_4_gib():
    pages = (4 << 30) // (64 * 576) + 5
    cache = torch.empty((pages, 64, 576), dtype=torch.int8, device="cuda")
    scale = torch.zeros((pages, 64, 2), device="cuda")
    g = torch.Generator().manual_seed(12)
    c, k = torch.randn((1, 3, 512), generator=g).half().cuda(), torch.randn((1, 3, 64), generator=g).half().cuda()
    lens = torch.tensor([10], dtype=torch.int32, device="cuda")
    for page in (0, pages - 1):
        ifa.paged_latent_append(cache, scale, c, k, torch.tensor([[page]], dtype=torch.int32, device="cuda"), lens)
    assert torch.equal(cache[0, 10:13], cache[-1, 10:13]) and torch.equal(scale[0], scale[-1]) and scale[0, 10:13].min() > 0

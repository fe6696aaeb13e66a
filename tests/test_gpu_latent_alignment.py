"""Inputs that are contiguous, but off their 16 bytes, or with a stride of a single entry that is: the result is that of aligned ones."""
import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import make_pool

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def off(x):
    """The same numbers from an odd place of a buffer on."""
    y = torch.empty(x.numel() + 9, dtype=x.dtype, device=x.device)[1:1 + x.numel()].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16
    return y


def single(x):
    """[1, ...] whose first stride is odd."""
    y = torch.empty(x.numel() + 8, dtype=x.dtype, device=x.device).as_strided(x.shape, (x.numel() + 1, *x.stride()[1:]))
    y.copy_(x)
    assert y.is_contiguous() and y.stride(0) % 8
    return y


@pytest.mark.parametrize("moved", [off, single])
def test_attention(moved):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g).bfloat16().cuda()  # noqa: E731
    x = r(1, 4, 20, 128), r(1, 4, 20, 64), r(1, 4, 33, 128), r(1, 1, 33, 64), r(1, 4, 33, 128)
    assert torch.equal(ifa.attention_latent(*(moved(t) for t in x), True, 0.07), ifa.attention_latent(*x, True, 0.07))
    pool, q = [t.cuda() for t in make_pool(g, 3, 16, 128, 64)], x[:2]
    rest = *pool, torch.tensor([[2, 0, 1]], **I32), torch.tensor([40], **I32), True, 0.07
    assert torch.equal(ifa.attention_paged_latent_int8(*(moved(t) for t in q), *rest), ifa.attention_paged_latent_int8(*q, *rest))


@pytest.mark.parametrize("moved", [off, single])
def test_append(moved):
    g = torch.Generator().manual_seed(2)
    c, k = torch.randn((1, 5, 256), generator=g).half().cuda(), torch.randn((1, 5, 32), generator=g).half().cuda()
    weight = torch.randn(256, generator=g).half().cuda()
    pools = [[t.cuda() for t in make_pool(torch.Generator().manual_seed(3), 2, 16, 256, 32)] for _ in range(2)]
    rest = torch.tensor([[1]], **I32), torch.tensor([2], **I32)
    ifa.paged_latent_append(*pools[0], c, k, *rest, norm_weight=weight)
    ifa.paged_latent_append(*pools[1], moved(c), moved(k), *rest, norm_weight=off(weight))
    for a, b in zip(*pools):
        assert torch.equal(a, b)

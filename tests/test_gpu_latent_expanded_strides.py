"""Keys and values of the expanded form whose rows lie otherwise than one behind the other: over each other, very far apart, a single one at any stride."""
import pytest
import torch

import int_flashattention_amd as ifa
from test_gpu_latent_expanded import DIMS

pytestmark = pytest.mark.gpu


def tensors(g, dims, Nk, H=3, N=5):
    dn, dr, dv = dims
    return [torch.randn(s, generator=g).half().cuda() for s in ((1, H, N, dn), (1, H, N, dr), (1, H, Nk, dn), (1, 1, Nk, dr), (1, H, Nk, dv))]


@pytest.mark.parametrize("dims", DIMS)
def test_broadcast_rows(dims):
    """One key for all places, and one head for all: strides of 0."""
    q, qr, k, kr, v = tensors(torch.Generator().manual_seed(1), dims, 90)
    k1, kr1, v1 = k[:, :, :1].expand_as(k), kr[:, :, :1].expand_as(kr), v[:, :1].expand_as(v)
    got = ifa.attention_latent(q, qr, k1, kr1, v1, True, 0.07)
    assert torch.equal(got, ifa.attention_latent(q, qr, k1.contiguous(), kr1.contiguous(), v1.contiguous(), True, 0.07)) and got.isfinite().all()


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("stride", [(1 << 24) - 8, 1 << 24, (1 << 25) + 8])
def test_rows_that_lie_far_apart(dims, stride):
    """200 rows of 2^24 elements and more apart (of one allocation, filled where they are)."""
    dn, dr, dv = dims
    q, qr, k, kr, v = tensors(torch.Generator().manual_seed(2), dims, 200, H=1)
    room = torch.empty(200 * stride, dtype=torch.float16, device="cuda")
    k2, kr2, v2 = (room[at:].as_strided((1, 1, 200, d), (0, 0, stride, 1)) for at, d in ((0, dn), (256, dr), (512, dv)))
    for a, b in ((k2, k), (kr2, kr), (v2, v)):
        a.copy_(b)
    for causal in (False, True):
        assert torch.equal(ifa.attention_latent(q, qr, k2, kr2, v2, causal, 0.07), ifa.attention_latent(q, qr, k, kr, v, causal, 0.07))


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("stride", [0, 8, 1 << 30])
def test_a_single_row(dims, stride):
    q, qr, k, kr, v = tensors(torch.Generator().manual_seed(3), dims, 1)
    a, b, c = (x.as_strided(x.shape, (x.stride(0), x.stride(1), stride, 1)) for x in (k, kr, v))
    assert torch.equal(ifa.attention_latent(q, qr, a, b, c, True, 0.07), ifa.attention_latent(q, qr, k, kr, v, True, 0.07))


def test_too_many_keys():
    x = torch.zeros((1, 1, 1, 128), dtype=torch.float16, device="cuda")
    k, kr = x.expand(1, 1, 1 << 25, 128), x[..., :64].expand(1, 1, 1 << 25, 64)
    with pytest.raises(ValueError):
        ifa.attention_latent(x, x[..., :64], k, kr, k, True, 0.1)

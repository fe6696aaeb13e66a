"""What the expanded form of latent attention reads of its keys and values: nothing behind a sequence's last one, and all of long ones whose rows lie far apart."""
import math

import pytest
import torch

import int_flashattention_amd as ifa
from test_gpu_latent_expanded import DIMS, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("copies", [1, 65])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nk", [[1, 10], [64, 129], [192, 63], [0, 65], [200, 128]])
def test_nothing_behind_the_keys_is_read(dims, copies, causal, nk):
    """Of both heads, in the split form (whose steps of the small ones take two tiles, the second of which may begin behind the last key) and in pairs of tiles: what lies there is no number, and
    would be one in no product."""
    g = torch.Generator().manual_seed(sum(nk))
    nq = [150, 100]
    x = inputs(g, 2, 2, 150, 200, dims, torch.bfloat16)
    want = run(x, causal, 0.07, nk=nk, nq=nq, copies=copies)
    for z, n in enumerate(nk):
        for t in x[2:]:
            t[z, :, n:] = math.nan
    for z, m in enumerate(nq):
        for t in x[:2]:
            t[z, :, m:] = math.nan
    for a, b in zip(run(x, causal, 0.07, nk=nk, nq=nq, copies=copies), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dims,H", [(DIMS[0], 128), (DIMS[1], 256)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N", [3, 300])
def test_keys_that_span_more_than_32_bits(dims, H, causal, N):
    """Slices of a projection of 128 wide heads, or 256 small ones: from 65408 keys on, a head's rows span 2^31 elements and more.  As the same rows side by side, to the bit, with few tiles and
    with many; nothing behind a sequence's length is read here either."""
    g = torch.Generator(device="cuda").manual_seed(N)
    (dn, dr, dv), Nk, held = dims, 65536 + 70, 65500
    kv = torch.randn((1, Nk, H, dn + dv), generator=g, device="cuda", dtype=torch.bfloat16)
    far = torch.randn((1, 1, Nk, dr), generator=g, device="cuda", dtype=torch.bfloat16)
    k, v = kv.transpose(1, 2)[..., :dn], kv.transpose(1, 2)[..., dn:]
    k_near, v_near = k.contiguous(), v.contiguous()
    q, q_rope = (torch.randn((1, H, N, d), generator=g, device="cuda", dtype=torch.bfloat16) for d in (dn, dr))
    for n in (65407, 65408, Nk):
        near = ifa.attention_latent(q, q_rope, k_near[:, :, :n], far[:, :, :n], v_near[:, :, :n], causal, 0.07, return_lse=True)
        for a, b in zip(ifa.attention_latent(q, q_rope, k[:, :, :n], far[:, :, :n], v[:, :, :n], causal, 0.07, return_lse=True), near):
            assert torch.equal(a, b)
    near = ifa.attention_latent(q, q_rope, k_near[:, :, :held], far[:, :, :held], v_near[:, :, :held], causal, 0.07)
    assert near.isfinite().all() and near.abs().max() > 0
    kv[:, held:], far[:, :, held:] = math.nan, math.nan
    assert torch.equal(ifa.attention_latent(q, q_rope, k, far, v, causal, 0.07, seqlens_k=torch.tensor([held], dtype=torch.int32, device="cuda")), near)

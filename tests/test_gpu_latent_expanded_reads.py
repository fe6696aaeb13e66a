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

"""Norms of the latent cache's append whose eps is large beside the rows: rows far under its root, whose squares are nothing beside it."""
import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import append, make_pool
from test_gpu_latent_append import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [1e-38, 1e-6, 1.0, 2.0 ** 40, 2.0 ** 60, 2.0 ** 100, 2.0 ** 127])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -38, 1.0, 2.0 ** 60, 2.0 ** 120])
@pytest.mark.parametrize("dc", [128, 512])
def test_eps_of_any_size(dc, size, eps):
    """Normalised rows from 2^-100 of a step on (their formula's scale is 2^-100 or more) and up to fp32's range."""
    g = torch.Generator().manual_seed(dc)
    cache, scale = make_pool(g, 2, 16, dc, 32)
    c, k = (torch.randn((1, 9, dc), generator=g).clamp(-1.9, 1.9) * size).bfloat16(), torch.randn((1, 9, 32), generator=g).bfloat16()
    weight = (1 + 0.3 * torch.randn((dc,), generator=g)).bfloat16()
    table, lens = torch.tensor([[1]], dtype=torch.int32), [3]
    eps = float(torch.tensor(eps))             # (as the kernel has it)
    want = append(cache, scale, c, k, table, lens, weight=weight, eps=eps)
    dev = cache.cuda(), scale.cuda()
    ifa.paged_latent_append(*dev, c.cuda(), k.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), norm_weight=weight.cuda(), norm_eps=eps)
    check(*dev, (cache, scale), *want, dc)

"""Appends to a latent cache of as many tokens as a call takes."""
import pytest
import torch

import int_flashattention_amd as ifa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dc,N", [(512, (1 << 26) + 5), (512, (1 << 28) - 16), (128, (1 << 29) - 32)])
def test_as_many_tokens_as_a_call_takes(dc, N):
    """One row over and over (the new rows' stride is 0), of which the table has places for the first and the last alone."""
    page, dr = 256, 64
    g = torch.Generator().manual_seed(N % 1000)
    c, k = (torch.randn((1, 1, d), generator=g).bfloat16().cuda() for d in (dc, dr))
    i32 = dict(dtype=torch.int32, device="cuda")
    columns = (N + page - 1) // page
    table = torch.full((1, columns), -1, **i32)
    table[0, 0], table[0, -1] = 2, 1
    cache, scale = torch.full((3, page, dc + dr), 55, dtype=torch.int8, device="cuda"), torch.full((3, page, 2), 7.0, device="cuda")
    ifa.paged_latent_append(cache, scale, c.expand(1, N, dc), k.expand(1, N, dr), table, torch.tensor([0], **i32))
    one, one_scale = torch.zeros((1, page, dc + dr), dtype=torch.int8, device="cuda"), torch.zeros((1, page, 2), device="cuda")
    ifa.paged_latent_append(one, one_scale, c, k, torch.tensor([[0]], **i32), torch.tensor([0], **i32))
    last = N - (columns - 1) * page
    for p, n in ((2, page), (1, last)):
        assert (cache[p, :n] == one[0, 0]).all() and (scale[p, :n] == one_scale[0, 0]).all()
    assert (cache[1, last:] == 55).all() and (cache[0] == 55).all() and (scale[1, last:] == 7.0).all() and (scale[0] == 7.0).all()

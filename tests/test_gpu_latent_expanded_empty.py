"""Rows of the expanded form that see no key are zeros, whatever the values that they are computed together with."""
import math

import pytest
import torch

from test_gpu_latent_expanded import DIMS, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("copies", [1, 65])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_without_a_key(bad, dims, copies, dtype):
    """More queries than keys: the first 70 of 200 rows see none, the others see values that are no number."""
    g = torch.Generator().manual_seed(21)
    x = inputs(g, 2, 2, 200, 130, dims, dtype)
    x[4][0, 1, 0], x[4][0, 1, 90, 5], x[4][1, 0, 129] = bad, bad, bad
    out, lse = run(x, True, 0.07, copies=copies)
    assert (out[:, :, :70] == 0).all() and (lse[:, :, :70] == -math.inf).all() and lse[:, :, 70:].isfinite().all()
    assert not out[0, 1, 70:].isfinite().any(-1).all() and out[0, 0, 70:].isfinite().all()
    # queries that hold no number are undefined where they see a key, and zeros where they do not
    x[0][0, 0, [3, 100]] = math.nan
    out, lse = run(x, True, 0.07, copies=copies)
    assert (out[0, 0, 3] == 0).all() and lse[0, 0, 3] == -math.inf and out[0, 0, 100].isnan().all() and lse[0, 0, 100].isnan()

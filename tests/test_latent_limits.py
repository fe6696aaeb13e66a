"""Sizes and strides that are past what the latent cache's entry points take, refused ahead of any GPU call (the largest that they do take are run in the GPU tests)."""
import math

import pytest

from int_flashattention_amd import _capi
from test_latent_host import _append, _attn_bytes, _expanded


@pytest.mark.parametrize("kw", [dict(seqlen_k=1 << 25), dict(kn_stride_n=1 << 24), dict(v_stride_n=1 << 24), dict(kr_stride_n=1 << 24), dict(kr_stride_n=56), dict(seqlen_k=(1 << 31) - 1)])
def test_keys_too_many_or_too_far_apart(kw):
    assert _expanded(**kw) == -7


@pytest.mark.parametrize("kw", [dict(batch=1, seqlen_new=(1 << 28) - 15), dict(batch=1 << 14, seqlen_new=1 << 14), dict(batch=1, seqlen_new=(1 << 29) - 31, cache__latent_dim=256),
                                dict(batch=1, seqlen_new=(1 << 29) - 31, cache__latent_dim=128), dict(batch=(1 << 31) - 1, seqlen_new=1 << 30)])
def test_appends_of_too_many_tokens(kw):
    assert _append(**kw) == -7


@pytest.mark.parametrize("kw,rows,workgroups", [
    (dict(batch=3, heads=64, seqlen=1, cache__table_width=(1 << 25) - 1), 64, 256),      # (units of 128 keys: 3 (2 + 2^23) 256 is below 2^32)
    (dict(batch=1 << 22, heads=1, seqlen=1), 32, 256),                                   # (of two units ahead and one with keys each: 3 * 2^22 * 256 is)
    (dict(batch=5_600_000, heads=1, seqlen=1), 32, 255),
    (dict(batch=1 << 24, heads=1, seqlen=1), 32, 85),
    (dict(batch=(1 << 30) - 1, heads=1, seqlen=1), 32, 1)])
def test_workspace_where_the_workgroups_become_fewer(kw, rows, workgroups):
    """Two slots of fp32 rows for each, their maxima and sums, and an open item: units are numbered in 32 bits, times the workgroups."""
    assert _attn_bytes(**kw) == workgroups * (2 * rows * (512 * 4 + 8) + 16)


def test_what_a_refusal_says():
    text = _capi.load().intfa_error_string(_append(norm_eps=math.nan)).decode()
    assert _append(norm_eps=math.nan) == _expanded(kn_stride_n=1 << 24) == -7 and "eps" in text and "strides" in text and "sizes" in text

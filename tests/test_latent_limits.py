"""Sizes and strides that are past what the latent cache's entry points take, refused ahead of any GPU call (the largest that they do take are run in the GPU tests)."""
import pytest

from test_latent_host import _append, _expanded


@pytest.mark.parametrize("kw", [dict(seqlen_k=1 << 25), dict(kn_stride_n=1 << 24), dict(v_stride_n=1 << 24), dict(kr_stride_n=1 << 24), dict(kr_stride_n=56), dict(seqlen_k=(1 << 31) - 1)])
def test_keys_too_many_or_too_far_apart(kw):
    assert _expanded(**kw) == -7


@pytest.mark.parametrize("kw", [dict(batch=1, seqlen_new=(1 << 28) - 15), dict(batch=1 << 14, seqlen_new=1 << 14), dict(batch=1, seqlen_new=(1 << 29) - 31, cache__latent_dim=256),
                                dict(batch=1, seqlen_new=(1 << 29) - 31, cache__latent_dim=128), dict(batch=(1 << 31) - 1, seqlen_new=1 << 30)])
def test_appends_of_too_many_tokens(kw):
    assert _append(**kw) == -7

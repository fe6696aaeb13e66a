"""Rotary positions and the paged cache on the host: parameter blocks, refusals ahead of any GPU call, frequencies."""
import ctypes
import math
import os
import subprocess
import tempfile

import pytest
import torch

import int_flashattention_amd as M
from int_flashattention_amd import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ADDRESS = 0x10000                      # not memory: every call below is refused before it is used


@pytest.mark.parametrize("name,mirror", [("intfa_rope", _capi.Rope), ("intfa_rotary_params", _capi.RotaryParams), ("intfa_paged_cache", _capi.PagedCache),
                                          ("intfa_paged_append_params", _capi.PagedAppendParams), ("intfa_paged_attn_params", _capi.PagedAttnParams)])
def test_blocks_match_the_header(name, mirror):
    body = "".join(f'printf("%zu ", offsetof({name}, {f[0]}));' for f in mirror._fields_)
    src = f'#include <stdio.h>\n#include <stddef.h>\n#include "intfa.h"\nint main(void){{{body}printf("%zu", sizeof({name}));return 0;}}\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "layout.c"), os.path.join(td, "layout")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(mirror, f[0]).offset for f in mirror._fields_] + [ctypes.sizeof(mirror)]


def _set(block, changes):
    for name, value in changes.items():
        at = block
        *path, last = name.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, value)
    return block


def _rope(r):
    r.freqs, r.pairs, r.magnitude = ADDRESS, 32, 1.0


def _cache(c):
    c.k = c.v = c.k_scale = c.v_scale = c.block_table = ADDRESS
    for t in "kv":
        setattr(c, f"{t}_stride_p", 2 * 32 * 64); setattr(c, f"{t}_stride_h", 32 * 64); setattr(c, f"{t}_stride_n", 64)
    c.ks_stride_p = c.vs_stride_p = 2
    c.ks_stride_h = c.vs_stride_h = 1
    c.num_pages, c.page_size, c.table_width, c.heads_kv, c.head_dim, c.bt_stride_b = 10, 32, 4, 2, 64, 4


def _rotary(**kw):
    p = _capi.RotaryParams()
    p.x = p.out = p.positions = ADDRESS
    for t in "xo":
        setattr(p, f"{t}_stride_b", 4 * 8 * 64); setattr(p, f"{t}_stride_h", 8 * 64); setattr(p, f"{t}_stride_n", 64)
    _rope(p.rope)
    p.batch, p.heads, p.seqlen, p.head_dim, p.dtype = 2, 4, 8, 64, _capi.INTFA_F16
    return _capi.load().intfa_rotary(ctypes.byref(_set(p, kw)), None)


def _append(**kw):
    p = _capi.PagedAppendParams()
    _cache(p.cache)
    _rope(p.rope)
    p.k_new = p.v_new = p.seqlens_k = ADDRESS
    for t in ("kn", "vn"):
        setattr(p, f"{t}_stride_b", 2 * 8 * 64); setattr(p, f"{t}_stride_h", 8 * 64); setattr(p, f"{t}_stride_n", 64)
    p.batch, p.seqlen_new, p.dtype = 2, 8, _capi.INTFA_F16
    return _capi.load().intfa_paged_append_int8(ctypes.byref(_set(p, kw)), None)


def _attn_block(**kw):
    p = _capi.PagedAttnParams()
    _cache(p.cache)
    _rope(p.rope)
    p.q = p.out = p.seqlens_k = ADDRESS
    for t in "qo":
        setattr(p, f"{t}_stride_b", 4 * 8 * 64); setattr(p, f"{t}_stride_h", 8 * 64); setattr(p, f"{t}_stride_n", 64)
    p.batch, p.heads, p.seqlen, p.dtype, p.sm_scale = 2, 4, 8, _capi.INTFA_F16, 0.125
    return _set(p, kw)


def _attn(**kw):
    return _capi.load().intfa_paged_attn_int8(ctypes.byref(_attn_block(**kw)), None)


NAN = float("nan")


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), -1), (dict(out=None), -1), (dict(rope__freqs=None), -1), (dict(batch=0), -7), (dict(heads=0), -7), (dict(seqlen=0), -3),
    (dict(head_dim=48), -2), (dict(dtype=_capi.INTFA_F32), -5), (dict(rope__pairs=12), -12), (dict(rope__pairs=40), -12), (dict(rope__pairs=0), -12),
    (dict(rope__magnitude=0.0), -12), (dict(rope__magnitude=NAN), -12), (dict(rope__magnitude=math.inf), -12), (dict(x=ADDRESS + 8), -4),
    (dict(o_stride_n=68), -4), (dict(positions=ADDRESS + 2), -4), (dict(rope__freqs=ADDRESS + 4), -4), (dict(batch=1 << 20, seqlen=1 << 20), -7),
    (dict(positions=None, position_first=(1 << 31) - 8, seqlen=9), -7)])
def test_rotary_refusals(kw, code):
    assert _rotary(**kw) == code
    assert _capi.load().intfa_error_string(code).decode() not in ("", "ok", "unknown error")


CACHE = [(dict(cache__k=None), -1), (dict(cache__v_scale=None), -1), (dict(cache__block_table=None), -1), (dict(cache__heads_kv=0), -7),
         (dict(cache__head_dim=32), -2), (dict(cache__page_size=48), -11), (dict(cache__page_size=8), -11), (dict(cache__page_size=512), -11),
         (dict(cache__num_pages=0), -11), (dict(cache__table_width=0), -11), (dict(cache__table_width=1 << 26), -7), (dict(cache__k=ADDRESS + 8), -4),
         (dict(cache__v_stride_h=8), -4), (dict(cache__k_scale=ADDRESS + 2), -4), (dict(cache__k_stride_n=48), -7), (dict(cache__v_stride_n=1 << 23), -7),
         (dict(rope__pairs=20), -12), (dict(rope__magnitude=-1.0), -12), (dict(batch=0), -7), (dict(dtype=_capi.INTFA_F32), -5), (dict(seqlens_k=None), -1),
         (dict(seqlens_k=ADDRESS + 1), -4)]


@pytest.mark.parametrize("kw,code", CACHE + [(dict(k_new=None), -1), (dict(v_new=None), -1), (dict(seqlen_new=0), -3), (dict(seqlen_new=-1), -3),
                                             (dict(v_new=ADDRESS + 2), -4), (dict(kn_stride_n=68), -4), (dict(seqlens_new=ADDRESS + 2), -4),
                                             (dict(batch=1 << 30), -7), (dict(batch=1 << 24, seqlen_new=256), -7)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code


@pytest.mark.parametrize("kw,code", CACHE + [(dict(q=None), -1), (dict(out=None), -1), (dict(seqlen=0), -3), (dict(heads=5), -7), (dict(q_stride_h=4), -4),
                                             (dict(out=ADDRESS + 4), -4), (dict(lse=ADDRESS + 2), -4), (dict(seqlens_q=ADDRESS + 1), -4),
                                             (dict(batch=1 << 16, seqlen=1 << 16), -7)])
def test_attention_refusals(kw, code):
    assert _attn(**kw) == code


def test_sizes_whose_products_pass_64_bits():
    assert _rotary(batch=1 << 30, seqlen=1 << 30, head_dim=256) == -7
    assert _rotary(batch=(1 << 31) - 1, seqlen=(1 << 31) - 1, head_dim=256) == -7
    assert _append(batch=1 << 30, seqlen_new=1 << 30, cache__page_size=16, cache__table_width=1 << 25, cache__heads_kv=1 << 9) == -7
    assert _attn(batch=1 << 20, heads=1 << 22, seqlen=1 << 22) == -7
    assert _capi.load().intfa_paged_attn_workspace_bytes(ctypes.byref(_attn_block(batch=1 << 20, heads=1 << 22, seqlen=1 << 22))) == 0


def test_null_blocks():
    lib = _capi.load()
    assert lib.intfa_rotary(None, None) == lib.intfa_paged_append_int8(None, None) == lib.intfa_paged_attn_int8(None, None) == -1
    assert lib.intfa_paged_attn_workspace_bytes(None) == 0


def test_frequencies():
    f, m = M.rotary_frequencies(64, device="cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert f.dtype == torch.float64 and m == 1.0 and torch.allclose(f, 10000.0 ** (-i / 32), rtol=1e-14)
    lin, m = M.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.allclose(lin, f / 4.0, rtol=1e-14)
    base, m = M.rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert base[0] == 1.0 and torch.allclose(base[-1], f[-1] / 4.0, rtol=1e-12) and (base[1:] < f[1:]).all()
    parts, m = M.rotary_frequencies(64, scaling="parts", factor=8.0, original_length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert abs(m - (0.1 * math.log(8.0) + 1.0)) < 1e-15
    assert torch.equal(parts[turns > 32], f[turns > 32]) and torch.allclose(parts[turns < 1], f[turns < 1] / 8.0, rtol=1e-14)
    assert ((parts <= f) & (parts >= f / 8.0 * (1 - 1e-12))).all()
    same, m = M.rotary_frequencies(64, scaling="parts", factor=1.0, original_length=4096, device="cpu")
    assert m == 1.0 and torch.allclose(same, f, rtol=1e-14)


@pytest.mark.parametrize("kw", [dict(rot_dim=24), dict(rot_dim=0), dict(rot_dim=64, base=1.0), dict(rot_dim=64, factor=0.5), dict(rot_dim=64, scaling="other"),
                                dict(rot_dim=64, scaling="parts", factor=2.0), dict(rot_dim=64, scaling="parts", original_length=9, fast_turns=1.0)])
def test_frequencies_refusals(kw):
    with pytest.raises(ValueError):
        M.rotary_frequencies(device="cpu", **kw)


def test_cpu_tensors_are_refused():
    x = torch.zeros((1, 2, 3, 64), dtype=torch.float16)
    f = torch.ones(32, dtype=torch.float64)
    i8, sc, t = torch.zeros((4, 2, 16, 64), dtype=torch.int8), torch.ones((4, 2)), torch.zeros((1, 2), dtype=torch.int32)
    n = torch.zeros((1,), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        M.rotary(x, 0, f)
    with pytest.raises(RuntimeError, match="GPU"):
        M.rotary(x.clone().requires_grad_(), 0, f)
    with pytest.raises(RuntimeError, match="GPU"):
        M.paged_kvcache_append(i8, sc, i8, sc, x, x, t, n)
    with pytest.raises(RuntimeError, match="GPU"):
        M.attention_paged_int8(x, i8, i8, sc, sc, t, n, True, 0.125)

"""The latent cache's entry points and the pages of a cache on the host: parameter blocks, sizes of workspaces, refusals ahead of any GPU call."""
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
NAN = float("nan")


@pytest.mark.parametrize("name,mirror", [("intfa_latent_cache", _capi.LatentCache), ("intfa_latent_append_params", _capi.LatentAppendParams),
                                          ("intfa_latent_attn_params", _capi.LatentAttnParams), ("intfa_latent_expanded_params", _capi.LatentExpandedParams),
                                          ("intfa_page_pool", _capi.PagePool), ("intfa_page_table", _capi.PageTable)])
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


def _strides(p, prefix, *values):
    for a, v in zip("bhn" if len(values) == 3 else "bn", values):
        setattr(p, f"{prefix}_stride_{a}", v)


def _cache(c):
    c.rows = c.scale = c.block_table = ADDRESS
    c.r_stride_p, c.r_stride_n, c.s_stride_p, c.s_stride_n, c.bt_stride_b = 32 * 576, 576, 64, 2, 4
    c.num_pages, c.page_size, c.table_width, c.latent_dim, c.rope_dim = 10, 32, 4, 512, 64


def _append_block(**kw):
    p = _capi.LatentAppendParams()
    _cache(p.cache)
    p.rope.freqs, p.rope.pairs, p.rope.magnitude = ADDRESS, 32, 1.0
    p.c_new = p.k_new = p.seqlens_k = p.norm_weight = ADDRESS
    _strides(p, "cn", 8 * 512, 512)
    _strides(p, "kn", 8 * 64, 64)
    p.norm_eps, p.batch, p.seqlen_new, p.dtype = 1e-6, 2, 8, _capi.INTFA_F16
    return _set(p, kw)


def _append(**kw):
    return _capi.load().intfa_latent_append_int8(ctypes.byref(_append_block(**kw)), None)


def _attn_block(**kw):
    p = _capi.LatentAttnParams()
    _cache(p.cache)
    p.rope.freqs, p.rope.pairs, p.rope.magnitude = ADDRESS, 32, 1.0
    p.q_latent = p.q_rope = p.out = p.seqlens_k = ADDRESS
    for t, d in (("ql", 512), ("qr", 64), ("o", 512)):
        _strides(p, t, 4 * 8 * d, 8 * d, d)
    p.batch, p.heads, p.seqlen, p.dtype, p.sm_scale = 2, 4, 8, _capi.INTFA_F16, 0.1
    return _set(p, kw)


def _attn(**kw):
    return _capi.load().intfa_latent_attn_int8(ctypes.byref(_attn_block(**kw)), None)


def _attn_bytes(**kw):
    return _capi.load().intfa_latent_attn_workspace_bytes(ctypes.byref(_attn_block(**kw)))


def _expanded(**kw):
    p = _capi.LatentExpandedParams()
    p.q_nope = p.q_rope = p.k_nope = p.k_rope = p.v = p.out = ADDRESS
    for t, d in (("qn", 128), ("qr", 64), ("kn", 128), ("v", 128), ("o", 128)):
        _strides(p, t, 4 * 8 * d, 8 * d, d)
    _strides(p, "kr", 8 * 64, 64)
    p.batch, p.heads, p.seqlen, p.seqlen_k, p.nope_dim, p.rope_dim, p.v_dim, p.dtype, p.sm_scale = 2, 4, 8, 8, 128, 64, 128, _capi.INTFA_F16, 0.1
    return _capi.load().intfa_latent_expanded(ctypes.byref(_set(p, kw)), None)


CACHE = [(dict(cache__rows=None), -1), (dict(cache__scale=None), -1), (dict(cache__block_table=None), -1), (dict(cache__latent_dim=384), -2),
         (dict(cache__rope_dim=16), -2), (dict(cache__page_size=48), -11), (dict(cache__page_size=8), -11), (dict(cache__page_size=512), -11),
         (dict(cache__num_pages=0), -11), (dict(cache__table_width=0), -11), (dict(cache__table_width=1 << 26), -7), (dict(cache__rows=ADDRESS + 8), -4),
         (dict(cache__r_stride_n=584), -4), (dict(cache__r_stride_n=560), -7), (dict(cache__r_stride_n=1 << 22), -7), (dict(cache__r_stride_p=8), -4),
         (dict(cache__scale=ADDRESS + 4), -4), (dict(cache__s_stride_n=3), -4), (dict(cache__s_stride_n=0), -7), (dict(cache__block_table=ADDRESS + 2), -4),
         (dict(rope__pairs=20), -12), (dict(rope__pairs=40), -12), (dict(rope__magnitude=NAN), -12), (dict(batch=0), -7), (dict(dtype=_capi.INTFA_F32), -5),
         (dict(seqlens_k=None), -1), (dict(seqlens_k=ADDRESS + 1), -4), (dict(rope__freqs=ADDRESS + 4), -4)]


@pytest.mark.parametrize("kw,code", CACHE + [(dict(c_new=None), -1), (dict(k_new=None), -1), (dict(seqlen_new=0), -3), (dict(seqlen_new=-1), -3), (dict(c_new=ADDRESS + 8), -4),
                                             (dict(cn_stride_n=516), -4), (dict(kn_stride_b=4), -4), (dict(norm_weight=ADDRESS + 2), -4), (dict(seqlens_new=ADDRESS + 2), -4),
                                             (dict(norm_eps=0.0), -7), (dict(norm_eps=NAN), -7), (dict(norm_eps=math.inf), -7), (dict(batch=1 << 30), -7),
                                             (dict(batch=1 << 24, seqlen_new=256), -7), (dict(batch=1 << 30, seqlen_new=1 << 30), -7)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code


@pytest.mark.parametrize("kw,code", CACHE + [(dict(q_latent=None), -1), (dict(q_rope=None), -1), (dict(out=None), -1), (dict(seqlen=0), -3), (dict(heads=0), -7),
                                             (dict(ql_stride_h=4), -4), (dict(qr_stride_n=68), -4), (dict(out=ADDRESS + 4), -4), (dict(lse=ADDRESS + 2), -4),
                                             (dict(seqlens_q=ADDRESS + 1), -4), (dict(batch=1 << 16, seqlen=1 << 16), -7), (dict(batch=1 << 20, heads=1 << 22, seqlen=1 << 22), -7)])
def test_attention_refusals(kw, code):
    assert _attn(**kw) == code
    assert _attn_bytes(**kw) == 0


def test_attention_workspace():
    """Nothing runs without one that is large enough and aligned; its size follows the work, not the pool."""
    need = _attn_bytes()
    assert need > 0 and need % 16 == 0
    assert _attn() == -6 == _attn(workspace=ADDRESS, workspace_bytes=need - 1) == _attn(workspace=ADDRESS + 4, workspace_bytes=need)
    assert _attn_bytes(cache__num_pages=1 << 20) == need
    assert _attn_bytes(batch=64, heads=128, seqlen=1, cache__table_width=1 << 14) <= 256 * 2 * 64 * (512 * 4 + 8) + 256 * 16


@pytest.mark.parametrize("kw,code", [
    (dict(q_nope=None), -1), (dict(q_rope=None), -1), (dict(k_nope=None), -1), (dict(k_rope=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(batch=0), -7),
    (dict(heads=-1), -7), (dict(seqlen=0), -3), (dict(seqlen_k=-1), -3), (dict(nope_dim=64), -2), (dict(rope_dim=32), -2), (dict(v_dim=192), -2),
    (dict(nope_dim=64, rope_dim=32, v_dim=128), -2), (dict(dtype=_capi.INTFA_F32), -5), (dict(q_nope=ADDRESS + 2), -4), (dict(kr_stride_n=68), -4), (dict(o_stride_h=4), -4),
    (dict(lse=ADDRESS + 1), -4), (dict(seqlens_q=ADDRESS + 2), -4), (dict(seqlens_k=ADDRESS + 2), -4), (dict(kn_stride_n=120), -7), (dict(v_stride_n=1 << 28), -7),
    (dict(seqlen_k=1 << 25), -7), (dict(seqlen=(1 << 30) + 1), -7), (dict(batch=1 << 20, heads=1 << 20), -7), (dict(batch=1 << 15, heads=1 << 10), -7)])
def test_expanded_refusals(kw, code):
    assert _expanded(**kw) == code


def _table(**kw):
    t = _capi.PageTable()
    t.refs = t.block_table = t.seqlens_k = ADDRESS
    t.bt_stride_b, t.num_pages, t.page_size, t.table_width, t.batch = 4, 10, 32, 4, 6
    return _set(t, kw)


def _pools(n=2, **kw):
    pools = (_capi.PagePool * max(1, n))()
    for p in pools:
        p.data, p.page_stride, p.page_bytes = ADDRESS, 4096, 4096
    _set(pools[-1], kw)
    return pools, n


TABLE = [(dict(refs=None), -1), (dict(block_table=None), -1), (dict(num_pages=0), -11), (dict(num_pages=1 << 30), -11), (dict(table_width=0), -11), (dict(table_width=1 << 30), -11),
         (dict(batch=0), -7), (dict(refs=ADDRESS + 2), -4), (dict(block_table=ADDRESS + 1), -4), (dict(bt_stride_b=3), -7), (dict(bt_stride_b=0), -7), (dict(bt_stride_b=-2), -7)]
LENS = [(dict(seqlens_k=None), -1), (dict(seqlens_k=ADDRESS + 2), -4)]
PAGE = [(dict(page_size=8), -11), (dict(page_size=48), -11), (dict(page_size=512), -11)]
POOLS = [(dict(data=None), -1), (dict(page_bytes=0), -13), (dict(page_bytes=-4), -13), (dict(page_bytes=(1 << 40) + 1), -13), (dict(page_stride=0), -13), (dict(page_stride=4095), -13),
         (dict(page_stride=-4095), -13)]


@pytest.mark.parametrize("kw,code", TABLE + LENS)
def test_fork_refusals(kw, code):
    assert _capi.load().intfa_pages_fork(ctypes.byref(_table(**kw)), ADDRESS, ADDRESS, 3, None) == code


@pytest.mark.parametrize("parents,children,n,code", [(None, ADDRESS, 3, -1), (ADDRESS, None, 3, -1), (ADDRESS, ADDRESS, 0, -7), (ADDRESS, ADDRESS, 4097, -7), (ADDRESS + 2, ADDRESS, 3, -4)])
def test_fork_refusals_of_its_own(parents, children, n, code):
    assert _capi.load().intfa_pages_fork(ctypes.byref(_table()), parents, children, n, None) == code


@pytest.mark.parametrize("kw,code", TABLE + LENS + PAGE)
def test_free_refusals(kw, code):
    assert _capi.load().intfa_pages_free(ctypes.byref(_table(**kw)), ADDRESS, None, 3, None) == code


def test_free_refusals_of_its_own():
    free, t = _capi.load().intfa_pages_free, ctypes.byref(_table())
    assert free(t, None, None, 3, None) == -1 and free(t, ADDRESS, None, 0, None) == free(t, ADDRESS, None, 65536, None) == -7
    assert free(t, ADDRESS + 1, None, 3, None) == free(t, ADDRESS, ADDRESS + 2, 3, None) == -4


@pytest.mark.parametrize("kw,code", TABLE + LENS + PAGE)
def test_reserve_refusals_of_tables(kw, code):
    lib = _capi.load()
    assert lib.intfa_pages_reserve(ctypes.byref(_table(**kw)), *_pools(), ADDRESS, 0, ADDRESS, ADDRESS, 1 << 20, None) == code
    assert lib.intfa_pages_reserve_workspace_bytes(ctypes.byref(_table(**kw))) == 0


@pytest.mark.parametrize("kw,code", TABLE)
def test_compact_refusals_of_tables(kw, code):
    lib = _capi.load()
    assert lib.intfa_pages_compact(ctypes.byref(_table(**kw)), *_pools(), ADDRESS, ADDRESS, 1 << 20, None) == code
    assert lib.intfa_pages_compact_workspace_bytes(ctypes.byref(_table(**kw))) == 0


@pytest.mark.parametrize("kw,code", POOLS)
def test_refusals_of_pools(kw, code):
    lib, t = _capi.load(), ctypes.byref(_table())
    assert lib.intfa_pages_copy(*_pools(2, **kw), 10, ADDRESS, ADDRESS, 3, None) == code
    assert lib.intfa_pages_reserve(t, *_pools(2, **kw), ADDRESS, 0, ADDRESS, ADDRESS, 1 << 20, None) == code
    assert lib.intfa_pages_compact(t, *_pools(2, **kw), ADDRESS, ADDRESS, 1 << 20, None) == code


def test_refusals_of_their_own():
    lib, t = _capi.load(), ctypes.byref(_table())
    copy = lambda *a: lib.intfa_pages_copy(*a, None)  # noqa: E731
    assert copy(*_pools(0), 10, ADDRESS, ADDRESS, 3) == copy(None, 1, 10, ADDRESS, ADDRESS, 3) == copy(_pools()[0], 4097, 10, ADDRESS, ADDRESS, 3) == -13
    assert copy(*_pools(), 10, None, ADDRESS, 3) == -1 and copy(*_pools(), 0, ADDRESS, ADDRESS, 3) == -11 and copy(*_pools(), 10, ADDRESS, ADDRESS, 0) == -7
    assert copy(*_pools(), 10, ADDRESS, ADDRESS + 2, 3) == -4
    need = lib.intfa_pages_reserve_workspace_bytes(t)
    reserve = lambda fresh, granted, ws, n, table=t: lib.intfa_pages_reserve(table, *_pools(), fresh, 0, granted, ws, n, None)  # noqa: E731
    assert reserve(ADDRESS, None, ADDRESS, need) == -1 and reserve(ADDRESS, ADDRESS, None, need) == reserve(ADDRESS, ADDRESS, ADDRESS, need - 1) == -6
    assert reserve(ADDRESS, ADDRESS, ADDRESS + 8, need) == -6 and reserve(ADDRESS + 2, ADDRESS, ADDRESS, need) == reserve(ADDRESS, ADDRESS + 1, ADDRESS, need) == -4
    assert reserve(ADDRESS, ADDRESS, ADDRESS, 1 << 30, ctypes.byref(_table(batch=8193))) == -7
    need = lib.intfa_pages_compact_workspace_bytes(t)
    compact = lambda index, ws, n: lib.intfa_pages_compact(t, *_pools(), index, ws, n, None)  # noqa: E731
    assert compact(None, ADDRESS, need) == -1 and compact(ADDRESS, None, need) == compact(ADDRESS, ADDRESS, need - 1) == compact(ADDRESS, ADDRESS + 4, need) == -6
    assert compact(ADDRESS + 2, ADDRESS, need) == -4
    assert lib.intfa_error_string(-13).decode() not in ("", "ok", "unknown error")


def test_null_blocks():
    lib = _capi.load()
    assert lib.intfa_latent_append_int8(None, None) == lib.intfa_latent_attn_int8(None, None) == lib.intfa_latent_expanded(None, None) == -1
    assert lib.intfa_pages_fork(None, ADDRESS, ADDRESS, 1, None) == lib.intfa_pages_free(None, ADDRESS, None, 1, None) == -1
    assert lib.intfa_latent_attn_workspace_bytes(None) == lib.intfa_pages_reserve_workspace_bytes(None) == lib.intfa_pages_compact_workspace_bytes(None) == 0


def test_cpu_tensors_are_refused():
    x, i = torch.zeros((1, 1, 1, 128), dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    cache, scale, table = torch.zeros((2, 16, 160), dtype=torch.int8), torch.zeros((2, 16, 2)), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: M.paged_latent_append(cache, scale, x[0], x[0, ..., :32], table, i), lambda: M.attention_paged_latent_int8(x, x[..., :32], cache, scale, table, i, True, 0.1),
                 lambda: M.attention_latent(x, x[..., :64], x, x[..., :64], x, True, 0.1), lambda: M.paged_copy([cache], i, i), lambda: M.paged_fork(i, table, i, i, i),
                 lambda: M.paged_free(i, table, i, i, 16), lambda: M.paged_reserve([cache], i, table, i, 1, 16), lambda: M.paged_compact([cache], i, table)):
        with pytest.raises(RuntimeError):
            call()

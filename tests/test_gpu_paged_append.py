"""The append to a paged int8 cache: values bit for bit by the formula's fp32 steps, rotated keys within half a step of the page's scale."""
import pytest
import torch

import int_flashattention_amd as M
from paged_reference import append, make_cache, make_table, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run_both(case, k, v, lens, fresh=None, extra=0, freqs=None, magnitude=1.0, interleaved=False, seed=1, table=None, spread=1.0):
    Z, Hkv, N, d = k.shape
    page = case
    g = torch.Generator().manual_seed(seed)
    ends = [max(0, n) + N for n in lens]
    pages = sum((n + page - 1) // page for n in ends) + 3
    cache, kv, sc = make_cache(g, pages, Hkv, page, d, spread)
    if table is None:
        table = make_table(g, ends, page, pages, extra)
    kv_d, sc_d = kv.to(DEV), sc.to(DEV)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    fresh_t = None if fresh is None else torch.tensor(fresh, dtype=torch.int32)
    M.paged_kvcache_append(kv_d[:, 0], sc_d[:, 0], kv_d[:, 1], sc_d[:, 1], k.to(DEV), v.to(DEV), table.to(DEV), lens_t.to(DEV),
                           freqs, interleaved=interleaved, magnitude=magnitude, seqlens_new=None if fresh is None else fresh_t.to(DEV))
    torch.cuda.synchronize()
    before_k, before_s = cache["k"].clone(), cache["ks"].clone()
    counts = [N] * Z if fresh is None else fresh
    append(cache["v"], cache["vs"], v.float(), table, lens, counts)
    assert torch.equal(kv_d[:, 1].cpu(), cache["v"]) and torch.equal(sc_d[:, 1].cpu(), cache["vs"])
    if freqs is None:
        append(cache["k"], cache["ks"], k.float(), table, lens, counts)
        assert torch.equal(kv_d[:, 0].cpu(), cache["k"]) and torch.equal(sc_d[:, 0].cpu(), cache["ks"])
        return kv_d, sc_d
    # rotated keys: the scale to fp32's rounding of the rotation, each value within half a step, the rest as by the formula
    pos = lens_t.clamp(min=0)[:, None] + torch.arange(N)
    turned = rotate(k, pos, freqs.cpu(), magnitude, interleaved)
    got_k, got_s = kv_d[:, 0].cpu(), sc_d[:, 0].cpu()
    want_k, want_s = before_k.clone(), before_s.clone()
    append(want_k, want_s, turned.float(), table, lens, counts)
    assert torch.allclose(got_s, want_s, rtol=3e-6, atol=0.0)
    # a value next to a border may fall either way: one step, and (a border's surroundings being 2e-5 of a step) in few places
    off = (got_k.int() - want_k.int()).abs()
    assert off.max() <= 1 and off.float().mean() <= 1e-3
    for z in range(Z):
        for i in range(min(counts[z], N)):
            at = max(0, lens[z]) + i
            p = int(table[z, at // page]) if at // page < table.shape[1] else -1
            if 0 <= p < pages:
                value = got_k[p, :, at % page].double() * got_s[p].double()[:, None]
                assert ((value - turned[z, :, i]).abs() <= got_s[p].double()[:, None] * (0.5 + 1e-3)).all()
    return kv_d, sc_d


@pytest.mark.parametrize("Z,Hkv,N,d,page,lens,dtype", [
    (1, 1, 1, 64, 16, [0], torch.float16),
    (1, 2, 1, 128, 64, [63], torch.bfloat16),                # the last row of a page
    (2, 1, 1, 128, 64, [64, 1], torch.float16),              # the first of the next one; the second of a page
    (3, 2, 7, 64, 16, [0, 13, 30], torch.bfloat16),          # within, over one border, over two
    (2, 3, 130, 256, 32, [5, 31], torch.float16),
    (2, 2, 300, 128, 128, [0, 100], torch.bfloat16),
    (1, 2, 513, 64, 256, [255], torch.float16),
    (4, 2, 64, 128, 64, [0, 64, 1, 63], torch.float16),
])
@pytest.mark.parametrize("rot", [0, 1, 2])
def test_formula(Z, Hkv, N, d, page, lens, dtype, rot):
    g = torch.Generator().manual_seed(N + page + rot)
    k = (torch.randn((Z, Hkv, N, d), generator=g) * torch.exp(torch.randn((Z, Hkv, N, 1), generator=g))).to(dtype)
    v = (torch.randn((Z, Hkv, N, d), generator=g) * torch.exp(torch.randn((Z, Hkv, N, 1), generator=g))).to(dtype)
    freqs = None if rot == 0 else M.rotary_frequencies(d if rot == 1 else d // 2, device=DEV)[0]
    run_both(page, k, v, lens, freqs=freqs, magnitude=1.25 if rot == 2 else 1.0, interleaved=rot == 2, extra=2)


def test_counts_negative_lengths_and_rows_without_a_place():
    """Sequences with fewer new rows (none, more than there are), a negative length, tables that end early or name no page."""
    g = torch.Generator().manual_seed(31)
    k, v = torch.randn((6, 2, 40, 64), generator=g).half(), torch.randn((6, 2, 40, 64), generator=g).half()
    run_both(16, k, v, [0, 10, 20, -5, 3, 7], fresh=[0, 1, 40, 99, -2, 17])
    table = torch.arange(18, dtype=torch.int32).reshape(6, 3)
    table[1, 1], table[2, 0], table[3, 2] = -1, 18 + 2 ** 20, -(2 ** 31)
    run_both(16, k, v, [0, 10, 15, 40, 48, 1000], table=table)              # the fifth table is full, the sixth sequence past its end


def test_rows_behind_the_new_ones_stay():
    g = torch.Generator().manual_seed(32)
    k, v = torch.randn((1, 1, 3, 64), generator=g).half(), torch.randn((1, 1, 3, 64), generator=g).half()
    kv = torch.full((1, 2, 1, 64, 64), 99, dtype=torch.int8, device=DEV)
    sc = torch.full((1, 2, 1), 1e-4, device=DEV)
    M.paged_kvcache_append(kv[:, 0], sc[:, 0], kv[:, 1], sc[:, 1], k.to(DEV), v.to(DEV), torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                           torch.tensor([20], dtype=torch.int32, device=DEV))
    assert (kv[..., 23:, :] == 99).all() and not (kv[..., :20, :] == 99).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_not_finite_or_tiny(dtype):
    g = torch.Generator().manual_seed(33)
    k, v = torch.randn((1, 2, 20, 64), generator=g).to(dtype), torch.randn((1, 2, 20, 64), generator=g).to(dtype)
    v[0, 0, 3, 5], v[0, 0, 4, 6], v[0, 1, 2, 1] = float("nan"), float("inf"), float("-inf")
    k[0, 1, 16:] = 0.0                                       # a page of zeros: the least scale
    v[0, 1, 16:] = torch.finfo(dtype).tiny * torch.randn((4, 64), generator=g).to(dtype)
    k[0, 0, 16:] = torch.finfo(dtype).max                    # the largest ones
    kv, sc = run_both(16, k, v, [0])
    assert sc.isfinite().all() and (sc > 0).all()


def test_a_page_that_is_refilled_takes_its_scale_from_its_new_rows():
    k = torch.full((1, 1, 16, 64), 0.5).half()
    kv, sc = torch.zeros((1, 2, 1, 16, 64), dtype=torch.int8, device=DEV), torch.full((1, 2, 1), 1e6, device=DEV)
    args = (kv[:, 0], sc[:, 0], kv[:, 1], sc[:, 1], k.to(DEV), k.to(DEV), torch.zeros((1, 1), dtype=torch.int32, device=DEV))
    M.paged_kvcache_append(*args, torch.zeros((1,), dtype=torch.int32, device=DEV))
    assert (kv == 127).all() and torch.allclose(sc.cpu(), torch.tensor(0.5 / 127))


def test_strided_new_rows():
    g = torch.Generator().manual_seed(34)
    qkv = torch.randn((2, 21, 3, 4, 128), generator=g).bfloat16()           # [Z, N, (q, k, v), H, d]
    run_both(32, qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2), [11, 0])


def test_several_heads_a_workgroup():
    """Enough pages that a workgroup takes several heads of one, and a number of heads that its share does not divide."""
    g = torch.Generator().manual_seed(35)
    k, v = (torch.randn((4, 11, 1030, 64), generator=g).half() for _ in range(2))
    v[1, 7, 500, 3] = float("inf")
    run_both(16, k, v, [0, 9, 16, 40], freqs=M.rotary_frequencies(64, device=DEV)[0])


def test_pages_whose_heads_lie_side_by_side():
    g = torch.Generator().manual_seed(36)
    k, v = (torch.randn((2, 3, 50, 128), generator=g).bfloat16().to(DEV) for _ in range(2))
    table, lens = torch.arange(8, dtype=torch.int32, device=DEV).reshape(2, 4), torch.tensor([5, 30], dtype=torch.int32, device=DEV)
    side = torch.zeros((8, 32, 2, 3, 128), dtype=torch.int8, device=DEV)            # [page, row, (k, v), head, d]
    plain = torch.zeros((8, 2, 3, 32, 128), dtype=torch.int8, device=DEV)
    s1, s2 = (torch.full((8, 2, 3), 0.01, device=DEV) for _ in range(2))
    M.paged_kvcache_append(side[:, :, 0].transpose(1, 2), s1[:, 0], side[:, :, 1].transpose(1, 2), s1[:, 1], k, v, table, lens)
    M.paged_kvcache_append(plain[:, 0], s2[:, 0], plain[:, 1], s2[:, 1], k, v, table, lens)
    assert torch.equal(side.permute(0, 2, 3, 1, 4), plain) and torch.equal(s1, s2) and plain.any()


@pytest.mark.parametrize("rot", [False, True])
@pytest.mark.parametrize("Z,Hkv,N,d,page,lens,dtype", [
    (4, 5, 1030, 64, 32, [0, 9, 31, 40], torch.float16),                # two heads a workgroup, then four and eight: the last one's share is smaller
    (4, 11, 1030, 64, 32, [0, 9, 31, 40], torch.bfloat16),
    (4, 17, 1030, 64, 32, [3, 0, 64, 100], torch.float16),
    (2, 7, 4500, 256, 64, [0, 50], torch.bfloat16),                     # two units a thread
    (2, 2, 520, 256, 256, [0, 100], torch.float16),                     # pages of more units than the threads hold
    (2, 3, 300, 256, 128, [77, 0], torch.bfloat16),
    (2, 1, 700, 128, 256, [255, 3], torch.float16),
])
def test_large_launches(Z, Hkv, N, d, page, lens, dtype, rot):
    """Workgroups of several heads, and of pages that the threads read again; values that are not numbers in a middle head and in the last rows of a page."""
    g = torch.Generator().manual_seed(N + Hkv)
    k, v = (torch.randn((Z, Hkv, N, d), generator=g).to(dtype) for _ in range(2))
    last = page - lens[0] % page - 1                                    # the first sequence's last row of its first page
    for x in (v,) if rot else (k, v):
        x[0, Hkv // 2, last, 5], x[0, Hkv // 2, last - 1, d - 1] = float("inf"), float("nan")
        x[1, Hkv - 1, N - 1, 0] = float("-inf")
    run_both(page, k, v, lens, freqs=M.rotary_frequencies(d, device=DEV)[0] if rot else None)


@pytest.mark.parametrize("Z,Hkv,N,d,page", [(4, 11, 1030, 64, 32), (1, 2, 300, 256, 256), (1, 2, 20, 64, 16)])
def test_rotated_keys_that_are_not_finite(Z, Hkv, N, d, page):
    """A pair with a NaN becomes zeros, one with an infinity +-127 twice, and the others keep the scale of the finite ones."""
    g = torch.Generator().manual_seed(37)
    k = torch.randn((Z, Hkv, N, d), generator=g).half()
    at = min(page, N) - 1
    k[0, Hkv // 2, at, 5], k[0, Hkv // 2, at - 2, 9] = float("nan"), float("inf")
    freqs = M.rotary_frequencies(d, device=DEV)[0]
    pages = Z * -(-N // page)
    table = torch.arange(pages, dtype=torch.int32).reshape(Z, -1)
    kv, sc = torch.zeros((pages, 2, Hkv, page, d), dtype=torch.int8), torch.zeros((pages, 2, Hkv))
    kv_d, sc_d = kv.to(DEV), sc.to(DEV)
    M.paged_kvcache_append(kv_d[:, 0], sc_d[:, 0], kv_d[:, 1], sc_d[:, 1], k.to(DEV), k.to(DEV), table.to(DEV), torch.zeros((Z,), dtype=torch.int32, device=DEV), freqs)
    turned = rotate(k, torch.arange(N).expand(Z, N), freqs.cpu())
    append(kv[:, 0], sc[:, 0], turned.float(), table, [0] * Z, [N] * Z)
    got, scale = kv_d[:, 0].cpu(), sc_d[:, 0].cpu()
    assert scale.isfinite().all() and torch.allclose(scale, sc[:, 0], rtol=3e-6, atol=0.0)
    off = (got.int() - kv[:, 0].int()).abs()
    assert off.max() <= 1 and off.float().mean() <= 1e-3
    first = got[0, Hkv // 2]
    assert (first[at, [5, 5 + d // 2]] == 0).all() and (first[at - 2, [9, 9 + d // 2]].abs() == 127).all()

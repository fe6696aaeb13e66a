"""Attention over a paged int8 cache against its formula in float64, within a bound that counts the kernel's roundings."""
import pytest
import torch

import int_flashattention_amd as M
from paged_reference import attend, bound, make_cache, make_table

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(q, cache, kv, sc, table, lens, causal, sm=None, fresh=None, freqs=None, **turn):
    """Runs the call, compares output and lse; returns the output."""
    d = q.shape[-1]
    sm = d ** -0.5 if sm is None else sm
    kv_d, sc_d = kv.to(DEV), sc.to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    fresh_d = None if fresh is None else torch.tensor(fresh, dtype=torch.int32, device=DEV)
    o, lse = M.attention_paged_int8(q.to(DEV), kv_d[:, 0], kv_d[:, 1], sc_d[:, 0], sc_d[:, 1], table.to(DEV), lens_d, causal, sm,
                                    freqs=freqs, seqlens_q=fresh_d, return_lse=True, **turn)
    torch.cuda.synchronize()
    rope = None if freqs is None else dict(freqs=freqs.cpu(), **turn)
    want, want_lse, mean_v, size = attend(q, cache, table, lens, causal, sm, fresh, rope)
    o, lse = o.cpu(), lse.cpu()
    assert o.isfinite().all()
    # rotated bf16 queries of more than 64 rows a K/V head are held to 11 bits
    step = 2.0 ** -12 if freqs is not None and q.dtype == torch.bfloat16 and q.shape[1] // kv.shape[2] * q.shape[2] > 64 else 0.0
    far = (o.double() - want).abs() - bound(want, mean_v, size, q.dtype, step)
    assert (far <= 0).all(), f"{far.max().item():.3g} past the bound"
    empty = want_lse == -float("inf")
    assert torch.equal(lse == -float("inf"), empty) and (o[empty] == 0).all()
    # lse: the scores' error and the sum's, in base 2
    assert ((lse.double() - want_lse)[~empty].abs() <= (2.0 ** -12 + 2.0 * (2.0 ** -19 + step) * size[..., 0] + 2.0 ** -23 * want_lse.abs())[~empty]).all()
    return o


def problem(seed, Z, H, Hkv, N, d, page, lens, dtype, spread=0.5, extra=1):
    g = torch.Generator().manual_seed(seed)
    pages = sum((n + page - 1) // page for n in lens) + 2
    cache, kv, sc = make_cache(g, pages, Hkv, page, d, spread)
    table = make_table(g, lens, page, pages, extra)
    q = (1.5 * torch.randn((Z, H, N, d), generator=g)).to(dtype)
    return q, cache, kv, sc, table


@pytest.mark.parametrize("H,Hkv,N,d,page,lens,causal,dtype", [
    (1, 1, 1, 64, 16, [1], False, torch.float16),
    (4, 4, 1, 128, 16, [0, 1, 15, 16, 17], False, torch.float16),            # an empty sequence among others
    (8, 2, 1, 128, 64, [63, 64, 65, 300], False, torch.bfloat16),
    (8, 1, 1, 256, 32, [31, 33, 500, 257], False, torch.float16),
    (20, 4, 1, 64, 128, [1000, 3, 129], False, torch.bfloat16),              # five query heads a K/V head
    (6, 2, 5, 64, 32, [5, 100, 33], True, torch.float16),                    # drafts
    (4, 4, 3, 128, 64, [2, 1, 0, 130], True, torch.bfloat16),                # more new tokens than keys: rows that see none
    (2, 2, 17, 256, 16, [17, 400], True, torch.float16),
    (3, 1, 33, 128, 256, [33, 700], True, torch.bfloat16),
    (8, 2, 70, 64, 64, [70, 71, 200], True, torch.float16),
    (2, 1, 130, 128, 32, [130, 515], True, torch.float16),
    (4, 2, 100, 128, 64, [300, 1], False, torch.bfloat16),
    (2, 2, 300, 64, 16, [300, 450], True, torch.bfloat16),
    (2, 1, 140, 256, 64, [140, 333], True, torch.bfloat16),
    (32, 8, 1, 128, 64, [4000, 2777], False, torch.float16),
    (1, 1, 600, 128, 128, [600], True, torch.float16),
])
def test_formula(H, Hkv, N, d, page, lens, causal, dtype):
    q, cache, kv, sc, table = problem(N * 7 + d, len(lens), H, Hkv, N, d, page, lens, dtype)
    run(q, cache, kv, sc, table, lens, causal)


@pytest.mark.parametrize("N,rot,interleaved,dtype", [(1, 128, False, torch.float16), (1, 64, True, torch.bfloat16), (6, 32, True, torch.float16),
                                                      (40, 128, False, torch.float16), (150, 64, False, torch.float16), (200, 128, True, torch.bfloat16)])
def test_queries_are_rotated_on_the_way(N, rot, interleaved, dtype):
    """As by the formula without rounding the turned queries to 16 bits, whatever the number of rows."""
    lens = [N, 700, N + 64]
    q, cache, kv, sc, table = problem(N + rot, 3, 8, 2, N, 128, 64, lens, dtype)
    freqs, magnitude = M.rotary_frequencies(rot, device=DEV, scaling="parts", factor=8.0, original_length=256)
    run(q, cache, kv, sc, table, lens, True, freqs=freqs, magnitude=magnitude, interleaved=interleaved)


@pytest.mark.parametrize("N", [32, 33, 64, 65])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rotated_queries_where_the_kernels_take_turns(N, d, dtype):
    """64, 66, 128 and 130 rows a K/V head."""
    lens = [N + 70, N]
    q, cache, kv, sc, table = problem(92 + N, 2, 4, 2, N, d, 32, lens, dtype)
    freqs, _ = M.rotary_frequencies(d, device=DEV)
    run(q, cache, kv, sc, table, lens, True, freqs=freqs)


@pytest.mark.parametrize("N,fresh,lens", [(4, [4, 0, 1, 9, -3], [100, 50, 1, 70, 20]), (200, [200, 7, 0, 129], [260, 7, 100, 129]),
                                          (80, [3, 80, 1], [500, 80, 3])])
def test_new_tokens_of_each_sequence(N, fresh, lens):
    q, cache, kv, sc, table = problem(N, len(lens), 4, 2, N, 64, 32, lens, torch.float16)
    freqs, _ = M.rotary_frequencies(64, device=DEV)
    run(q, cache, kv, sc, table, lens, True, fresh=fresh, freqs=freqs)
    run(q, cache, kv, sc, table, lens, False, fresh=fresh)


@pytest.mark.parametrize("N,causal", [(1, False), (5, True), (150, True)])
def test_pages_that_the_table_does_not_name_are_hidden(N, causal):
    lens = [400, 200, 64]
    q, cache, kv, sc, table = problem(50 + N, 3, 4, 2, N, 128, 32, lens, torch.float16)
    table[0, 3], table[0, 12], table[1, 0], table[2, :2] = -1, 2 ** 30, -(2 ** 31), -1        # the third sequence has no page left
    run(q, cache, kv, sc, table, lens, causal)


@pytest.mark.parametrize("N", [1, 7, 160])
def test_what_no_row_sees_has_no_part(N):
    """Lengths past the table are cut; pages of other sequences and columns behind the last key may hold anything, scales that are not numbers too."""
    lens = [130, 40]
    q, cache, kv, sc, table = problem(60 + N, 2, 4, 4, N, 64, 16, lens, torch.bfloat16, extra=3)
    used = torch.zeros(kv.shape[0], dtype=torch.bool)
    for z, n in enumerate(lens):
        used[table[z, :(n + 15) // 16].long()] = True
    sc[~used] = float("nan")
    first = int(torch.nonzero(~used)[0])
    sc[first] = float("inf")
    table[0, 9:], table[1, 3:] = first, int(torch.nonzero(~used)[1])
    run(q, cache, kv, sc, table, lens, True)
    full = [10 ** 6, -4]
    table = table[:, :9].clone()
    table[1] = table[0]
    run(q, cache, kv, sc, table, full, False)


@pytest.mark.parametrize("spread,N", [(4.0, 1), (8.0, 1), (4.0, 140), (8.0, 140)])
def test_pages_of_very_different_scales(spread, N):
    """V's scales over e^-8 .. e^8 (seven decades) in the same rows; K's over e^-1 .. e^1, so that the softmax keeps many keys."""
    lens = [500, 300 + N]
    q, cache, kv, sc, table = problem(70, 2, 4, 2, N, 128, 16, lens, torch.float16, spread=1.0)
    sc[:, 1] = torch.exp(spread * (2.0 * torch.rand(sc[:, 1].shape, generator=torch.Generator().manual_seed(71)) - 1.0)) / 31.75 / 127
    run(q, cache, kv, sc, table, lens, True)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e4])
def test_queries_of_any_size(scale):
    """Rows of zeros, rows below fp16's range (bf16 has them) and large ones, whose softmax is one key."""
    q, cache, kv, sc, table = problem(80, 1, 4, 2, 3, 64, 32, [90], torch.bfloat16)
    run((q.float() * scale).bfloat16(), cache, kv, sc, table, [90], True)


def test_a_query_that_is_not_a_number_stays_in_its_row():
    q, cache, kv, sc, table = problem(81, 1, 4, 2, 3, 64, 32, [90], torch.float16)
    q[0, 1, 1, 7] = float("nan")
    kv_d, sc_d = kv.to(DEV), sc.to(DEV)
    o = M.attention_paged_int8(q.to(DEV), kv_d[:, 0], kv_d[:, 1], sc_d[:, 0], sc_d[:, 1], table.to(DEV), torch.tensor([90], dtype=torch.int32, device=DEV),
                               False, 0.125).cpu()
    assert o[0, 1, 1].isnan().all()
    o[0, 1, 1] = 0.0
    assert o.isfinite().all()


@pytest.mark.parametrize("N,fresh,lens", [(4, [2, 0, 4], [100, 60, 9]), (4, [3, 1], [20000, 9000]), (90, [33, 90], [400, 90])])
def test_what_pads_a_batch_may_be_anything(N, fresh, lens):
    """Rows past a sequence's new tokens are zeros even where the padding is no number, in sequences of one piece and of many."""
    q, cache, kv, sc, table = problem(84 + N, len(lens), 4, 2, N, 64, 64, lens, torch.bfloat16)
    freqs, _ = M.rotary_frequencies(64, device=DEV)
    for z, m in enumerate(fresh):
        q[z, :, m:] = float("nan")
    run(q, cache, kv, sc, table, lens, True, fresh=fresh, freqs=freqs)


@pytest.mark.parametrize("N,n", [(1, 90), (3, 20000), (70, 300)])
def test_a_row_that_is_not_a_number_has_no_lse(N, n):
    q, cache, kv, sc, table = problem(85, 1, 4, 2, N, 128, 32, [n], torch.float16)
    q[0, 2, N // 2, 9] = float("nan")
    kv_d, sc_d = kv.to(DEV), sc.to(DEV)
    o, lse = M.attention_paged_int8(q.to(DEV), kv_d[:, 0], kv_d[:, 1], sc_d[:, 0], sc_d[:, 1], table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
                                    True, 0.125, return_lse=True)
    bad = torch.zeros((4, N), dtype=torch.bool, device=DEV)
    bad[2, N // 2] = True
    assert o[0][bad].isnan().all() and o[0][~bad].isfinite().all()
    assert lse[0][bad].isnan().all() and lse[0][~bad].isfinite().all()


@pytest.mark.parametrize("N", [1, 9, 100])
def test_a_negative_scale_of_scores(N):
    """The sign goes to the queries, which are held to as many bits either way: the same as the positive scale with the queries' signs changed."""
    lens = [N + 30, 500]
    q, cache, kv, sc, table = problem(86, 2, 8, 2, N, 128, 64, lens, torch.float16)
    assert torch.equal(run(-q, cache, kv, sc, table, lens, True, sm=0.1), run(q, cache, kv, sc, table, lens, True, sm=-0.1))
    run(q, cache, kv, sc, table, lens, True, sm=0.0)


@pytest.mark.parametrize("N", [2, 100])
def test_scales_of_values_near_nothing(N):
    """Values of 2^-130 and less: below fp16's smallest, and no scale's reciprocal is formed that would not be a number."""
    lens = [N + 100]
    q, cache, kv, sc, table = problem(87, 1, 4, 2, N, 64, 16, lens, torch.float16)
    sc[:, 1] = 2.0 ** -135
    run(q, cache, kv, sc, table, lens, True)


@pytest.mark.parametrize("H,Hkv,N,d", [(96, 1, 1, 128), (71, 1, 1, 64), (130, 2, 1, 256)])
def test_many_query_heads_of_one_key_head(H, Hkv, N, d):
    lens = [1, 777, 64]
    q, cache, kv, sc, table = problem(88 + d, 3, H, Hkv, N, d, 32, lens, torch.bfloat16)
    freqs, _ = M.rotary_frequencies(64, device=DEV)
    run(q, cache, kv, sc, table, lens, False, freqs=freqs)


def test_wide_tables_of_many_sequences():
    """9600 items over tables of 320000 keys: more units of work than are numbered, so they are larger ones."""
    Z, H, d, page, columns = 600, 16, 64, 16, 20000
    lens = [1 + 7 * z % 50 for z in range(Z)]
    q, cache, kv, sc, narrow = problem(89, Z, H, H, 1, d, page, lens, torch.float16)
    table = torch.full((Z, columns), -1, dtype=torch.int32)
    table[:, :narrow.shape[1]] = narrow
    run(q, cache, kv, sc, table, lens, False)


def test_strides():
    """Queries as [Z, N, H, d], pages as [page, head, (k, v), row]: any strides with a contiguous d."""
    lens = [77, 200]
    q, cache, kv, sc, table = problem(82, 2, 8, 2, 2, 128, 32, lens, torch.bfloat16)
    want = run(q, cache, kv, sc, table, lens, True)
    other = kv.transpose(1, 2).contiguous().to(DEV)
    scales = sc.permute(2, 1, 0).contiguous().to(DEV)
    o = M.attention_paged_int8(q.transpose(1, 2).contiguous().to(DEV).transpose(1, 2), other[:, :, 0], other[:, :, 1], scales[:, 0].T, scales[:, 1].T,
                               table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), True, 128 ** -0.5)
    assert torch.equal(o.cpu(), want)


@pytest.mark.parametrize("N", [1, 30, 100])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 128), (256, 16), (256, 32), (256, 256), (128, 16)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rotated_queries_of_all_head_dims(N, d, page, dtype):
    """Both kernels of each head_dim, pages smaller and larger than the keys that they take at a time."""
    lens = [N + 333, N, 1]
    q, cache, kv, sc, table = problem(90 + d + page, 3, 4, 2, N, d, page, lens, dtype)
    freqs, magnitude = M.rotary_frequencies(d, device=DEV, scaling="base", factor=2.0)
    run(q, cache, kv, sc, table, lens, True, freqs=freqs, magnitude=magnitude, interleaved=page == 16)


@pytest.mark.parametrize("N,d", [(1, 64), (1, 128), (20, 256), (150, 64), (150, 128), (150, 256)])
def test_pages_whose_heads_lie_side_by_side(N, d):
    """Pages as [page, row, head, d]: a row's next one is all heads further."""
    lens = [N + 100, 300]
    q, cache, kv, sc, table = problem(91, 2, 6, 3, N, d, 64, lens, torch.float16)
    want = run(q, cache, kv, sc, table, lens, True)
    k, v = (kv[:, i].transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for i in range(2))
    sc_d = sc.to(DEV)
    o = M.attention_paged_int8(q.to(DEV), k, v, sc_d[:, 0], sc_d[:, 1], table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), True, d ** -0.5)
    assert torch.equal(o.cpu(), want)


def test_offsets_past_32_bits():
    """Two pages at the ends of a pool of 4.3 GB."""
    page, Hkv, d = 256, 8, 256
    pages = (1 << 32) // (Hkv * page * d) + 8
    k = torch.zeros((pages, Hkv, page, d), dtype=torch.int8, device=DEV)
    v = torch.zeros((pages, Hkv, page, d), dtype=torch.int8, device=DEV)
    g = torch.Generator().manual_seed(83)
    small, kv, sc = make_cache(g, 2, Hkv, page, d)
    at = torch.tensor([pages - 1, 0])
    k[at], v[at] = small["k"].to(DEV), small["v"].to(DEV)
    ks, vs = torch.zeros((pages, Hkv), device=DEV), torch.zeros((pages, Hkv), device=DEV)
    ks[at], vs[at] = small["ks"].to(DEV), small["vs"].to(DEV)
    q = torch.randn((1, 16, 1, d), generator=g).half()
    lens = torch.tensor([400], dtype=torch.int32, device=DEV)
    o = M.attention_paged_int8(q.to(DEV), k, v, ks, vs, at.to(torch.int32)[None].to(DEV), lens, False, 0.0625)
    want, _, mean_v, size = attend(q, small, torch.tensor([[0, 1]]), [400], False, 0.0625)
    assert ((o.cpu().double() - want).abs() <= bound(want, mean_v, size, torch.float16)).all()
    M.paged_kvcache_append(k, ks, v, vs, q[:, :Hkv].to(DEV), q[:, 8:].to(DEV), at.flip(0).to(torch.int32)[None].to(DEV),
                           torch.tensor([256], dtype=torch.int32, device=DEV))
    assert (v[pages - 1, :, 0].cpu().float() * vs[pages - 1].cpu()[:, None] - q[0, 8:, 0].float()).abs().max() <= vs[pages - 1].max().item() * 0.51

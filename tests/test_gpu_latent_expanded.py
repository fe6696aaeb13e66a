"""The expanded form of latent attention against its formula in float64."""
import math

import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import expanded

pytestmark = pytest.mark.gpu
DIMS = [(128, 64, 128), (64, 32, 64)]


def bound(out, mean_v, size, dtype):
    """How far the kernel may be from the formula: half a step of the output's type; P rounded to the values' type, half a step of it of the mean of |v|; scores off by dS move
    a weight by dS and their sum as much: dS is at most fourteen roundings in fp32 (a score's sums over up to 192 products, its scale, the exponent) of the largest sum of |q k|,
    2^-19 of it; sums over keys 2^-14."""
    half = torch.finfo(dtype).eps / 2
    return half * out.abs() + 1.05 * (half + 2.0 ** -14 + 2.0 ** -18 * size) * mean_v + 2.0 ** -24


def inputs(g, Z, H, N, Nk, dims, dtype, size=1.2):
    dn, dr, dv = dims
    r = lambda *s: (torch.randn(s, generator=g) * size).to(dtype)  # noqa: E731
    return r(Z, H, N, dn), r(Z, H, N, dr), r(Z, H, Nk, dn), r(Z, 1, Nk, dr), torch.randn((Z, H, Nk, dv), generator=g).to(dtype)


def run(x, causal, sm, nq=None, nk=None, copies=1):
    """copies: of the heads, side by side; all give the same."""
    i32 = dict(dtype=torch.int32, device="cuda")
    heads = x[0].shape[1]
    x = [t.cuda() if i == 3 else t.cuda().repeat(1, copies, 1, 1) for i, t in enumerate(x)]      # (the rotary keys are all heads')
    out, lse = ifa.attention_latent(*x, causal, sm, seqlens_q=None if nq is None else torch.tensor(nq, **i32),
                                    seqlens_k=None if nk is None else torch.tensor(nk, **i32), return_lse=True)
    for i in range(heads, heads * copies, heads):
        assert torch.equal(out[:, i:i + heads].nan_to_num(7.0), out[:, :heads].nan_to_num(7.0)) and torch.equal(lse[:, i:i + heads].nan_to_num(7.0), lse[:, :heads].nan_to_num(7.0))
    return out[:, :heads].cpu(), lse[:, :heads].cpu()


def check(x, causal, sm=0.07, nq=None, nk=None, copies=1):
    out, lse = run(x, causal, sm, nq, nk, copies)
    want, want_lse, mean_v, size = expanded(*x, causal, sm, nq, nk)
    assert out.dtype == x[4].dtype and out.shape == want.shape
    # (inputs past their type's range are infinities, and where the formula has no number the kernel has none)
    none = want.isnan()
    assert torch.equal(out.isnan(), none) and torch.equal(lse.isnan(), want_lse.isnan())
    if none.all():
        return
    d, b = (out.double() - want)[~none].abs(), bound(want, mean_v, size, out.dtype)[~none]
    assert (d <= b).all(), f"{(d / b).max():.3f} of the bound at {int((d / b).view(-1).argmax())}"
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all()
    assert ((lse.double() - want_lse)[~empty].abs() <= (2.0 ** -18 * size)[..., 0][~empty] + 2.0 ** -14 + 2.0 ** -22 * want_lse[~empty].abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N,Nk", [(1, 1), (1, 64), (5, 5), (64, 64), (65, 200), (127, 128), (128, 127), (200, 130), (257, 257), (300, 700), (600, 600), (1, 1000), (900, 40)])
def test_lengths(dtype, dims, causal, N, Nk):
    """One query and many, one tile and pairs of them, an odd number of tiles, fewer keys than queries (rows that see none)."""
    g = torch.Generator().manual_seed(N + Nk)
    check(inputs(g, 2, 3, N, Nk, dims, dtype), causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N,Nk", [(1, 1), (5, 5), (64, 64), (65, 200), (128, 127), (200, 130), (257, 257), (300, 700), (1, 1000), (900, 40)])
def test_lengths_of_many_heads(dtype, dims, causal, N, Nk):
    """More tiles than compute units: a workgroup has pairs of them, each half one with all keys."""
    g = torch.Generator().manual_seed(N + Nk + 1)
    check(inputs(g, 2, 3, N, Nk, dims, dtype), causal, copies=43)


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_that_differ_of_many_heads(dims, causal):
    g = torch.Generator().manual_seed(4)
    nq, nk = [300, 0, 1, 129, 7, -3, 999], [300, 300, 10, 64, 0, 50, 255]
    check(inputs(g, 7, 2, 300, 310, dims, torch.bfloat16), causal, nq=nq, nk=nk, copies=13)
    check(inputs(g, 7, 2, 300, 310, dims, torch.float16), causal, nk=nk, copies=13)
    check(inputs(g, 7, 2, 300, 310, dims, torch.float16), causal, nq=nq, copies=13)


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_that_differ(dims, causal):
    g = torch.Generator().manual_seed(3)
    nq, nk = [300, 0, 1, 129, 7, -3, 999], [300, 300, 10, 64, 0, 50, 255]
    check(inputs(g, 7, 2, 300, 310, dims, torch.bfloat16), causal, nq=nq, nk=nk)
    check(inputs(g, 7, 2, 300, 310, dims, torch.float16), causal, nk=nk)
    check(inputs(g, 7, 2, 300, 310, dims, torch.float16), causal, nq=nq)


@pytest.mark.parametrize("Z,H", [(1, 1), (1, 8), (3, 5), (2, 20)])
def test_heads(Z, H):
    """(Sequence, head)s that the XCDs share evenly, and those left over."""
    g = torch.Generator().manual_seed(H)
    check(inputs(g, Z, H, 130, 150, DIMS[1], torch.float16), True)


def test_nothing_behind_the_keys_is_read():
    g = torch.Generator().manual_seed(5)
    x, nk = inputs(g, 2, 2, 150, 200, DIMS[0], torch.bfloat16), [70, 129]
    want = run(x, True, 0.07, nk=nk, nq=[70, 100])
    for z, n in enumerate(nk):
        for t in x[2:]:
            t[z, :, n:] = math.nan
    for z, m in enumerate([70, 100]):
        for t in x[:2]:
            t[z, :, m:] = math.nan
    for a, b in zip(run(x, True, 0.07, nk=nk, nq=[70, 100]), want):
        assert torch.equal(a, b)


def test_strides():
    """Slices of projections as they come, rows off their 16 bytes, a shared rotary key that is a slice."""
    g = torch.Generator().manual_seed(7)
    q = torch.randn((2, 140, 3, 192), generator=g).half().cuda().transpose(1, 2)
    kv = torch.randn((2, 190, 3, 256), generator=g).half().cuda().transpose(1, 2)
    rest = torch.randn((2, 190, 512 + 64), generator=g).half().cuda()
    x = q[..., :128], q[..., 128:], kv[..., :128], rest[:, None, :, 512:], kv[..., 128:]
    want = ifa.attention_latent(*(t.contiguous() for t in x), True, 0.07)
    assert torch.equal(ifa.attention_latent(*x, True, 0.07), want)
    odd = torch.randn((2, 3, 140, 129), generator=g).half().cuda()[..., 1:]
    assert torch.equal(ifa.attention_latent(odd, *x[1:], True, 0.07), ifa.attention_latent(odd.contiguous(), *x[1:], True, 0.07))


@pytest.mark.parametrize("sm", [-0.07, 0.0, 3.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("copies", [1, 65])
def test_scales_of_scores(sm, dtype, copies):
    g = torch.Generator().manual_seed(9)
    check(inputs(g, 1, 2, 140, 200, DIMS[0], dtype, 1.2 if abs(sm) < 1 else 0.2), True, sm, copies=copies)
    check(inputs(g, 1, 2, 140, 200, DIMS[1], dtype, 1.2 if abs(sm) < 1 else 0.2), False, sm, copies=copies)


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 14])
@pytest.mark.parametrize("copies", [1, 65])
def test_large_scores(size, copies):
    """Scores far past what an exponent's rounding leaves: the largest key has the row, to the bit of a tie."""
    g = torch.Generator().manual_seed(11)
    for dtype in (torch.float16, torch.bfloat16):
        qn, qr, kn, kr, v = inputs(g, 1, 2, 140, 200, DIMS[0], dtype)
        qn, kn = (qn * 0).to(dtype), (kn * 0).to(dtype)
        qr, kr = (qr * 0).to(dtype), (kr * 0).to(dtype)
        qn[..., 0] = size
        kn[..., 0] = (size * (1 + torch.arange(200) % 7)).to(dtype)            # exact products: seven sizes of score, ties among them
        check((qn, qr, kn, kr, v), False, 1.0, copies=copies)
        check((qn, qr, kn, kr, v), True, 1.0, copies=copies)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 120), (torch.float16, 3e4), (torch.bfloat16, 2.0 ** -100)])
@pytest.mark.parametrize("copies", [1, 65])
def test_values_of_any_size(dtype, size, copies):
    g = torch.Generator().manual_seed(13)
    x = list(inputs(g, 1, 2, 200, 1500, DIMS[0], dtype))
    x[4] = (torch.rand(x[4].shape, generator=g) * size).to(dtype)
    check(tuple(x), False, copies=copies)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("copies", [1, 65])
def test_queries_that_hold_no_number(bad, copies):
    g = torch.Generator().manual_seed(15)
    x = inputs(g, 1, 2, 200, 200, DIMS[0], torch.float16)
    want, want_lse = run(x, True, 0.07, copies=copies)
    x[0][0, 1, 50, 3] = bad
    out, lse = run(x, True, 0.07, copies=copies)
    assert out[0, 1, 50].isnan().all() and lse[0, 1, 50].isnan()
    keep = torch.ones((1, 2, 200), dtype=torch.bool)
    keep[0, 1, 50] = False
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


def test_no_keys_and_no_queries():
    g = torch.Generator().manual_seed(17)
    x = inputs(g, 2, 2, 5, 0, DIMS[0], torch.float16)
    out, lse = run(x, True, 0.07)
    assert (out == 0).all() and (lse == -math.inf).all()
    x = inputs(g, 2, 2, 0, 5, DIMS[0], torch.float16)
    assert run(x, True, 0.07)[0].shape == (2, 2, 0, 128)


def test_absorbed_and_expanded_agree():
    """The two forms of one layer: queries through the keys' matrix against the latent cache, and keys expanded by it."""
    g = torch.Generator().manual_seed(19)
    H, N, dc, dn, dr, dv, page = 4, 90, 512, 128, 64, 128, 32
    cache, scale = (t.cuda() for t in (torch.randint(-127, 128, (3, page, dc + dr), generator=g, dtype=torch.int8), torch.full((3, page, 2), 1 / 64.0)))
    table, lens = torch.tensor([[1, 0, 2]], dtype=torch.int32, device="cuda"), torch.tensor([N], dtype=torch.int32, device="cuda")
    rows = (cache.double() * scale.double()[..., :1])[table[0].long()].flatten(0, 1)[:N]
    wk, wv = ((torch.randn((H, dc, d), generator=g) / 24).double().cuda() for d in (dn, dv))
    q_nope, q_rope = (torch.randn((1, H, N, d), generator=g).half().cuda() for d in (dn, dr))
    q_latent = torch.matmul(q_nope.double(), wk.transpose(-1, -2).contiguous()).half()
    absorbed = ifa.attention_paged_latent_int8(q_latent, q_rope, cache, scale, table, lens, True, 0.07)
    a = torch.matmul(absorbed.double(), wv)
    b = ifa.attention_latent(q_nope, q_rope, torch.matmul(rows[:, :dc], wk)[None].half(), rows[None, None, :, dc:].half(), torch.matmul(rows[:, :dc], wv)[None].half(), True, 0.07)
    # (expanded keys, values and absorbed queries are rounded to fp16 here: 2^-11 each of what they are made of, and a score is a sum of 192 to 576 such products of about 2)
    assert (a - b.double()).abs().max() < 0.06 * b.double().abs().max()

"""Rotary positions against their formula in float64: layouts, parts of the head, strides, far positions, the gradient."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import int_flashattention_amd as M
from int_flashattention_amd import _capi
from paged_reference import rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(out, x, positions, freqs, magnitude=1.0, interleaved=False, inverse=False):
    """Half a step of the result; cos and sin within 8e-7 (the reduced angle in fp32 2e-7, the function 4 units of 2^-24 and its rounding,
    the two products and their sum one of 2^-24 each), so 1e-6 of |a| + |b|; fp16's smallest step."""
    want = rotate(x, positions, freqs, magnitude, interleaved, inverse)
    r, half = 2 * freqs.numel(), freqs.numel()
    size = x.double().abs().clone()
    a, b = (size[..., 0:r:2], size[..., 1:r:2]) if interleaved else (size[..., :half], size[..., half:r])
    both = (a + b).repeat_interleave(2, -1) if interleaved else torch.cat([a + b, a + b], -1)
    size[..., :r] = both
    tolerance = torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 1e-6) + 1e-6 * magnitude * size + 2.0 ** -25
    assert ((out.cpu().double() - want).abs() <= tolerance).all()
    assert torch.equal(out[..., r:].cpu(), x[..., r:])


@pytest.mark.parametrize("Z,H,N,d,rot,interleaved,inverse,dtype", [
    (1, 1, 1, 16, 16, False, False, torch.float16),
    (2, 3, 5, 32, 16, True, False, torch.bfloat16),
    (1, 32, 1, 128, 128, False, False, torch.float16),
    (3, 5, 67, 64, 32, True, True, torch.float16),
    (2, 9, 33, 128, 64, False, True, torch.bfloat16),
    (1, 4, 130, 256, 256, False, False, torch.bfloat16),
    (1, 2, 257, 256, 80, True, False, torch.float16),
    (2, 12, 300, 64, 64, False, False, torch.float16),
])
def test_formula(Z, H, N, d, rot, interleaved, inverse, dtype):
    g = torch.Generator().manual_seed(Z * 1000 + N)
    x = torch.randn((Z, H, N, d), generator=g).to(dtype)
    freqs, magnitude = M.rotary_frequencies(rot, device=DEV, scaling="parts", factor=4.0, original_length=2048)
    first = torch.randint(0, 5000, (Z,), generator=g, dtype=torch.int32)
    rows = torch.arange(N)
    out = M.rotary(x.to(DEV), first.to(DEV), freqs, interleaved=interleaved, inverse=inverse, magnitude=magnitude)
    assert out.is_contiguous() and out.dtype == dtype
    check(out, x, first[:, None] + rows, freqs.cpu(), magnitude, interleaved, inverse)
    each = torch.randint(-100, 100000, (Z, N), generator=g, dtype=torch.int32)
    check(M.rotary(x.to(DEV), each.to(DEV), freqs, interleaved=interleaved, inverse=inverse), x, each, freqs.cpu(), 1.0, interleaved, inverse)
    check(M.rotary(x.to(DEV), 17, freqs, interleaved=interleaved, inverse=inverse), x, (17 + rows).expand(Z, N), freqs.cpu(), 1.0, interleaved, inverse)


def test_strides_and_one_position_for_all_rows():
    g = torch.Generator().manual_seed(5)
    freqs, _ = M.rotary_frequencies(64, device=DEV)
    y = torch.randn((2, 37, 6, 128), generator=g).half()                       # [Z, N, H, d]
    x = y.transpose(1, 2)
    pos = torch.tensor([[40], [7]], dtype=torch.int32)
    out = M.rotary(y.to(DEV).transpose(1, 2), pos.to(DEV).expand(2, 37), freqs)   # a row stride of zero: every row at the same position
    check(out, x, pos.expand(2, 37), freqs.cpu())
    odd = torch.randn((2, 3, 9, 130), generator=g).bfloat16()[..., 1:129]       # rows that are not 16-byte aligned
    check(M.rotary(odd.to(DEV), 3, freqs), odd.contiguous(), (3 + torch.arange(9)).expand(2, 9), freqs.cpu())


MANY_HEADS = [          # (two, four, four, eight and eight heads a thread; the last thread's share is smaller)
    (1, 5, 4000, 128, 128, False, False, torch.float16),
    (1, 5, 8000, 128, 64, True, True, torch.bfloat16),
    (4, 9, 1500, 128, 128, True, False, torch.float16),
    (4, 13, 3000, 128, 64, False, True, torch.bfloat16),
    (2, 13, 2100, 256, 80, True, False, torch.float16),
]


@pytest.mark.parametrize("Z,H,N,d,rot,interleaved,inverse,dtype", MANY_HEADS)
def test_several_heads_a_thread(Z, H, N, d, rot, interleaved, inverse, dtype):
    g = torch.Generator().manual_seed(N)
    y = torch.randn((Z, N, H, d), generator=g).to(dtype)                       # (heads side by side)
    freqs, magnitude = M.rotary_frequencies(rot, device=DEV, scaling="parts", factor=4.0, original_length=2048)
    first = torch.randint(0, 5000, (Z,), generator=g, dtype=torch.int32)
    kw = dict(interleaved=interleaved, inverse=inverse, magnitude=magnitude)
    out = M.rotary(y.to(DEV).transpose(1, 2), first.to(DEV), freqs, **kw)
    check(out, y.transpose(1, 2), first[:, None] + torch.arange(N), freqs.cpu(), magnitude, interleaved, inverse)
    leaf = y.transpose(1, 2).contiguous().to(DEV).requires_grad_()
    grad = torch.randn((Z, H, N, d), generator=g).to(dtype).to(DEV)
    M.rotary(leaf, first.to(DEV), freqs, **kw).backward(grad)
    kw["inverse"] = not inverse
    assert torch.equal(leaf.grad, M.rotary(grad, first.to(DEV), freqs, **kw))
    check(leaf.grad, grad.cpu(), first[:, None] + torch.arange(N), freqs.cpu(), magnitude, interleaved, not inverse)


@pytest.mark.parametrize("Z,H,N,d,rot,interleaved,inverse,dtype", MANY_HEADS + [(2, 3, 7, 64, 32, False, False, torch.float16), (1, 32, 1, 128, 128, True, False, torch.bfloat16)])
def test_in_place(Z, H, N, d, rot, interleaved, inverse, dtype):
    """The C entry with out = x gives the bits of a result of its own."""
    x = torch.randn((Z, H, N, d), generator=torch.Generator().manual_seed(d)).to(dtype).to(DEV)
    freqs, _ = M.rotary_frequencies(rot, device=DEV)
    want = M.rotary(x, 11, freqs, interleaved=interleaved, inverse=inverse)
    p = _capi.RotaryParams()
    p.x = p.out = x.data_ptr()
    for t in "xo":
        setattr(p, f"{t}_stride_b", x.stride(0)); setattr(p, f"{t}_stride_h", x.stride(1)); setattr(p, f"{t}_stride_n", x.stride(2))
    p.position_first, p.inverse = 11, int(inverse)
    p.rope.freqs, p.rope.pairs, p.rope.interleaved, p.rope.magnitude = freqs.data_ptr(), freqs.numel(), int(interleaved), 1.0
    p.batch, p.heads, p.seqlen, p.head_dim, p.dtype = Z, H, N, d, _capi.INTFA_F16 if dtype == torch.float16 else _capi.INTFA_BF16
    assert _capi.load().intfa_rotary(ctypes.byref(p), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert torch.equal(x, want)


def test_far_positions_keep_their_angle():
    freqs, _ = M.rotary_frequencies(128, base=500000.0, device=DEV)
    x = torch.randn((1, 2, 6, 128), generator=torch.Generator().manual_seed(6)).half()
    pos = torch.tensor([[2 ** 31 - 1, 2 ** 30 + 12345, 16777217, 1 << 20, -(2 ** 31), -1]], dtype=torch.int32)
    check(M.rotary(x.to(DEV), pos.to(DEV), freqs), x, pos, freqs.cpu())


@pytest.mark.parametrize("first", [2 ** 31 - 1, 2 ** 31 - 3, -(2 ** 31)])
def test_rows_count_on_past_32_bits(first):
    """From a first position on the device that the last rows leave 32 bits behind."""
    freqs, _ = M.rotary_frequencies(128, base=500000.0, device=DEV)
    x = torch.randn((2, 2, 9, 128), generator=torch.Generator().manual_seed(10)).bfloat16()
    out = M.rotary(x.to(DEV), torch.tensor([first, 5], dtype=torch.int32, device=DEV), freqs)
    check(out, x, torch.tensor([[first], [5]]) + torch.arange(9), freqs.cpu())


def test_values_that_are_not_finite_stay_in_their_pair():
    freqs, _ = M.rotary_frequencies(32, device=DEV)
    x = torch.randn((1, 1, 4, 64), generator=torch.Generator().manual_seed(7)).half()
    x[0, 0, 1, 3], x[0, 0, 2, 40] = float("nan"), float("inf")
    out = M.rotary(x.to(DEV), 5, freqs).cpu()
    bad = torch.zeros(64, dtype=torch.bool)
    bad[3] = bad[3 + 16] = True
    assert out[0, 0, 1][bad].isnan().all() and out[0, 0, 1][~bad].isfinite().all()
    assert out[0, 0, 2, 40] == float("inf") and out[0, 0, 2].isfinite().sum() == 63


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved):
    """The map is linear: its gradient is the transposed map, <R x, y> = <x, R^T y>, and the difference quotient is exact."""
    g = torch.Generator().manual_seed(8)
    freqs, magnitude = M.rotary_frequencies(48, device=DEV, scaling="parts", factor=8.0, original_length=1024)
    x = torch.randn((2, 3, 11, 64), generator=g).bfloat16()
    y = torch.randn((2, 3, 11, 64), generator=g).bfloat16()
    first = torch.tensor([3, 900], dtype=torch.int32)
    leaf = x.to(DEV).requires_grad_()
    out = M.rotary(leaf, first.to(DEV), freqs, interleaved=interleaved, magnitude=magnitude)
    out.backward(y.to(DEV))
    pos = first[:, None] + torch.arange(11)
    check(leaf.grad, y, pos, freqs.cpu(), magnitude, interleaved, inverse=True)
    ref = rotate(x, pos, freqs.cpu(), magnitude, interleaved)
    d = torch.zeros_like(x).double()
    d[0, 1, 4, 5] = 1.0
    quotient = ((rotate(x.double() + d, pos, freqs.cpu(), magnitude, interleaved) - ref) * y.double()).sum()
    assert abs(leaf.grad[0, 1, 4, 5].item() - quotient.item()) <= 2.0 ** -8 * abs(quotient.item()) + 1e-5
    leaf.grad = None
    M.rotary(leaf, 4, freqs, interleaved=interleaved).sum().backward()           # (the gradient of a sum: one value, expanded)
    check(leaf.grad, torch.ones_like(x), (4 + torch.arange(11)).expand(2, 11), freqs.cpu(), 1.0, interleaved, inverse=True)
    with torch.no_grad():
        assert not M.rotary(leaf, 4, freqs).requires_grad


@pytest.mark.parametrize("first", [7, "tensor"])
@pytest.mark.parametrize("inverse", [False, True])
def test_tangents(first, inverse):
    """Forward mode: the map of the tangent, for inputs that require a gradient and for those that do not."""
    g = torch.Generator().manual_seed(11)
    freqs, magnitude = M.rotary_frequencies(32, device=DEV, scaling="parts", factor=4.0, original_length=512)
    x, t = (torch.randn((2, 3, 9, 64), generator=g).half().to(DEV) for _ in range(2))
    first = torch.tensor([3, 70], dtype=torch.int32, device=DEV) if first == "tensor" else first

    def turn(a):
        return M.rotary(a, first, freqs, inverse=inverse, interleaved=True, magnitude=magnitude)

    want = turn(t)
    for leaf in (x, x.clone().requires_grad_()):
        with forward_ad.dual_level():
            out, tangent = forward_ad.unpack_dual(turn(forward_ad.make_dual(leaf, t)))
            assert torch.equal(out, turn(x)) and torch.equal(tangent, want)
            assert forward_ad.unpack_dual(turn(x)).tangent is None
    out, tangent = torch.func.jvp(turn, (x,), (t,))
    assert torch.equal(out, turn(x)) and torch.equal(tangent, want)


def test_gradients_of_gradients():
    """d/dy <R^T y, t> = R t: the backward pass is differentiated, by reverse mode twice and by forward over reverse."""
    g = torch.Generator().manual_seed(12)
    freqs, _ = M.rotary_frequencies(64, device=DEV)
    x, y, t = (torch.randn((1, 2, 5, 64), generator=g).bfloat16().to(DEV) for _ in range(3))
    x.requires_grad_()
    y.requires_grad_()
    dx, = torch.autograd.grad(M.rotary(x, 6, freqs), x, y, create_graph=True)
    dy, = torch.autograd.grad(dx, y, t)
    assert torch.equal(dx, M.rotary(y, 6, freqs, inverse=True)) and torch.equal(dy, M.rotary(t, 6, freqs))
    _, tangent = torch.func.jvp(torch.func.grad(lambda a: (M.rotary(a, 6, freqs).float() ** 2).sum() / 2), (x.detach(),), (t,))
    want = M.rotary(M.rotary(t, 6, freqs), 6, freqs, inverse=True)
    assert torch.equal(tangent, want)


def test_a_captured_training_step():
    """Forward and backward in one captured graph, replayed over new inputs with eager work in between."""
    g = torch.Generator().manual_seed(9)
    freqs, _ = M.rotary_frequencies(64, device=DEV)
    x, y = (torch.zeros((2, 4, 50, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pos = torch.zeros((2,), dtype=torch.int32, device=DEV)
    leaf = x.requires_grad_()

    def step():
        out = M.rotary(leaf, pos, freqs)
        return out, *torch.autograd.grad(out, leaf, y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                                # (nothing of its graph is kept)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dx = step()
    for k in range(4):
        with torch.no_grad():
            leaf.copy_(torch.randn(x.shape, generator=g))
            y.copy_(torch.randn(x.shape, generator=g))
            pos.copy_(torch.randint(0, 9000, (2,), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(out, M.rotary(leaf, pos, freqs)) and torch.equal(dx, M.rotary(y, pos, freqs, inverse=True))

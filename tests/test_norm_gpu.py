"""GPU: add_rms_norm, its 8-bit rows and its gradient against the formulas in fp64.

Tolerances (u = half a unit in the last place of the output type, 2^-11 fp16, 2^-8 bf16, 2^-24 fp32):
  the kernel's fp32 part: a sum of squares over at most 16384 elements is a tree of at most 16 + 10 +
  10 additions, so its relative error is below 40 * 2^-24 = 2.4e-6, halved by the square root; with
  the products of y below F32 = 4e-6 relative. Then one rounding u.
  Gradients: the same relative error on every term of a sum whose terms may cancel: F32 times 2.5 on
  the sum of the terms' magnitudes; dweight adds up to T / groups terms in order (at most 512 here).
"""
import pytest
import torch

from muxi_race_b200 import add_rms_norm, add_rms_norm_backward, add_rms_norm_quant
from oracle.norm_ref import rms_norm_grad_ref, rms_norm_ref

pytestmark = pytest.mark.gpu
F16, BF16, F32T = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32T: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32T: 0.0}  # half the spacing of fp16's subnormal values
F32 = 4e-6


def randn(seed, *shape, dtype=F32T, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, worst {float((err - tol).max()):.3e} over"


def check_forward(x, w, res, eps=1e-6):
    r = add_rms_norm(x, w, res, eps=eps)
    y, h = r if res is not None else (r, None)
    ry, rh = rms_norm_ref(x, w, res, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    u, t = U[x.dtype], TINY[x.dtype]
    within(y, ry, (u + F32) * ry.abs() + t, "y")
    if res is not None:
        within(h, rh, (u + 2.0 ** -24) * rh.abs() + t, "h")
    return y, h


@pytest.mark.parametrize("H", [1, 7, 64, 100, 129, 1000, 1024, 2056, 4097, 7168, 8200, 12288, 16384])
@pytest.mark.parametrize("dtype,wdtype", [(F16, F16), (BF16, F32T), (F32T, F32T), (BF16, BF16), (F16, F32T)])
@pytest.mark.parametrize("T", [1, 5, 300])
def test_forward(cuda_device, H, dtype, wdtype, T):
    x, w = randn(1, T, H, dtype=dtype), randn(2, H, dtype=wdtype)
    check_forward(x, w, randn(3, T, H, dtype=dtype, scale=2.0))
    check_forward(x, w, None)


@pytest.mark.parametrize("H", [1, 60, 129, 1024, 4096, 5001, 7168, 16384])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("T", [1, 200])
def test_quant(cuda_device, H, dtype, q_dtype, T):
    """|q scale - y| is at most half a step: 0.5 scale for int8; for e4m3 2^-4 of the value, or half
    of the subnormal step 2^-9 of the scaled value."""
    x, w, res = randn(4, T, H, dtype=dtype), randn(5, H, dtype=F32T), randn(6, T, H, dtype=dtype)
    q, scale, h = add_rms_norm_quant(x, w, res, q_dtype=q_dtype)
    ry, rh = rms_norm_ref(x, w, res)
    assert q.dtype == q_dtype and scale.shape == (T,)
    kmax = 127.0 if q_dtype == torch.int8 else 448.0
    rscale = ry.abs().amax(-1) / kmax
    within(scale, rscale, 2 * F32 * rscale, "scale")
    s = rscale[:, None]
    step = 0.5 * s if q_dtype == torch.int8 else torch.maximum(ry.abs() * 2.0 ** -4, s * 2.0 ** -10)
    within(q.float().double() * scale.double()[:, None], ry, step + 4 * F32 * (ry.abs() + s * kmax), "q * scale")
    within(h, rh, (U[dtype] + 2.0 ** -24) * rh.abs() + TINY[dtype], "h")


@pytest.mark.parametrize("H", [1, 33, 256, 512, 1000, 4096, 4104, 7168, 8192, 9001, 16384])
@pytest.mark.parametrize("dtype,wdtype", [(F16, F16), (BF16, F32T), (F32T, F32T)])
@pytest.mark.parametrize("T", [1, 37, 1500])
def test_backward(cuda_device, H, dtype, wdtype, T):
    dy, h, w = randn(7, T, H, dtype=dtype), randn(8, T, H, dtype=dtype, scale=2.0), randn(9, H, dtype=wdtype)
    for dh in (None, randn(10, T, H, dtype=dtype)):
        dx, dw = add_rms_norm_backward(dy, h, w, dh)
        rdx, rdw, mx, mw = rms_norm_grad_ref(dy, h, w, dh)
        assert dx.dtype == dtype and dw.dtype == wdtype
        within(dx, rdx, U[dtype] * rdx.abs() + 2.5 * F32 * mx + TINY[dtype], "dx")
        within(dw, rdw, U[wdtype] * rdw.abs() + 2.5 * F32 * mw + TINY[wdtype], "dweight")
        dx2, dw2 = add_rms_norm_backward(dy, h, w, dh)
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2), "not the same bits on a second run"


def test_autograd_and_differences(cuda_device):
    """The autograd form gives the formula's gradients, and the loss moves along the gradient as they
    say: (L(x + e v) - L(x - e v)) / 2e against |dx|, v the gradient's direction. With e |v| = 1 % of
    |x| the third-order term is below 1e-4 of it, and fp32 rounding of L (6e-8 of a sum of 6 * 500
    terms of order 1, over e = 0.5) below 1e-3."""
    T, H = 6, 500
    x, w, res, dy = (randn(s, *shape) for s, shape in ((11, (T, H)), (12, (H,)), (13, (T, H)), (14, (T, H))))
    dhx = randn(15, T, H) * 0.1
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    y, h = add_rms_norm(*leaves)
    ((y * dy).sum() + (h * dhx).sum()).backward()
    rdx, rdw, mx, mw = rms_norm_grad_ref(dy, x + res, w, dhx)
    within(leaves[0].grad, rdx, 4 * F32 * mx, "dx")
    within(leaves[1].grad, rdw, 4 * F32 * mw, "dweight")
    assert torch.equal(leaves[0].grad, leaves[2].grad)

    def loss(xx, ww):
        y, h = add_rms_norm(xx, ww, res)
        return float((y.double() * dy.double()).sum() + (h.double() * dhx.double()).sum())

    for i, t in ((0, x), (1, w)):
        g = leaves[i].grad
        v = g / g.norm()
        e = 0.01 * float(t.norm())
        a = [x, w]
        a[i] = t + e * v
        up = loss(*a)
        a[i] = t - e * v
        slope = (up - loss(*a)) / (2 * e)
        assert abs(slope - float(g.norm())) <= 2e-3 * float(g.norm()), (i, slope, float(g.norm()))


def test_autograd_without_residual_and_of_the_sum_alone(cuda_device):
    x, w = randn(16, 3, 4, 64).requires_grad_(), randn(17, 64).requires_grad_()
    add_rms_norm(x, w).sum().backward()
    rdx, rdw, mx, mw = rms_norm_grad_ref(torch.ones(3, 4, 64).cuda(), x, w)
    within(x.grad, rdx, 4 * F32 * mx, "dx")
    within(w.grad, rdw, 4 * F32 * mw, "dweight")
    x.grad = w.grad = None
    res = randn(18, 1, 1, 64).requires_grad_()  # a broadcast residual: its gradient is summed
    _, h = add_rms_norm(x, w, res.expand(3, 4, 64).contiguous())
    (h * 2).sum().backward()
    assert bool((x.grad == 2).all()) and bool((res.grad == 24).all()) and w.grad is None


@pytest.mark.parametrize("H", [256, 250, 4096])
def test_pitches_and_alignment(cuda_device, H):
    """Rows inside wider tensors (16-byte and odd starts), one row for all tokens, leading dimensions."""
    big = randn(19, 40, H + 24, dtype=F16)
    w = randn(20, H, dtype=F16)
    for off in (0, 8, 3):
        x, res = big[:, off:off + H], big[:20].repeat(2, 1)[:, 24 - off:24 - off + H]
        check_forward(x, w, res)
    one = big[:1, :H].expand(40, H)
    check_forward(big[:, 1:H + 1], w, one)
    check_forward(big[:, :H].reshape(4, 10, H)[:, :, :], w, None)
    dy = big[:, 5:5 + H]
    dx, dw = add_rms_norm_backward(dy, one, w, big[:, 8:8 + H])
    rdx, rdw, mx, mw = rms_norm_grad_ref(dy, one, w, big[:, 8:8 + H])
    within(dx, rdx, U[F16] * rdx.abs() + 2.5 * F32 * mx + TINY[F16], "dx")
    within(dw, rdw, U[F16] * rdw.abs() + 2.5 * F32 * mw + TINY[F16], "dweight")


@pytest.mark.parametrize("H", [64, 7168, 999])
def test_in_place(cuda_device, H):
    x, w, res = randn(21, 33, H, dtype=BF16), randn(22, H, dtype=BF16), randn(23, 33, H, dtype=BF16)
    y, h = add_rms_norm(x, w, res)
    x2, res2 = x.clone(), res.clone()
    y2, h2 = add_rms_norm(x2, w, res2, out=x2, residual_out=res2)
    assert y2 is x2 and h2 is res2 and torch.equal(y, x2) and torch.equal(h, res2)


def test_values_at_the_edges(cuda_device):
    w = torch.ones(64, device="cuda", dtype=F16)
    zero = torch.zeros(2, 64, device="cuda", dtype=F16)
    assert bool((add_rms_norm(zero, w) == 0).all())
    q, scale, _ = add_rms_norm_quant(zero, w)
    assert bool((q == 0).all()) and bool((scale == 0).all())
    dx, dw = add_rms_norm_backward(torch.ones_like(zero), zero, w)
    within(dx, torch.full((2, 64), 1e3, device="cuda", dtype=torch.float64), 1.0, "dx of a zero row is dy / sqrt(eps)")
    # the sum of two values beyond fp16's range: the norm is finite, the stored sum is not
    y, h = add_rms_norm(torch.full((1, 64), 6e4, device="cuda", dtype=F16), w,
                        torch.full((1, 64), 6e4, device="cuda", dtype=F16))
    assert bool((y == 1).all()) and bool(h.isinf().all())
    x = torch.zeros(3, 64, device="cuda", dtype=F16)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    q, scale, _ = add_rms_norm_quant(x, w)
    assert float(scale[0]) == 0 and bool(scale[1:].isnan().all())  # a spoilt row says so, the others are whole
    y = add_rms_norm(x, w)
    assert bool(y[0].eq(0).all()) and bool(y[1].isnan().all())


def test_empty_and_other_stream(cuda_device):
    w = randn(24, 128, dtype=F16)
    assert add_rms_norm(torch.empty(0, 128, device="cuda", dtype=F16), w).shape == (0, 128)
    dx, dw = add_rms_norm_backward(torch.empty(0, 128, device="cuda", dtype=F16), torch.empty(0, 128, device="cuda", dtype=F16), w)
    assert dx.shape == (0, 128) and bool((dw == 0).all())
    x = randn(25, 64, 128, dtype=F16)
    ref = add_rms_norm(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = add_rms_norm(x, w)
    s.synchronize()
    assert torch.equal(y, ref)


def test_more_than_2_31_elements(cuda_device):
    T, H = 299_999, 7168  # 2.15e9 elements
    x = torch.empty(T, H, device="cuda", dtype=BF16)
    x[-300:] = randn(26, 300, H, dtype=BF16)
    x[:-300] = 1
    w = randn(27, H, dtype=BF16)
    y, h = add_rms_norm(x, w, x)
    ry, rh = rms_norm_ref(x[-300:], w, x[-300:])
    within(y[-300:], ry, (U[BF16] + F32) * ry.abs(), "y")
    within(h[-300:], rh, (U[BF16] + F32) * rh.abs(), "h")
    del y
    dx, _ = add_rms_norm_backward(x, h, w)
    rdx, _, mx, _ = rms_norm_grad_ref(x[-300:], h[-300:], w)
    within(dx[-300:], rdx, U[BF16] * rdx.abs() + 2.5 * F32 * mx, "dx")


def test_refusals(cuda_device):
    x, w = randn(28, 4, 64, dtype=F16), randn(29, 64, dtype=F16)
    with pytest.raises(ValueError, match="CUDA"):
        add_rms_norm(x.cpu(), w)
    with pytest.raises(ValueError, match="weight"):
        add_rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="dtype of x or fp32"):
        add_rms_norm(x, w.to(BF16))
    with pytest.raises(ValueError, match="residual must have the shape"):
        add_rms_norm(x, w, x[:2])
    with pytest.raises(ValueError, match="last dimension"):
        add_rms_norm(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="needs a residual"):
        add_rms_norm(x, w, residual_out=x)
    with pytest.raises(ValueError, match="q_dtype"):
        add_rms_norm_quant(x, w, q_dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="hidden must be"):
        add_rms_norm(torch.zeros(2, 16385, device="cuda", dtype=F16), torch.zeros(16385, device="cuda", dtype=F16))
    with pytest.raises(RuntimeError, match="8-bit rows need"):
        add_rms_norm_quant(x.float(), w.float())
    with pytest.raises(ValueError, match="not differentiable"):
        add_rms_norm(x.clone().requires_grad_(), w, out=torch.empty_like(x))

"""GPU: silu_mul with its gradient and 8-bit copies of rows against the formulas in fp64.

Tolerances (u: half a step of the output's type, 2^-11 fp16, 2^-8 bf16, 2^-24 fp32):
  e^-g by the approximate exponential is within 2 + 1.16 |g| units of 2^-23, its reciprocal and the up to eight products
  and sums behind it add less than 14 more: F(g) = (16 + 1.2 |g|) 2^-23 of a value's magnitude. A value is then rounded once.
  A row's sum dw adds at most 8192 / 512 * 16 terms in a lane, then 5 + 8 partial sums: below 300 * 2^-24 of the terms' sum more.
  8-bit copies are compared exactly with the codes of the definition; scales (one fp32 division) within 2^-24,
  and what is restored is one rounding of a product that is itself rounded to fp32: u + 2^-23.
"""
import pytest
import torch

import muxi_race_b200 as m
from oracle.train_ref import rows8_ref, silu_mul_grad_ref, silu_mul_ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
I8, F8 = torch.int8, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, torch.float32: 0.0}
WIDTHS = [1, 7, 8, 16, 100, 127, 128, 129, 136, 500, 512, 1000, 1024, 2048, 2056, 4100, 7168]


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def within(got, ref, tol, what):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off"


def values(saved):
    """What the codes say, in fp64, with the stored scales."""
    q = saved.q.float().double()
    R, W = q.shape
    w = W // saved.parts
    s = saved.scale.double().view(R, saved.parts, -1).repeat_interleave(128, 2)[:, :, :w].reshape(R, W)
    return q * s


def check_codes(saved, x):
    ref, scale = rows8_ref(x, saved.q.dtype, saved.parts)
    within(saved.scale, scale, 2.0 ** -24 * scale, "scale")
    got = values(saved)
    # codes are whole multiples of the scale: equal codes differ by the scale's own rounding only
    within(got, ref, 2.0 ** -23 * ref.abs(), "codes")


def F(gate):
    return (16 + 1.2 * gate.double().abs()) * 2.0 ** -23


@pytest.mark.parametrize("W", WIDTHS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_dtype", [I8, F8])
@pytest.mark.parametrize("R", [1, 67])
def test_save_and_restore(cuda_device, W, dtype, q_dtype, R):
    x = randn(1, R, W, dtype=dtype, scale=3.0)
    x[0, : W // 2] = 0
    saved = m.save_rows8(x, q_dtype)
    assert saved.q.dtype == q_dtype and saved.shape == (R, W) and saved.scale.shape == (R, -(-W // 128))
    check_codes(saved, x)
    back = m.restore_rows8(saved)
    v = values(saved)
    assert back.dtype == dtype
    within(back, v, (U[dtype] + 2.0 ** -23) * v.abs() + TINY[dtype], "restored")
    index = torch.tensor([R - 1, 0, -1, R, 0, R // 2], device="cuda")
    for idx in (index, index.int()):
        rows = m.restore_rows8(saved, idx)
        want = torch.stack([back[i] if 0 <= i < R else torch.zeros_like(back[0]) for i in idx.tolist()])
        assert torch.equal(rows, want)


@pytest.mark.parametrize("q_dtype", [I8, F8])
def test_every_ratio_of_two_values(cuda_device, q_dtype):
    """Codes of values that are ties or next to one: every bf16 mantissa against every maximum's mantissa."""
    mant = (1 + torch.arange(128).double() / 128)
    top = mant.repeat_interleave(4 * 4)                         # a maximum for each row, four rows of 2^0 .. 2^-8 each
    shift = torch.tensor([0.0, 1.0, 2.0, 5.0]).repeat_interleave(4).repeat(128).double()
    x = torch.where(torch.arange(2048)[:, None] % 2 == 0, 1.0, -1.0) * mant[None, :].repeat(2048, 1) * 2.0 ** -shift[:, None]
    x = torch.minimum(x.abs(), top[:, None]) * x.sign()
    x[:, 0] = top
    x = x.to(BF16).cuda()
    check_codes(m.save_rows8(x, q_dtype), x)


@pytest.mark.parametrize("q_dtype", [I8, F8])
def test_extreme_rows(cuda_device, q_dtype):
    """Subnormal groups, the largest values, zeros; a NaN or an infinity spoils its group and no other."""
    x = randn(2, 9, 300, dtype=BF16)
    x[0] *= 1e-38
    x[1] = torch.tensor(2.0 ** -133, dtype=BF16)
    x[2] *= 1e38
    x[3] = 0
    x[4, :128] *= 2.0 ** -101
    saved = m.save_rows8(x, q_dtype)
    ref, scale = rows8_ref(x, q_dtype)
    # a scale below 2^-126 is a whole number of 2^-149
    within(saved.scale, scale, 2.0 ** -24 * scale + 2.0 ** -150, "scale")
    # int8's codes follow the unrounded scale: off by the scale's rounding times the code
    within(values(saved), ref, 2.0 ** -23 * ref.abs() + 127 * 2.0 ** -150, "codes")
    x[5, 3], x[6, 200], x[7, 299] = float("nan"), float("inf"), float("-inf")
    back = m.restore_rows8(m.save_rows8(x, q_dtype))
    nan = torch.isnan(back)
    want = torch.zeros_like(nan)
    want[5, :128], want[6, 128:256], want[7, 256:] = True, True, True
    assert torch.equal(nan, want) and torch.isfinite(back[~nan]).all()


def test_save_of_strided_rows_and_parts(cuda_device):
    base = randn(3, 20, 600, dtype=BF16)
    for x in (base[:, 8:520], base[::2, 3:259], base[:1, 1:599]):
        check_codes(m.save_rows8(x), x)
        check_codes(m.save_rows8(x, F8, parts=2), x)
    cube = base.view(4, 5, 600)
    saved = m.save_rows8(cube)
    assert saved.shape == (4, 5, 600) and saved.scale.shape == (4, 5, 5)
    assert torch.equal(m.restore_rows8(saved).view(20, 600), m.restore_rows8(m.save_rows8(base)))
    out = torch.empty_like(cube)
    assert m.restore_rows8(saved, out=out) is out and torch.equal(out, m.restore_rows8(saved))


@pytest.mark.parametrize("I", WIDTHS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("weights", [None, torch.float32, BF16])
@pytest.mark.parametrize("R", [1, 150])
def test_silu_mul(cuda_device, I, dtype, weights, R):
    gate_up = randn(4, R, 2 * I, dtype=dtype, scale=2.0)
    w = None if weights is None else randn(5, R, dtype=weights).abs()
    h = m.silu_mul(gate_up, w)
    ref = silu_mul_ref(gate_up, w)
    assert h.dtype == dtype and h.shape == (R, I)
    within(h, ref, (U[dtype] + F(gate_up[:, :I])) * ref.abs() + TINY[dtype], "h")
    for q_dtype in (I8, F8):
        h2, saved = m.silu_mul_rows8(gate_up, w, q_dtype)
        assert torch.equal(h, h2)
        assert saved.parts == 2 and saved.dtype == dtype
        check_codes(saved, gate_up)


@pytest.mark.parametrize("I", WIDTHS)
@pytest.mark.parametrize("dtype,weights", [(F16, None), (BF16, torch.float32), (F16, F16)])
@pytest.mark.parametrize("kind", [None, I8, F8])
@pytest.mark.parametrize("R", [1, 150])
def test_silu_mul_backward(cuda_device, I, dtype, weights, kind, R):
    gate_up, dh = randn(6, R, 2 * I, dtype=dtype, scale=2.0), randn(7, R, I, dtype=dtype)
    w = None if weights is None else randn(8, R, dtype=weights)
    src = gate_up if kind is None else m.save_rows8(gate_up, kind, parts=2)
    x = gate_up if kind is None else values(src)
    dgu, dw, h = m.silu_mul_backward(dh, src, w)
    rd, rw, mag, mag_w = silu_mul_grad_ref(dh, x, w)
    f = F(x[:, :I])
    within(dgu, rd, U[dtype] * rd.abs() + torch.cat((f, f), -1) * mag + TINY[dtype], "dgate_up")
    rh = silu_mul_ref(x, w)
    within(h, rh, (U[dtype] + f) * rh.abs() + TINY[dtype], "h")
    if w is None:
        assert dw is None
    else:
        assert dw.dtype == weights and dw.shape == (R,)
        tol = f.amax(-1) + 300 * 2.0 ** -24
        within(dw, rw, U[weights] * rw.abs() + tol * mag_w + TINY[weights], "dweights")
    again = m.silu_mul_backward(dh, src, w)
    assert torch.equal(dgu, again[0]) and torch.equal(h, again[2]) and (w is None or torch.equal(dw, again[1]))


def test_far_gates(cuda_device):
    """Gates where e^-g is 0 or infinite in fp32: h and the gradients stay finite and take the limits."""
    g = torch.tensor([-3e4, -200.0, -100.0, -88.0, -50.0, 50.0, 88.0, 100.0, 3e4, 0.0], dtype=BF16)
    gate_up = torch.cat((g, torch.ones(10, dtype=BF16)))[None].cuda()
    h = m.silu_mul(gate_up)
    ref = silu_mul_ref(gate_up)
    # below 2^-126 the reciprocal is 0
    within(h, ref, (U[BF16] + F(gate_up[:, :10])) * ref.abs() + 1e-34, "h")
    dgu, _, _ = m.silu_mul_backward(torch.ones_like(h), gate_up)
    rd, _, mag, _ = silu_mul_grad_ref(torch.ones_like(h), gate_up)
    f = F(gate_up[:, :10])
    within(dgu, rd, U[BF16] * rd.abs() + torch.cat((f, f), -1) * mag + 1e-34, "dgate_up")


def test_autograd(cuda_device):
    R, I = 33, 200
    gate_up, w, dh = randn(9, R, 2 * I, dtype=BF16), randn(10, R), randn(11, R, I, dtype=BF16)
    for save in (None, I8, F8):
        a, b = gate_up.clone().requires_grad_(), w.clone().requires_grad_()
        h = m.silu_mul(a, b, save=save)
        h.backward(dh)
        src = gate_up if save is None else m.save_rows8(gate_up, save, parts=2)
        dgu, dw, _ = m.silu_mul_backward(dh, src, w)
        assert torch.equal(a.grad, dgu) and torch.equal(b.grad, dw)
    a = gate_up.clone().requires_grad_()
    m.silu_mul(a).backward(dh[:, :1].expand(R, I))  # a gradient without memory of its own
    assert torch.equal(a.grad, m.silu_mul_backward(dh[:, :1].expand(R, I).contiguous(), gate_up)[0])
    a = gate_up.clone().requires_grad_()
    g, = torch.autograd.grad(m.silu_mul(a).float().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.float().sum().backward()
    for call in (lambda t: m.restore_rows8(m.save_rows8(t)), lambda t: m.silu_mul_rows8(t)[0]):
        a = gate_up.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="not differentiable"):
            call(a).float().sum().backward()


def test_differences(cuda_device):
    """(L(x + e v) - L(x - e v)) / 2e along the gradient's direction v against the gradient's norm, in fp16: h's rounding is
    random, 2^-12 of L's terms, sqrt(R I) of them over e = 0.5; the third-order term is e^2 / 6 of order one: 5 %."""
    R, I = 64, 512
    gate_up, dh = randn(12, R, 2 * I, dtype=F16), randn(13, R, I, dtype=F16)
    dgu = m.silu_mul_backward(dh, gate_up)[0].double()
    v = dgu / dgu.norm() * 0.05 * gate_up.double().norm()

    def loss(sign):
        x = (gate_up.double() + sign * v).half()
        return float((m.silu_mul(x).double() * dh.double()).sum()), x.double()

    (up, xu), (down, xd) = loss(1), loss(-1)
    want = float((dgu * (xu - xd)).sum())
    assert abs(up - down - want) <= 0.05 * abs(want), (up - down, want)


def test_empty_streams_and_graph(cuda_device):
    e = torch.empty(0, 64, dtype=BF16, device="cuda")
    h, saved = m.silu_mul_rows8(e)
    assert h.shape == (0, 32) and m.restore_rows8(saved).shape == (0, 64)
    dgu, dw, h = m.silu_mul_backward(h, saved, torch.empty(0, device="cuda"))
    assert dgu.shape == (0, 64) and dw.shape == (0,)
    assert m.restore_rows8(m.save_rows8(e), torch.zeros(3, dtype=torch.int32, device="cuda")).eq(0).all()
    gate_up, dh, w = randn(14, 40, 400, dtype=BF16), randn(15, 40, 200, dtype=BF16), randn(16, 40)

    def step():
        h, saved = m.silu_mul_rows8(gate_up, w)
        return (h, *m.silu_mul_backward(dh, saved, w), m.restore_rows8(saved))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    gate_up.mul_(-1)
    w.mul_(0.5)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals(cuda_device):
    x, dh = randn(17, 4, 64, dtype=BF16), randn(18, 4, 32, dtype=BF16)
    saved = m.save_rows8(x)
    for call, msg in (
        (lambda: m.save_rows8(x.float()), "fp16 or bf16"),
        (lambda: m.save_rows8(x, torch.uint8), "q_dtype"),
        (lambda: m.save_rows8(x, parts=3), "parts"),
        (lambda: m.save_rows8(x.t()), "contiguous"),
        (lambda: m.save_rows8(x.cpu()), "CUDA"),
        (lambda: m.silu_mul(x[:, :63]), "2 I"),
        (lambda: m.silu_mul(x, torch.ones(5, device="cuda")), "row_weights"),
        (lambda: m.silu_mul(x, torch.ones(4)), "row_weights"),
        (lambda: m.silu_mul(x, save=torch.float32), "save"),
        (lambda: m.silu_mul_backward(dh, saved), "parts"),
        (lambda: m.silu_mul_backward(dh.half(), x), "dtype"),
        (lambda: m.silu_mul_backward(dh[:, :16], x), "twice"),
        (lambda: m.restore_rows8(saved, torch.zeros(3, device="cuda")), "index"),
        (lambda: m.restore_rows8(saved, out=torch.empty(4, 63, dtype=BF16, device="cuda")), "out"),
        (lambda: m.restore_rows8(saved, out=saved.q.view(-1)[:256].view(BF16).view(2, 64)), "out"),
        (lambda: m.Rows8(saved.q, saved.scale[:, :0], BF16), "scale"),
        (lambda: m.Rows8(saved.q.float(), saved.scale, BF16), "q must"),
    ):
        with pytest.raises(ValueError, match=msg):
            call()

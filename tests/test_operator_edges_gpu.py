"""GPU: edges of the norm, routing and 4-bit operators that their own test files leave out."""
import pytest
import torch

import muxi_race_b200 as m
from oracle.norm_ref import rms_norm_ref
from oracle.w4_ref import experts_ref, linear_ref, w4_values_ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e} over"


def test_w4_linear_refuses_an_output_over_its_rows(cuda_device):
    w = m.quantize_w4(randn(1, 256, 256, dtype=F16))
    big = randn(2, 8, 600, dtype=F16)
    x = big[:, :256]
    ref = m.w4_linear(x, w)
    for out in (x, big[:, 8:264], big[:, 255:511]):
        with pytest.raises(ValueError, match="share memory"):
            m.w4_linear(x, w, out=out)
    beside = big[:, 256:512]  # other columns of the same rows
    kept = x.clone()
    assert torch.equal(m.w4_linear(x, w, out=beside), ref) and torch.equal(x, kept)


def test_norm_refuses_outputs_over_other_rows(cuda_device):
    """Row t + 1 of x at the place of row t of the output: a row would be written while another reads it."""
    T, H = 64, 256
    big = randn(3, T + 1, H + 32, dtype=F16)
    w, res = randn(4, H, dtype=F16), randn(5, T, H, dtype=F16)
    x = big[1:, :H]
    y, h = m.add_rms_norm(x, w, res)
    for name in ("out", "residual_out"):
        for t in (big[:-1, :H], big[1:, 8:8 + H]):
            with pytest.raises(ValueError, match="share no memory"):
                m.add_rms_norm(x, w, res, **{name: t})
    with pytest.raises(ValueError, match="share no memory"):
        m.add_rms_norm_quant(x, w, res, residual_out=big[:-1, :H])
    both = torch.empty_like(y)
    with pytest.raises(ValueError, match="out and residual_out"):
        m.add_rms_norm(x, w, res, out=both, residual_out=both)
    # x and residual themselves stay allowed, each for either output, and other columns of the same rows
    x1, r1 = x.clone(), res.clone()
    m.add_rms_norm(x1, w, r1, out=r1, residual_out=x1)
    assert torch.equal(r1, y) and torch.equal(x1, h)
    wide = randn(6, T, 3 * H, dtype=F16)
    wide[:, :H], wide[:, H:2 * H] = x, res
    m.add_rms_norm(wide[:, :H], w, wide[:, H:2 * H], out=wide[:, 2 * H:], residual_out=wide[:, H:2 * H])
    assert torch.equal(wide[:, 2 * H:], y) and torch.equal(wide[:, H:2 * H], h) and torch.equal(wide[:, :H], x)


U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -25, BF16: 0.0}
F32 = 5e-6  # of the sum of |x| |W|, as derived in test_w4_gpu.py: the products are of exact q - z


def w4_random(seed, N, K, group, zeros, dtype):
    g = torch.Generator(device="cpu").manual_seed(seed)
    G = -(-K // group)
    v = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    s = ((torch.rand((N, G), generator=g) + 0.5) * 0.2 * K ** -0.5).to(dtype)
    z = torch.randint(0, 16, (N, G), generator=g, dtype=torch.uint8) if zeros else None
    return v, s, z


def w4_packed(v, s, z, group):
    """(the package's weights, their values in fp64) of codes v [N, K]."""
    N, K = v.shape
    v = torch.nn.functional.pad(v, (0, K % 2))
    q = (v[:, 0::2] | v[:, 1::2] << 4).contiguous().cuda()
    s, z = s.cuda(), None if z is None else z.cuda()
    return (m.pack_w4(q, s, z, in_features=K, group_size=group), w4_values_ref(q, s, z, K, group))


@pytest.mark.parametrize("M", [1, 8, 11, 16, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size,outlier", [(0.1, 1e4), (0.01, 2000.0), (1e-3, 6e4)])
def test_w4_outliers_where_the_weight_is_zero(cuda_device, M, group, zeros, dtype, size, outlier):
    """A few channels of x far above the others, whose codes are the zero point: they add exactly nothing."""
    N, K = 70, 700
    v, s, z = w4_random(7, N, K, group, zeros, dtype)
    x = randn(8, M, K, scale=size)
    for c in (3, 77, 130, 131, 400, 699):
        v[:, c] = 8 if z is None else z[:, c // group]
        x[:, c] = outlier * (1 if c % 2 else -0.7)
    w, values = w4_packed(v, s, z, group)
    x = x.to(dtype)
    ref, mag = linear_ref(x, values)
    assert float(mag.amax()) < 100 * size  # the outliers are in no term
    within(m.w4_linear(x, w), ref, U[dtype] * ref.abs() + F32 * mag + TINY[dtype], "y")
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
def test_w4_infinities_keep_their_sign(cuda_device, dtype, zeros):
    """An infinite value makes a sum infinite with the sign of its weight, and NaN where that is 0."""
    v, s, z = w4_random(9, 96, 300, 32, zeros, dtype)
    w, values = w4_packed(v, s, z, 32)
    x = randn(10, 12, 300).to(dtype)
    x[2, 5], x[7, 250], x[9, 0], x[9, 299] = float("inf"), float("-inf"), float("inf"), float("inf")
    y, ref = m.w4_linear(x, w).double(), x.double() @ values.mT
    spoilt = [2, 7, 9]
    assert torch.equal(y[spoilt].nan_to_num(nan=1e9), ref[spoilt].nan_to_num(nan=1e9)) and bool(ref[2].isinf().any())
    fine = [i for i in range(12) if i not in spoilt]
    within(y[fine], ref[fine], U[dtype] * ref[fine].abs() + F32 * (x.double().abs() @ values.abs().mT)[fine] + TINY[dtype], "y")


def sigmoid_grad64(l, ids, dw, scale):
    x = l.double().requires_grad_()
    s = torch.sigmoid(x).gather(1, ids.long())
    p = s / s.sum(-1, keepdim=True)
    (p * dw.double() * scale).sum().backward()
    p, g = p.detach(), dw.double().abs() * scale
    return x.grad, torch.zeros_like(x.grad).scatter_add_(1, ids.long(), p * (g + (g * p).sum(-1, keepdim=True)))


@pytest.mark.parametrize("size", [1.0, 100.0, 65536.0])
def test_route_gradient_of_far_sigmoids(cuda_device, size):
    """Renormalised sigmoid, every chosen logit far below 0 (a masked row, or a training that ran off) and
    large gradients. While the scores are numbers of fp32 (above -88) the gradient is the formula's; below,
    where every score and weight is 0, it is 0. W = 5e-6 as derived in test_route_topk_gpu.py; a subnormal
    score adds half its spacing, 2e-7 of it at -88.5."""
    T, E, k = 60, 16, 4
    l = randn(20, T, E, scale=0.3) - torch.linspace(60, 88, T).cuda()[:, None]
    l = l.clamp_min(-88.5)
    dw = randn(21, T, k, scale=size)
    _, ids = m.route_topk(l, k, scoring="sigmoid")
    got = m.route_topk_backward(dw, l, ids, scoring="sigmoid", scale=2.5)
    ref, mag = sigmoid_grad64(l, ids, dw, 2.5)
    within(got, ref, 4 * 5e-6 * mag + 1e-37, "dlogits")
    for far in (-100.0, -1e4):
        l = torch.full((8, E), far, device="cuda")
        l[4:] += randn(22, 4, E)
        _, ids = m.route_topk(l, k, scoring="sigmoid")
        got = m.route_topk_backward(dw[:8], l, ids, scoring="sigmoid", scale=2.5)
        assert bool((got == 0).all())
    l = torch.tensor([[-87.0, -88.0]], device="cuda")
    got = m.route_topk_backward(torch.tensor([[100.0, 1.0]], device="cuda"), l, torch.tensor([[0, 1]], device="cuda", dtype=torch.int32),
                                scoring="sigmoid")
    p = 1 / (1 + 2.718281828459045 ** -1)
    want = p * (100 - 100 * p - (1 - p))
    within(got, torch.tensor([[want, -want]], dtype=torch.float64, device="cuda"), 4 * 5e-6 * 200, "dlogits")


def test_route_weights_of_far_sigmoids_add_up_to_one(cuda_device):
    """Scores down to fp32's subnormal numbers (logits to -88.5, whose sum is below 1e-37) are divided by their
    own sum."""
    T, E, k = 100, 24, 5
    l = (randn(30, T, E, scale=0.2) - torch.linspace(20, 88, T).cuda()[:, None]).clamp_min(-88.5)
    w, ids = m.route_topk(l, k, scoring="sigmoid")
    s = torch.sigmoid(l.double()).gather(1, ids.long())
    ref = s / s.sum(-1, keepdim=True)
    within(w, ref, 5e-6 * ref, "weights")
    within(w.double().sum(-1), torch.ones(T, dtype=torch.float64, device="cuda"), 5e-6, "sum")


def test_second_derivatives_raise(cuda_device):
    x, w, l = randn(40, 4, 64).requires_grad_(), randn(41, 64).requires_grad_(), randn(42, 4, 16).requires_grad_()
    for leaf, loss in ((x, lambda: m.add_rms_norm(x, w).sum()), (w, lambda: m.add_rms_norm(x, w, x)[0].square().sum()),
                       (l, lambda: m.route_topk(l, 3)[0][:, 0].sum()), (l, lambda: m.route_topk(l, 3, "sigmoid")[0].square().sum())):
        plain, = torch.autograd.grad(loss(), leaf)
        g, = torch.autograd.grad(loss(), leaf, create_graph=True)
        assert torch.equal(g.detach(), plain)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(g.square().sum(), leaf)


@pytest.mark.parametrize("q_dtype,kmax", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("T,H", [(3, 64), (3, 100), (5, 4096), (400, 7168), (400, 999)])
@pytest.mark.parametrize("size", [1e-36, 1e-37, 1e-38, 1e-41, 1e-44])
def test_quant_of_tiny_rows(cuda_device, q_dtype, kmax, T, H, size):
    """Rows whose largest |y| is near or below fp32's least normal number, with zeros in them. Bounds as in
    test_norm_gpu.py, with half a spacing of the subnormal numbers (2^-150) for y and, times a code of up to
    kmax, for the scale."""
    x, w = randn(50, T, H, dtype=F16), randn(51, H, scale=size)
    x[:, ::7] = 0
    x[0] = 0
    q, scale, _ = m.add_rms_norm_quant(x, w, q_dtype=q_dtype)
    codes = q.float().double()
    assert bool(codes.isfinite().all()) and bool((codes[:, ::7] == 0).all()) and bool((codes[0] == 0).all())
    y, _ = rms_norm_ref(x, w)
    rscale, tiny = y.abs().amax(-1) / kmax, 2.0 ** -150
    within(scale, rscale, 8e-6 * rscale + 2 * tiny, "scale")
    s = rscale[:, None]
    step = 0.5 * s if q_dtype == torch.int8 else torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10)
    within(codes * scale.double()[:, None], y, step + 1.6e-5 * (y.abs() + s * kmax) + (kmax + 2) * tiny, "q * scale")
    if size >= 1e-37:  # the largest value of a row still has the largest code
        assert bool((codes[1:].abs().amax(-1) == kmax).all())


@pytest.mark.parametrize("kind,kmax", [("int8", 127.0), ("fp8", 448.0)])
@pytest.mark.parametrize("size", [1e-36, 1e-37, 1e-38, 3e-40])
def test_quantised_tiny_rows(cuda_device, kind, kmax, size):
    """The same at the quantisation of 16-bit rows, by itself and inside the experts' calls (bf16: fp16 has no
    values this small). Bounds: half a step, and half a spacing of fp32's subnormal numbers for the scale."""
    quantize, fused = {"int8": (m.quantize_rows_int8, m.fused_moe_int8), "fp8": (m.quantize_rows_fp8, m.fused_moe_fp8)}[kind]
    x = randn(52, 20, 256, dtype=BF16, scale=size)
    x[:, ::5] = 0
    q, scale = quantize(x)
    codes, y = q.float().double(), x.double()
    assert bool(codes.isfinite().all()) and bool((codes[:, ::5] == 0).all())
    s = y.abs().amax(-1, keepdim=True) / kmax
    step = 0.5 * s if kind == "int8" else torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10)
    within(codes * scale.double()[:, None], y, step + 1e-6 * s * kmax + kmax * 2.0 ** -150, "q * scale")
    w13, w2 = quantize(randn(53, 4, 256, 256, dtype=BF16)), quantize(randn(54, 4, 256, 128, dtype=BF16))
    ids = torch.arange(20, device="cuda", dtype=torch.int32)[:, None] % 4
    out = fused(x, *w13, *w2, ids, torch.ones(20, 1, device="cuda"))
    assert bool((out == 0).all())  # silu(gate) * up is below the least bf16 number
    assert m.device_status() == 0


@pytest.mark.parametrize("groups", [(32, 128), (128, 32)])
def test_one_w13_with_w2_of_other_groups(cuda_device, groups):
    """At I = 5632 and 16 rows a tile, w2 in groups of 128 takes two slices of K and in groups of 32 one: each
    call asks for its own workspace."""
    T, H, I, E, k = 16, 64, 5632, 4, 2
    size = m._lib.lib().moe_fused_w4_workspace_bytes
    assert size(T, k, E, H, I, 64, 32, m._lib.MOE_F16) != size(T, k, E, H, I, 64, 128, m._lib.MOE_F16)

    def experts(seed, N, K, group, gate_up):  # (packed, values in fp64) of E matrices
        g = torch.Generator(device="cpu").manual_seed(seed)
        q = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=torch.uint8).cuda()
        s = ((torch.rand((E, N, -(-K // group)), generator=g) + 0.5) * 0.2 * K ** -0.5).half().cuda()
        return m.pack_w4(q, s, group_size=group, gate_up=gate_up), w4_values_ref(q, s, None, K, group)

    q13, w13 = experts(60, 2 * I, H, 64, True)
    x = randn(62, T, H, dtype=F16)
    ids = torch.stack([torch.arange(T) % E, (torch.arange(T) + 1) % E], 1).int().cuda()
    weights = torch.full((T, k), 0.5, device="cuda")
    for group in groups:
        q2, w2 = experts(61, H, I, group, False)
        ref, tol = experts_ref(x, w13, w2, ids, weights, U[F16], F32)
        within(m.fused_moe_w4(x, q13, q2, ids, weights), ref, tol + TINY[F16], "out")
    assert m.device_status() == 0


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_out_dtype_is_refused_where_it_has_no_effect(cuda_device, kind):
    quantize, fused = {"int8": (m.quantize_rows_int8, m.fused_moe_int8), "fp8": (m.quantize_rows_fp8, m.fused_moe_fp8)}[kind]
    x = randn(70, 6, 256, dtype=F16)
    w = (*quantize(randn(71, 4, 256, 256, dtype=F16, scale=0.06)), *quantize(randn(72, 4, 256, 128, dtype=F16, scale=0.09)))
    ids, tw = torch.arange(6, device="cuda", dtype=torch.int32)[:, None] % 4, torch.ones(6, 1, device="cuda")
    for dtype in (F16, BF16):
        with pytest.raises(ValueError, match="needs hidden_scale"):
            fused(x, *w, ids, tw, out_dtype=dtype)
    q, scale = quantize(x)
    want = fused(x, *w, ids, tw)
    assert want.dtype == F16
    with pytest.raises(ValueError, match="out_dtype"):
        fused(q, *w, ids, tw, out=torch.empty_like(x), hidden_scale=scale, out_dtype=BF16)
    assert fused(q, *w, ids, tw, hidden_scale=scale).dtype == BF16
    out = torch.empty_like(x)
    assert fused(q, *w, ids, tw, out=out, hidden_scale=scale) is out and torch.equal(out, want)  # one route a token
    assert torch.equal(fused(q, *w, ids, tw, hidden_scale=scale, out_dtype=F16), want)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_w4_quantise_shows_spoilt_groups(cuda_device, symmetric, dtype):
    """NaN or an infinity spoils its group of 32 and leaves the others as they are."""
    w = randn(80, 6, 200, dtype=dtype)
    want = m.dequantize_w4(m.quantize_w4(w, 32, symmetric))
    bad = torch.zeros_like(w, dtype=torch.bool)
    for r, c, v in ((0, 5, "nan"), (1, 64, "inf"), (2, 199, "-inf"), (4, 40, "nan"), (4, 41, "inf")):
        w[r, c] = float(v)
        bad[r, c // 32 * 32:c // 32 * 32 + 32] = True
    got = m.dequantize_w4(m.quantize_w4(w, 32, symmetric))
    assert not bool(got[bad].isfinite().any())
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("size", [1e38, 1e-37, 1e-38, 1e-39])
def test_w4_quantise_the_ends_of_the_range(cuda_device, symmetric, size):
    """bf16 weights near fp32's largest and least numbers: the bound of test_w4_gpu.py, and where the scale is
    subnormal half its spacing (2^-134) for each of up to 8 (15) steps."""
    w = randn(81, 4, 256).clamp(-3, 3)
    w[:, ::9] = 0
    w = (w * size).to(BF16)
    d = m.dequantize_w4(m.quantize_w4(w, 64, symmetric)).double()
    groups = w.double().view(4, 4, 64)
    span = groups.abs().amax(-1) / 7 if symmetric else (groups.amax(-1).clamp_min(0) - groups.amin(-1).clamp_max(0)) / 15
    step = span.repeat_interleave(64, -1)
    within(d, w.double(), step * (0.5 if symmetric else 1.0) * 1.01 + 16 * U[BF16] * step + 16 * 2.0 ** -134, "weight")
    assert bool((d[:, ::9] == 0).all())


def test_operators_without_a_gradient_say_so(cuda_device):
    """A loss that also has another path to x: the operator's part is not left out in silence."""
    x, norm = randn(90, 4, 64, dtype=F16), randn(91, 64, dtype=F16)
    lin, w13, w2 = (m.quantize_w4(randn(s, *shape, dtype=F16), 32, gate_up=g)
                    for s, shape, g in ((92, (64, 64), False), (93, (4, 64, 64), True), (94, (4, 64, 32), False)))
    ids, tw = torch.zeros(4, 1, device="cuda", dtype=torch.int32), torch.ones(4, 1, device="cuda")
    calls = (("w4_linear", lambda x, t: m.w4_linear(x, lin)), ("fused_moe_w4", lambda x, t: m.fused_moe_w4(x, w13, w2, ids, t)),
             ("add_rms_norm_quant", lambda x, t: m.add_rms_norm_quant(x, norm, x)[1]),
             ("add_rms_norm_quant", lambda x, t: m.add_rms_norm_quant(x, norm, x)[2]))
    for name, call in calls:
        plain = call(x, tw)
        assert not plain.requires_grad
        leaf = x.clone().requires_grad_()
        y = call(leaf, tw)
        assert torch.equal(y.detach(), plain)
        with pytest.raises(RuntimeError, match=f"{name} is not differentiable"):
            (y.float().sum() + leaf.float().sum()).backward()
        with torch.no_grad():
            assert not call(leaf, tw).requires_grad
    t = tw.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="fused_moe_w4 is not differentiable"):
        (m.fused_moe_w4(x, w13, w2, ids, t).float().sum() + t.sum()).backward()
    out = torch.empty_like(x)
    assert m.w4_linear(x.clone().requires_grad_(), lin, out=out) is out and not out.requires_grad


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_w4_zero_points_of_16(cuda_device, group, dtype):
    """Checkpoints that store z - 1 in 4 bits have zero points up to 16."""
    v, s, z = w4_random(95, 70, 300, group, True, dtype)
    z[::2] = 16
    w, values = w4_packed(v, s, z, group)
    assert torch.equal(m.dequantize_w4(w), values.to(dtype))
    for M in (1, 11):
        x = randn(96, M, 300).to(dtype)
        ref, mag = linear_ref(x, values)
        within(m.w4_linear(x, w), ref, U[dtype] * ref.abs() + F32 * mag + TINY[dtype], "y")
    z[3, 0] = 17
    with pytest.raises(ValueError, match="zeros must be in 0..16"):
        w4_packed(v, s, z, group)
    assert m.device_status() == 0

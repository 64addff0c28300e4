"""GPU: 4-bit weights (layout, quantisation) and their products against fp64.

Tolerances: u = half a unit in the last place of the output type (2^-11 fp16, 2^-8 bf16) for the final
rounding. The products q - z are exact; a sum is at most 8 tensor instructions per group of 128 (whose
accumulation may truncate, 2^-23), then at most 16 groups of a warp and 8 warps: 32 steps, so an error
below 32 * 2^-23 = 3.8e-6 of the sum of the terms' magnitudes: F32 = 5e-6 with the scaling products.
(A plan may give one warp all of a long K, 128 steps of 2^-24 at K = 16384, whose rounding errors are of
either sign and stay far below their bound.)
"""
import pytest
import torch

from muxi_race_b200 import dequantize_w4, device_status, fused_moe_w4, pack_w4, quantize_w4, w4_linear
from oracle.w4_ref import experts_ref, linear_ref, w4_values_ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -25, BF16: 0.0}
F32 = 5e-6


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def w4_inputs(seed, lead, N, K, group, zeros, dtype):
    g = gen(seed)
    G = -(-K // group)
    q = torch.randint(0, 256, (*lead, N, (K + 1) // 2), generator=g, dtype=torch.uint8).cuda()
    s = ((torch.rand((*lead, N, G), generator=g) + 0.5) * 0.2 * K ** -0.5).to(dtype).cuda()
    z = torch.randint(0, 16, (*lead, N, G), generator=g, dtype=torch.uint8).cuda() if zeros else None
    return q, s, z


def randn(seed, *shape, dtype):
    return torch.randn(shape, generator=gen(seed)).to(dtype).cuda()


def within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e} over"


@pytest.mark.parametrize("N,K", [(16, 128), (1, 1), (17, 100), (100, 257), (64, 4096), (40, 130)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_layout_round_trip(cuda_device, N, K, group, zeros, dtype):
    """Unpacking gives every weight back, to its one rounding."""
    for lead, gate_up in (((), False), ((3,), False), ((2,), True)):
        if gate_up and N % 2:
            continue
        q, s, z = w4_inputs(1, lead, N, K, group, zeros, dtype)
        w = pack_w4(q, s, z, in_features=K, group_size=group, gate_up=gate_up)
        assert w.shape == (*lead, N, K)
        assert torch.equal(dequantize_w4(w), w4_values_ref(q, s, z, K, group).to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize(cuda_device, dtype, group, symmetric):
    """No weight is further than half a step from its value (symmetric: 7 steps reach amax; otherwise
    15 steps span the range, and the rounding of the zero point may cost another half)."""
    w = randn(2, 3, 50, 333, dtype=dtype)
    w[0, 0] = 0  # a row of zeros stays zero
    d = dequantize_w4(quantize_w4(w, group, symmetric)).double()
    pad = torch.nn.functional.pad(w.double(), (0, -333 % group)).view(3, 50, -1, group)
    span = pad.abs().amax(-1) / 7 if symmetric else (pad.amax(-1).clamp_min(0) - pad.amin(-1).clamp_max(0)) / 15
    step = span.repeat_interleave(group, -1)[..., :333]
    within(d, w.double(), step * (0.5 if symmetric else 1.0) * 1.01 + 16 * U[dtype] * step, "weight")
    assert bool((d[0, 0] == 0).all())


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 24, 32, 33, 70])
@pytest.mark.parametrize("N,K", [(16, 64), (33, 200), (130, 600), (256, 1024), (200, 2000), (48, 7168)])
@pytest.mark.parametrize("group,zeros", [(128, False), (32, True), (64, False)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear(cuda_device, M, N, K, group, zeros, dtype):
    q, s, z = w4_inputs(3, (), N, K, group, zeros, dtype)
    x = randn(4, M, K, dtype=dtype)
    y = w4_linear(x, pack_w4(q, s, z, in_features=K, group_size=group))
    ref, mag = linear_ref(x, w4_values_ref(q, s, z, K, group))
    within(y, ref, U[dtype] * ref.abs() + F32 * mag + TINY[dtype], "y")
    assert device_status() == 0


@pytest.mark.parametrize("K", [99, 1001, 4096, 16384])
def test_linear_strides_and_odd_sizes(cuda_device, K):
    """Rows inside a wider tensor at odd and at 16-byte starts, one row for all, a wider output."""
    N = 77
    q, s, z = w4_inputs(5, (), N, K, 64, True, F16)
    w = pack_w4(q, s, z, in_features=K, group_size=64)
    values = w4_values_ref(q, s, z, K, 64)
    big = randn(6, 12, K + 16, dtype=F16)
    for x in (big[:, 3:3 + K], big[:, 8:8 + K], big[:1, :K].expand(12, K), big[:, :K].reshape(3, 4, K)):
        ref, mag = linear_ref(x, values)
        tol = U[F16] * ref.abs() + F32 * mag + TINY[F16]
        within(w4_linear(x, w), ref, tol, "y")
        out = torch.full((12, N + 9), 7.0, device="cuda", dtype=F16)
        if x.dim() == 2:
            w4_linear(x, w, out=out[:, 1:1 + N])
            within(out[:, 1:1 + N], ref, tol, "out")
            assert bool((out[:, 0] == 7).all()) and bool((out[:, 1 + N:] == 7).all())


def moe_case(seed, T, H, I, E, k, group, zeros, dtype, skew=False):
    q13 = w4_inputs(seed, (E,), 2 * I, H, group, zeros, dtype)
    q2 = w4_inputs(seed + 1, (E,), H, I, group, zeros, dtype)
    x = randn(seed + 2, T, H, dtype=dtype)
    scores = torch.randn(T, E, generator=gen(seed + 3))
    if skew:
        scores[:, 0] += 10  # every token chooses expert 0
    w, ids = torch.softmax(scores, -1).topk(k, -1)
    return q13, q2, x, ids.int().cuda(), w.cuda()


def run_moe(q13, q2, x, ids, w, group):
    H, I = x.shape[1], q13[0].shape[1] // 2
    w13 = pack_w4(*q13, in_features=H, group_size=group, gate_up=True)
    w2 = pack_w4(*q2, in_features=I, group_size=group)
    out = fused_moe_w4(x, w13, w2, ids, w)
    ref, tol = experts_ref(x, w4_values_ref(*q13, H, group), w4_values_ref(*q2, I, group), ids, w, U[x.dtype], F32)
    within(out, ref, tol + TINY[x.dtype], "out")
    assert torch.equal(out, fused_moe_w4(x, w13, w2, ids, w)), "not the same bits on a second run"
    assert device_status() == 0
    return out


@pytest.mark.parametrize("T", [1, 2, 5, 16, 33, 128])
@pytest.mark.parametrize("H,I,E,k", [(256, 128, 8, 2), (1024, 512, 8, 2), (200, 36, 5, 3), (512, 1000, 60, 4),
                                     (7168, 64, 16, 8)])
@pytest.mark.parametrize("group,zeros,dtype", [(128, False, F16), (32, True, BF16), (64, True, F16)])
def test_experts(cuda_device, T, H, I, E, k, group, zeros, dtype):
    run_moe(*moe_case(10, T, H, I, E, k, group, zeros, dtype), group)


@pytest.mark.parametrize("T", [7, 100, 300])
def test_experts_with_uneven_loads(cuda_device, T):
    """One expert gets a route of every token (tiles of 32, an uneven last one), others few or none."""
    run_moe(*moe_case(20, T, 384, 200, 40, 2, 128, False, BF16, skew=True), 128)


@pytest.mark.parametrize("T,H,I,E,k", [(100, 96, 40, 600, 8), (60, 130, 70, 1000, 4), (250, 64, 16, 700, 8), (9, 1024, 300, 900, 8)])
@pytest.mark.parametrize("group,zeros,dtype", [(128, False, F16), (64, True, BF16), (32, True, F16)])
def test_many_experts_of_few_tokens(cuda_device, T, H, I, E, k, group, zeros, dtype):
    """A CTA's strips belong to many experts of one to a few tokens each, whose rows it holds together."""
    run_moe(*moe_case(25, T, H, I, E, k, group, zeros, dtype), group)


def test_experts_ids(cuda_device):
    """Skipped ids, a token without any expert, an expert twice in a token, int64 ids, 16-bit weights,
    rows at odd starts."""
    q13, q2, x, ids, w = moe_case(30, 40, 264, 136, 16, 4, 64, True, F16)
    ids[3] = -1
    ids[4, 1] = 16
    ids[5, 2] = -7
    ids[6, 1] = ids[6, 0]
    wide = torch.zeros(40, 264 + 13, device="cuda", dtype=F16)
    wide[:, 5:5 + 264] = x
    wide_x = wide[:, 5:5 + 264]
    a = run_moe(q13, q2, x, ids, w, 64)
    assert bool((a[3] == 0).all())
    assert torch.equal(a, run_moe(q13, q2, wide_x, ids, w, 64))
    ids64 = ids.long()
    ids64[4, 1] = 2 ** 40 + 1
    assert torch.equal(a, run_moe(q13, q2, x, ids64, w, 64))
    run_moe(q13, q2, x, ids, w.half(), 64)
    run_moe(q13, q2, x, torch.full_like(ids, -1), w, 64)


def test_spoilt_rows_stay_alone(cuda_device):
    """NaN or infinity in one row of x changes that row only."""
    q, s, z = w4_inputs(40, (), 64, 1024, 128, False, F16)
    w = pack_w4(q, s, z)
    x = randn(41, 20, 1024, dtype=F16)
    y = w4_linear(x, w)
    x2 = x.clone()
    x2[3, 100], x2[11, 7] = float("nan"), float("inf")
    y2 = w4_linear(x2, w)
    assert bool(y2[3].isnan().all()) and not bool(y2[11].isfinite().any())
    keep = [i for i in range(20) if i not in (3, 11)]
    assert torch.equal(y[keep], y2[keep])


@pytest.mark.parametrize("group,zeros", [(128, False), (32, True)])
def test_bf16_rows_of_any_range(cuda_device, group, zeros):
    """Tiny and huge rows (1e37: the products of whole numbers would overflow fp32), rows of zeros and of
    subnormal values, values of any size in one row; NaN and infinity stay in their row."""
    M, N, K = 14, 50, 700
    q, s, z = w4_inputs(42, (), N, K, group, zeros, BF16)
    w, values = pack_w4(q, s, z, in_features=K, group_size=group), w4_values_ref(q, s, z, K, group)
    x = torch.randn(M, K, generator=gen(43))
    scale = torch.tensor([1e-30, 1e30, 0.0, 1e-39, 1, 1e-6, 3e4, 1e37, 1e-20, 1, 1, 1, 1, 1])
    x = x * scale[:, None]
    x[9] *= 2.0 ** torch.randint(-30, 1, (K,), generator=gen(44))
    x[9, 5] = 4.0
    x = x.to(BF16).cuda()
    x[11, 3], x[12, 4] = float("nan"), float("-inf")
    y = w4_linear(x, w)
    fine = [i for i in range(M) if i not in (11, 12)]
    ref, mag = linear_ref(x[fine], values)
    tiny = 2.0 ** -133  # subnormal results and products are not part of the bound
    within(y[fine], ref, U[BF16] * ref.abs() + F32 * mag + tiny, "y")
    assert bool(y[11].isnan().all()) and not bool(y[12].isfinite().any())
    assert device_status() == 0


def test_empty_and_other_stream(cuda_device):
    q13, q2, x, ids, w = moe_case(50, 9, 256, 128, 8, 2, 128, False, F16)
    w13, w2 = pack_w4(*q13, group_size=128, gate_up=True), pack_w4(*q2, group_size=128)
    assert fused_moe_w4(x[:0], w13, w2, ids[:0], w[:0]).shape == (0, 256)
    q, s, _ = w4_inputs(51, (), 32, 64, 32, False, F16)
    lin = pack_w4(q, s, group_size=32)
    assert w4_linear(x[:0, :64], lin).shape == (0, 32)
    ref = fused_moe_w4(x, w13, w2, ids, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [fused_moe_w4(x, w13, w2, ids, w) for _ in range(20)]
    here = [fused_moe_w4(x, w13, w2, ids, w) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(ref, t) for t in got + here)


def test_graph_replay(cuda_device):
    """The calls can be captured, and a replay reads the inputs as they are then."""
    q13, q2, x, ids, w = moe_case(60, 6, 256, 128, 8, 2, 128, False, F16)
    w13, w2 = pack_w4(*q13, group_size=128, gate_up=True), pack_w4(*q2, group_size=128)
    fused_moe_w4(x, w13, w2, ids, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_moe_w4(x, w13, w2, ids, w)
    x.copy_(randn(61, 6, 256, dtype=F16))
    ids.copy_((ids + 3) % 8)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, fused_moe_w4(x, w13, w2, ids, w))


def test_refusals(cuda_device):
    q, s, z = w4_inputs(70, (), 32, 128, 64, True, F16)
    w = pack_w4(q, s, z, group_size=64)
    x = randn(71, 4, 128, dtype=F16)
    with pytest.raises(ValueError, match="group_size"):
        pack_w4(q, s, z, group_size=48)
    with pytest.raises(ValueError, match="scales"):
        pack_w4(q, s[:, :1], z, group_size=64)
    with pytest.raises(ValueError, match="zeros"):
        pack_w4(q, s, z.int(), group_size=64)
    with pytest.raises(ValueError, match="in_features"):
        pack_w4(q, s, z, in_features=126, group_size=64)
    with pytest.raises(ValueError, match="even number of rows"):
        pack_w4(q[:31].contiguous(), s[:31].contiguous(), z[:31].contiguous(), group_size=64, gate_up=True)
    with pytest.raises(ValueError, match="x must be"):
        w4_linear(x.bfloat16(), w)
    with pytest.raises(ValueError, match="x must be"):
        w4_linear(x[:, :64], w)
    with pytest.raises(ValueError, match="CUDA"):
        w4_linear(x.cpu(), w)
    with pytest.raises(ValueError, match="without gate_up"):
        w4_linear(x, pack_w4(q, s, z, group_size=64, gate_up=True))
    q13, q2, x, ids, tw = moe_case(72, 4, 128, 64, 4, 2, 64, False, F16)
    w13, w2 = pack_w4(*q13, group_size=64, gate_up=True), pack_w4(*q2, group_size=64)
    with pytest.raises(ValueError, match="gate_up"):
        fused_moe_w4(x, w2, w13, ids, tw)
    with pytest.raises(ValueError, match="topk"):
        fused_moe_w4(x, w13, w2, ids[:2], tw[:2])
    with pytest.raises(ValueError, match="int32 or int64"):
        fused_moe_w4(x, w13, w2, ids.short(), tw)
    with pytest.raises(ValueError, match="hidden_states"):
        fused_moe_w4(x.bfloat16(), w13, w2, ids, tw)

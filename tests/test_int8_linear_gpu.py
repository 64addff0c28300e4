"""GPU: int8_linear against exact whole-number sums.

Tolerance: the sum is exact; its conversion, two factors and the bias are a rounding of 2^-24 each, of the product P = |sum| xs ws
(three) and of |P| + |bias| (one): 4 * 2^-24 (P + |bias|); then the output's rounding u.
"""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


def make(M, N, K, seed=0, low=-127):
    g = torch.Generator(device="cpu").manual_seed(seed)
    x, w = (torch.randint(low, 128, (r, K), generator=g, dtype=torch.int8).cuda() for r in (M, N))
    xs, ws = (torch.rand(r, generator=g).add_(0.1).mul_(K ** -0.5 / 40).cuda() for r in (M, N))
    return x, xs, w, ws, torch.randn(N, generator=g).cuda()


def check(y, x, xs, w, ws, bias):
    acc = x.double() @ w.double().T  # exact: below 2^53
    p = acc * xs.double()[:, None] * ws.double()
    b = torch.zeros_like(ws) if bias is None else bias
    ref = p + b.double()
    tol = U[y.dtype] * ref.abs() + (1 + U[y.dtype]) * 4 * 2.0 ** -24 * (p.abs() + b.double().abs()) + (2.0 ** -25 if y.dtype == F16 else 0)
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off"


SHAPES = [(1, 1, 16), (1, 17, 4096), (3, 100, 48), (8, 512, 1024), (9, 333, 2064), (16, 1000, 80), (17, 64, 4112), (32, 130, 176),
          (33, 257, 1024), (64, 1000, 7168), (100, 24, 14336), (129, 4096, 528), (256, 256, 128), (257, 513, 144), (300, 1, 64),
          (1000, 1100, 272), (2049, 520, 1040)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("with_bias", [False, True])
def test_products(cuda_device, M, N, K, out_dtype, with_bias):
    x, xs, w, ws, bias = make(M, N, K)
    bias = bias if with_bias else None
    y = m.int8_linear(x, xs, w, ws, bias, out_dtype=out_dtype)
    assert y.dtype == out_dtype and y.shape == (M, N)
    check(y, x, xs, w, ws, bias)
    assert torch.equal(y, m.int8_linear(x, xs, w, ws, bias, out_dtype=out_dtype))
    assert m.device_status() == 0


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_largest_sums(cuda_device, M):
    """All values -128 at the longest K: 2^14 K = 2147221504 fits 31 bits."""
    K = 131056
    x, w = (torch.full((r, K), -128, dtype=torch.int8, device="cuda") for r in (M, 40))
    ones = torch.ones(max(M, 40), device="cuda")
    y = m.int8_linear(x, ones[:M], w, ones[:40], out_dtype=F32)
    assert bool((y == float(torch.tensor(16384 * K, dtype=F32))).all())


@pytest.mark.parametrize("M", [5, 33, 260])
def test_strides_leading_dimensions_and_out(cuda_device, M):
    N, K = 264, 320
    x, xs, w, ws, bias = make(M, N, K + 64)
    x, w = x[:, 16:16 + K], w[:, :K].contiguous()
    y = m.int8_linear(x, xs, w, ws, bias)
    check(y, x, xs, w, ws, bias)
    for start, pitch in ((0, N + 8), (3, N + 7), (8, N + 8)):
        base = torch.full((M, pitch + 8), 3.0, dtype=BF16, device="cuda")
        out = base[:, start:start + N]
        assert m.int8_linear(x, xs, w, ws, bias, out=out) is out and torch.equal(out, y)
        out.fill_(3.0)
        assert bool((base == 3.0).all())
    x3, s3 = x.contiguous().view(1, M, K), xs.view(1, M)
    assert torch.equal(m.int8_linear(x3, s3, w, ws, bias), y.view(1, M, N))
    assert m.int8_linear(x[:0], xs[:0], w, ws).shape == (0, N)


def test_from_the_norm(cuda_device):
    """The rows that the norm writes, times weights of quantize_rows_int8: within the quantisation of the 16-bit product."""
    g = torch.Generator(device="cpu").manual_seed(1)
    x, w = torch.randn((40, 1024), generator=g).to(BF16).cuda(), (torch.randn((512, 1024), generator=g) / 32).to(BF16).cuda()
    nw = torch.ones(1024, dtype=BF16, device="cuda")
    q, scale, _ = m.add_rms_norm_quant(x, nw)
    wq, wscale = m.quantize_rows_int8(w)
    y = m.int8_linear(q, scale, wq, wscale)
    check(y, q, scale, wq, wscale.view(-1), None)
    assert torch.equal(m.int8_linear(*m.quantize_rows_int8(x), wq, wscale), m.int8_linear(*m.quantize_rows_int8(x), wq, wscale.view(-1)))


def test_stream_and_graph(cuda_device):
    for M in (4, 50, 400):
        x, xs, w, ws, bias = make(M, 300, 1024, seed=2)
        want = m.int8_linear(x, xs, w, ws, bias)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = [m.int8_linear(x, xs, w, ws, bias) for _ in range(3)]
        s.synchronize()
        assert all(torch.equal(t, want) for t in got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = m.int8_linear(x, xs, w, ws, bias)
            b = m.int8_linear(x, xs, w, ws)
        x.neg_()
        graph.replay()
        assert torch.equal(a, m.int8_linear(x, xs, w, ws, bias)) and torch.equal(b, m.int8_linear(x, xs, w, ws))


def test_refusals(cuda_device):
    x, xs, w, ws, bias = make(4, 64, 128)
    for call, msg in (
        (lambda: m.int8_linear(x.float(), xs, w, ws), "int8"),
        (lambda: m.int8_linear(x, xs, w.float(), ws), "int8"),
        (lambda: m.int8_linear(x[:, :112], xs, w, ws), "x must be"),
        (lambda: m.int8_linear(x, xs, w[:, :112], ws), "contiguous"),
        (lambda: m.int8_linear(x[:, :120].contiguous(), xs, w[:, :120].contiguous(), ws), "multiple of 16"),
        (lambda: m.int8_linear(make(4, 64, 136)[0][:, 8:], xs, w, ws), "16 bytes"),
        (lambda: m.int8_linear(x, xs[:3], w, ws), "x_scale"),
        (lambda: m.int8_linear(x, xs.half(), w, ws), "x_scale"),
        (lambda: m.int8_linear(x, xs, w, ws[:3]), "w_scale"),
        (lambda: m.int8_linear(x, xs, w, ws, bias[:3]), "bias"),
        (lambda: m.int8_linear(x, xs, w, ws, bias.half()), "bias"),
        (lambda: m.int8_linear(x, xs, w, ws, out_dtype=torch.int32), "out_dtype"),
        (lambda: m.int8_linear(x, xs, w, ws, out=torch.empty(4, 65, device="cuda")), "out must be"),
        (lambda: m.int8_linear(x, xs, w, ws, out=x.view(-1).view(BF16)[:256].view(4, 64)), "share"),
        (lambda: m.int8_linear(x.cpu(), xs, w, ws), "CUDA"),
    ):
        with pytest.raises(ValueError, match=msg):
            call()
    xs = xs.requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        m.int8_linear(x, xs, w, ws).float().sum().backward()

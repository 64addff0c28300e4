"""GPU: products grouped by expert and their gradients against sums in fp64.

Tolerance: the tensor core adds up to 16 products and the accumulator at a time, each addend cut to the largest one's
place: less than 2^-22 of the largest magnitude, which is at most the sum S of all terms' magnitudes. n terms take
n / 16 such steps (one more where the last is short): (n / 16 + 1) 2^-22 S. Then one rounding u of the result (half a
step: 2^-11 fp16, 2^-8 bf16, 2^-24 fp32; half of fp16's subnormal step).
"""
import pytest
import torch

import muxi_race_b200 as m
from oracle.train_ref import grouped_dw_ref, grouped_ref

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}
NAN = float("nan")

# rows of the experts, N, K
CASES = [
    ([1], 8, 8), ([0, 1, 0], 16, 24), ([7, 0, 130], 64, 72), ([256], 256, 64), ([257], 264, 128), ([512, 1], 512, 64),
    ([33, 95, 16, 64, 255], 264, 1032), ([0, 0, 0, 0], 64, 64), ([300, 17, 0, 256], 256, 192), ([700], 520, 512), ([2, 1300], 768, 520),
    ([15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65], 136, 200), ([40] * 70, 72, 264), ([5] * 300, 40, 48),
    ([2500], 1032, 136), ([1, 2, 3, 1000, 4, 5], 2048, 1024), ([128] * 8, 4096, 512),
]


def randn(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def within(got, ref, mag, terms, what):
    u, tiny = U[got.dtype], TINY[got.dtype]
    tol = u * ref.abs() + (1 + u) * (terms / 16 + 1) * 2.0 ** -22 * mag + tiny
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off"


def offsets_of(sizes, first=0, dtype=torch.int32):
    return (torch.tensor([0] + sizes).cumsum(0) + first).to(dtype).cuda()


def make(sizes, N, K, dtype, first=3, rest=5, odtype=torch.int32):
    R = first + sum(sizes) + rest
    x, dy = randn(1, R, K, dtype=dtype), randn(2, R, N, dtype=dtype)
    for t in (x, dy):  # rows of no expert must not matter
        t[:first], t[R - rest:] = NAN, float("inf")
    return x, randn(3, len(sizes), N, K, dtype=dtype, scale=K ** -0.5), dy, offsets_of(sizes, first, odtype)


def check_all(x, w, dy, offsets, dw_dtype):
    E, N, K = w.shape
    ends = offsets.tolist()
    y = m.grouped_linear(x, w, offsets)
    dx, dw = m.grouped_linear_backward(dy, x, w, offsets, dw_dtype=dw_dtype)
    assert y.dtype == dx.dtype == w.dtype and dw.dtype == dw_dtype
    inside = torch.zeros(x.shape[0], 1, dtype=torch.bool, device="cuda")
    inside[ends[0]:ends[-1]] = True
    within(y, *grouped_ref(torch.where(inside, x, 0), w, offsets), K, "y")
    within(dx, *grouped_ref(torch.where(inside, dy, 0), w.mT, offsets), N, "dx")
    ref, mag = grouped_dw_ref(dy, x, offsets)
    rows = torch.tensor(ends).diff().cuda()[:, None, None]
    within(dw, ref, mag, rows, "dw")
    return y, dx, dw


@pytest.mark.parametrize("sizes,N,K", CASES)
@pytest.mark.parametrize("dtype,dw_dtype,odtype", [(F16, F16, torch.int32), (BF16, F32, torch.int64), (BF16, BF16, torch.int32)])
def test_products(cuda_device, sizes, N, K, dtype, dw_dtype, odtype):
    x, w, dy, offsets = make(sizes, N, K, dtype, odtype=odtype)
    first = check_all(x, w, dy, offsets, dw_dtype)
    again = check_all(x, w, dy, offsets, dw_dtype)
    assert all(torch.equal(a, b) for a, b in zip(first, again)), "not the same bits on a second run"
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_ragged(cuda_device, dtype):
    """Enough tiles for tiles of 512 lanes with a ragged last one, several rounds of the SMs and many tails."""
    g = torch.Generator().manual_seed(4)
    sizes = torch.randint(0, 400, (24,), generator=g).tolist()
    x, w, dy, offsets = make(sizes, 1288, 1640, dtype)
    check_all(x, w, dy, offsets, F32)


def test_every_tail(cuda_device):
    """Experts of every number of rows up to 80: the rows of the next one, which hold NaN and infinities here, stay out."""
    for n in range(1, 81):
        x, dy = randn(5, 200, 64, dtype=BF16), randn(6, 200, 64, dtype=BF16)
        offsets = torch.tensor([0, n, n, n + 1], dtype=torch.int32).cuda()
        x[n + 1:], dy[n + 1:] = NAN, NAN
        x[n], dy[n] = float("inf"), NAN
        _, dw = m.grouped_linear_backward(dy, x, randn(7, 3, 64, 64, dtype=BF16), offsets, dw_dtype=F32, need_dx=False)
        ref, mag = grouped_dw_ref(dy[:n], x[:n], offsets[:2])
        within(dw[:1], ref, mag, n, f"dw of {n} rows")
        assert bool((dw[1] == 0).all()) and bool(torch.isnan(dw[2]).all())


def test_strided_rows_and_out(cuda_device):
    sizes, N, K = [70, 0, 33, 129], 136, 200
    R = sum(sizes) + 6
    wide, wide_dy = randn(8, R, K + 56, dtype=BF16), randn(9, R, N + 24, dtype=BF16)
    x, dy = wide[:, 8:8 + K], wide_dy[:, 16:16 + N]
    w, offsets = randn(10, 4, N, K, dtype=BF16), offsets_of(sizes, 2)
    y, dx, dw = m.grouped_linear(x, w, offsets), *m.grouped_linear_backward(dy, x, w, offsets)
    y2, (dx2, dw2) = m.grouped_linear(x.contiguous(), w, offsets), m.grouped_linear_backward(dy.contiguous(), x.contiguous(), w, offsets)
    assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    for start, pitch in ((0, N), (8, N + 16), (3, N + 5), (1, N + 8)):  # also rows that TMA and 16-byte stores cannot address
        base = torch.full((R, pitch + 8), 7.0, dtype=BF16, device="cuda")
        out = base[:, start:start + N]
        assert m.grouped_linear(x, w, offsets, out=out) is out
        assert torch.equal(out[2:-4], y[2:-4])
        out[2:-4] = 7.0
        assert bool((base == 7.0).all()), "rows of no expert, or memory around out, were written"
    assert bool((y[:2] == 0).all()) and bool((y[-4:] == 0).all()) and bool((dx[:2] == 0).all()) and bool((dx[-4:] == 0).all())


def test_offsets_beyond_the_rows_are_clamped(cuda_device):
    x, w, dy, _ = make([64], 64, 64, F16, 0, 0)
    w = w.repeat(3, 1, 1)
    for bad, good in (([0, 20, 10 ** 6, 10 ** 6], [0, 20, 64, 64]), ([-9, 20, 30, 64], [0, 20, 30, 64]), ([0, 30, 30, 2 ** 31 - 1], [0, 30, 30, 64])):
        for dt in (torch.int32, torch.int64):
            a, b = (torch.tensor(t, dtype=dt).cuda() for t in (bad, good))
            assert torch.equal(m.grouped_linear(x, w, a), m.grouped_linear(x, w, b))
            assert all(torch.equal(p, q) for p, q in zip(m.grouped_linear_backward(dy, x, w, a), m.grouped_linear_backward(dy, x, w, b)))


def test_no_rows(cuda_device):
    x, w, dy, offsets = make([0, 0], 64, 128, BF16, 0, 0)
    assert m.grouped_linear(x, w, offsets).shape == (0, 64)
    dx, dw = m.grouped_linear_backward(dy, x, w, offsets, dw_dtype=F32)
    assert dx.shape == (0, 128) and dw.dtype == F32 and bool((dw == 0).all())
    dx, dw = m.grouped_linear_backward(dy, None, w, offsets, need_dw=False)
    assert dx is not None and dw is None


def test_infinities_and_nan_of_a_row_stay_in_it(cuda_device):
    x, w, dy, offsets = make([100, 60], 72, 64, F16, 0, 0)
    ref = m.grouped_linear(x, w, offsets)
    x[10, 3], x[120, 5] = NAN, float("inf")
    y = m.grouped_linear(x, w, offsets)
    keep = torch.ones(160, dtype=torch.bool, device="cuda")
    keep[10] = keep[120] = False
    assert torch.equal(y[keep], ref[keep]) and bool(torch.isnan(y[10]).all()) and not bool(torch.isfinite(y[120]).any())


@pytest.mark.parametrize("save", [None, torch.int8, torch.float8_e4m3fn])
def test_autograd(cuda_device, save):
    x, w, dy, offsets = make([50, 0, 77], 72, 136, BF16, 2, 3)
    x[:2], x[-3:], dy[:2], dy[-3:] = 1.0, 1.0, 1.0, 1.0
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = m.grouped_linear(a, b, offsets, save=save)
    y.backward(dy)
    kept = x if save is None else m.restore_rows8(m.save_rows8(x, save))
    dx, dw = m.grouped_linear_backward(dy, kept, w, offsets)
    assert torch.equal(y, m.grouped_linear(x, w, offsets)) and torch.equal(a.grad, dx) and torch.equal(b.grad, dw)
    if save is not None:
        assert torch.equal(dw, m.grouped_linear_backward(dy, m.save_rows8(x, save), w, offsets)[1])
    a = x.clone().requires_grad_()
    m.grouped_linear(a, w, offsets).backward(dy.t().contiguous().t())  # a gradient with other strides
    assert torch.equal(a.grad, dx)
    b = w.clone().requires_grad_()
    m.grouped_linear(x, b, offsets).sum().backward()  # and one without memory of its own
    assert torch.equal(b.grad, m.grouped_linear_backward(torch.ones_like(dy), x, w, offsets)[1])
    a = x.clone().requires_grad_()
    g, = torch.autograd.grad(m.grouped_linear(a, w, offsets).float().square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.float().sum().backward()


def test_differences(cuda_device):
    """The product is linear in x and in w: (L(x + v) - L(x - v)) / 2 is dx . v but for the outputs' rounding, 2^-11 of each of
    R N terms at random: below 2^-11 |y| |dy|, some 1e-3 of the terms."""
    x, w, dy, offsets = make([90, 31], 64, 96, F16, 0, 0)
    dx, dw = m.grouped_linear_backward(dy, x, w, offsets, dw_dtype=F32)
    for t, grad in ((x, dx), (w, dw)):
        v = randn(11, *t.shape, dtype=F16, scale=0.25 * float(t.float().std()))
        up, down = (t + v), (t - v)
        args = (lambda s: (s, w)) if t is x else (lambda s: (x, s))
        ys = [m.grouped_linear(*args(s), offsets).double() for s in (up, down)]
        got = float(((ys[0] - ys[1]) * dy.double()).sum())
        want = float((grad.double() * (up.double() - down.double())).sum())
        noise = sum(float(2.0 ** -11 * y.norm() * dy.double().abs().max()) * 4 for y in ys)
        assert abs(got - want) <= noise + 2.0 ** -10 * abs(want), (got, want, noise)


def test_stream_and_graph(cuda_device):
    x, w, dy, offsets = make([64, 200, 0, 31], 136, 264, BF16, 1, 2)

    def step():
        return (m.grouped_linear(x, w, offsets), *m.grouped_linear_backward(dy, x, w, offsets))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [step() for _ in range(3)]
    s.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    offsets.copy_(torch.tensor([0, 100, 101, 250, 298], dtype=torch.int32))
    x.nan_to_num_(1.0, 1.0, 1.0).mul_(0.5)
    dy.nan_to_num_(1.0, 1.0, 1.0)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals(cuda_device):
    x, w, dy, offsets = make([30, 34], 64, 128, BF16, 0, 0)
    for call, msg in (
        (lambda: m.grouped_linear(x.half(), w, offsets), "x must be"),
        (lambda: m.grouped_linear(x.float(), w.float(), offsets), "fp16 or bf16"),
        (lambda: m.grouped_linear(x[:, :120], w, offsets), "x must be"),
        (lambda: m.grouped_linear(x, w, offsets[:2]), "offsets"),
        (lambda: m.grouped_linear(x, w, offsets.float()), "offsets"),
        (lambda: m.grouped_linear(x, w, offsets.cpu()), "offsets"),
        (lambda: m.grouped_linear(x, w[:, :60], offsets), "contiguous"),
        (lambda: m.grouped_linear(x, w[:, :60].contiguous(), offsets), "multiples of 8"),
        (lambda: m.grouped_linear(randn(1, 64, 132, dtype=BF16)[:, 1:129], w, offsets), "16 bytes"),
        (lambda: m.grouped_linear(x.t(), w, offsets), "x must be"),
        (lambda: m.grouped_linear(x, w, offsets, out=x[:, :64]), "share"),
        (lambda: m.grouped_linear(x, w, offsets, out=torch.empty(64, 65, dtype=BF16, device="cuda")), "out must be"),
        (lambda: m.grouped_linear(x, w, offsets, out=torch.empty(64, dtype=BF16, device="cuda").expand(64, 64)), "overlap"),
        (lambda: m.grouped_linear(x, w, offsets, save=torch.uint8), "save"),
        (lambda: m.grouped_linear(x.clone().requires_grad_(), w, offsets, out=torch.empty(64, 64, dtype=BF16, device="cuda")), "differentiable"),
        (lambda: m.grouped_linear_backward(dy, x, w, offsets, dw_dtype=F16), "dw_dtype"),
        (lambda: m.grouped_linear_backward(dy, x[:60], w, offsets), "x must be"),
        (lambda: m.grouped_linear_backward(dy, m.save_rows8(x[:60]), w, offsets), "saved x"),
        (lambda: m.grouped_linear_backward(dy[:, :56], x, w, offsets), "dy must be"),
    ):
        with pytest.raises(ValueError, match=msg):
            call()
    many = torch.zeros(1026, dtype=torch.int32, device="cuda")
    with pytest.raises(m._lib.MoeError, match="1024"):
        m.grouped_linear(torch.zeros(8, 8, dtype=BF16, device="cuda"), torch.zeros(1025, 8, 8, dtype=BF16, device="cuda"), many)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_long_sums_in_32_bits(cuda_device, dtype):
    """A 32-bit dW of many rows: parts of at most 768 rows are 48 steps of the tensor core, each off by at most 2^-23 of the sum so
    far and towards zero, and their sums are added with rounding. Of normal data the sum so far is on average two thirds of
    sqrt(rows of the part) and the parts' errors add up like their values: below 48 * 2^-24 * 2 / 3 = 1.9e-6 of dW's norm, for any
    number of rows; in one piece 6000 rows would have 1.5e-5."""
    R, N, K = 6001, 264, 512
    x, dy = randn(20, R, K, dtype=dtype), randn(21, R, N, dtype=dtype)
    offsets = torch.tensor([0, 770, 770, R], dtype=torch.int32, device="cuda")
    _, dw = m.grouped_linear_backward(dy, x, torch.empty(3, N, K, dtype=dtype, device="cuda"), offsets, dw_dtype=F32, need_dx=False)
    ref, mag = grouped_dw_ref(dy, x, offsets)
    for e in (0, 2):
        assert float((dw[e].double() - ref[e]).norm() / ref[e].norm()) < 1.9e-6
    assert bool((dw[1] == 0).all())
    again = m.grouped_linear_backward(dy, x, torch.empty(3, N, K, dtype=dtype, device="cuda"), offsets, dw_dtype=F32, need_dx=False)[1]
    assert torch.equal(dw, again)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,K", [(64, 13000), (4104, 1544), (264, 4096)])
def test_a_row_does_not_depend_on_the_others(cuda_device, N, K, dtype):
    """The same bits of y and dx for one row, a few and thousands, which take tiles of other sizes and cuts."""
    x, w, dy, _ = make([0, 4700], N, K, dtype, 0, 0)

    def products(rows):
        offsets = torch.tensor([0, 0, rows], dtype=torch.int32).cuda()
        return m.grouped_linear(x[:rows], w, offsets), m.grouped_linear_backward(dy[:rows], None, w, offsets, need_dw=False)[0]

    y, dx = products(4700)
    for rows in (1, 2, 33, 300, 1100, 2600):
        y2, dx2 = products(rows)
        assert torch.equal(y[:rows], y2) and torch.equal(dx[:rows], dx2), rows
    first = torch.tensor([0, 1000, 4700], dtype=torch.int64).cuda()
    y2 = m.grouped_linear(x, w[1:].expand(2, N, K).contiguous(), first)
    assert torch.equal(y, y2)

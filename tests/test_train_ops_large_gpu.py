"""GPU: tensors whose element offsets pass 2^31, and calls of two threads at once. Values are compared with those of small
calls on the same rows, bit for bit (a row's result does not depend on the others; the tiles' sums have one order)."""
import threading

import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROWS = 270000  # times 8192 columns: 2.2e9


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def test_grouped_rows(cuda_device):
    x, w = randn(1, ROWS, 64, dtype=BF16), randn(2, 2, 8192, 64, dtype=BF16)
    offsets = torch.tensor([0, ROWS - 300, ROWS], dtype=torch.int64, device="cuda")
    y = m.grouped_linear(x, w, offsets)
    ref = m.grouped_linear(x[-300:], w[1:], torch.tensor([0, 300], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[-300:], ref)
    dx, _ = m.grouped_linear_backward(y, x, w, offsets, need_dw=False)  # reads what lies past 2^31
    assert torch.equal(dx[-300:], m.grouped_linear_backward(ref, None, w[1:], torch.tensor([0, 300], dtype=torch.int32, device="cuda"),
                                                            need_dw=False)[0])
    _, dw = m.grouped_linear_backward(y, x, w, offsets, need_dx=False)
    want = m.grouped_linear_backward(ref, x[-300:].contiguous(), w[1:], torch.tensor([0, 300], dtype=torch.int32, device="cuda"), need_dx=False)[1]
    assert torch.equal(dw[1], want[0])


def test_grouped_weights(cuda_device):
    E, N, K = 40, 8192, 8192  # 2.7e9 elements
    x, dy = randn(3, 80, K, dtype=BF16), randn(4, 80, N, dtype=BF16)
    offsets = torch.arange(0, 81, 2, dtype=torch.int32, device="cuda")
    w = torch.empty(E, N, K, dtype=BF16, device="cuda")
    w.copy_(randn(5, 1, N, K, dtype=BF16).expand(E, N, K))
    two = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    y = m.grouped_linear(x, w, offsets)
    assert torch.equal(y[-2:], m.grouped_linear(x[-2:], w[-1:], two))
    dx, dw = m.grouped_linear_backward(dy, x, w, offsets)
    sdx, sdw = m.grouped_linear_backward(dy[-2:], x[-2:], w[-1:], two)
    assert torch.equal(dx[-2:], sdx) and torch.equal(dw[-1], sdw[0])


def test_activation_and_copies(cuda_device):
    I = 4096
    gate_up, w = torch.empty(ROWS, 2 * I, dtype=BF16, device="cuda"), randn(6, ROWS)
    tail = randn(7, 100, 2 * I, dtype=BF16)
    gate_up[:-100], gate_up[-100:] = 0.5, tail
    h, saved = m.silu_mul_rows8(gate_up, w)
    h2, s2 = m.silu_mul_rows8(tail, w[-100:].contiguous())
    assert torch.equal(h[-100:], h2) and torch.equal(saved.q[-100:], s2.q) and torch.equal(saved.scale[-100:], s2.scale)
    del gate_up
    dh = h  # any values
    dgu, dw, again = m.silu_mul_backward(dh, saved, w)
    d2 = m.silu_mul_backward(h2, s2, w[-100:].contiguous())
    assert torch.equal(dgu[-100:], d2[0]) and torch.equal(dw[-100:], d2[1]) and torch.equal(again[-100:], d2[2])
    del dgu, again
    copy = m.Rows8(saved.q, m.save_rows8(torch.zeros(1, 2 * I, dtype=BF16, device="cuda")).scale.expand(ROWS, -1).contiguous() + 1.0, BF16)
    rows = m.restore_rows8(copy, torch.tensor([ROWS - 1, 0], device="cuda"))
    assert torch.equal(rows[0].float(), saved.q[-1].float())


def test_int8_rows(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randint(-127, 128, (ROWS, 64), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (8192, 64), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = randn(9, ROWS).abs(), randn(10, 8192).abs()
    y = m.int8_linear(x, xs, w, ws)
    assert torch.equal(y[-50:], m.int8_linear(x[-50:], xs[-50:].contiguous(), w, ws))


def test_two_threads(cuda_device):
    """Two threads, each with its data, on the default stream and on one of their own: the results of calls one after another."""
    def data(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        ids = torch.rand((60, 8), generator=g, device="cuda").topk(2, -1).indices.int()
        return (randn(seed, 60, 128, dtype=BF16), randn(seed + 1, 8, 128, 128, dtype=BF16) / 8, randn(seed + 2, 8, 128, 64, dtype=BF16) / 8, ids,
                torch.rand((60, 2), generator=g, device="cuda"), randn(seed + 3, 60, 128, dtype=BF16))

    def step(d):
        leaves = [t.clone().requires_grad_() for t in (*d[:3], d[4])]
        out = m.moe_mlp(leaves[0], leaves[1], leaves[2], d[3], leaves[3], save=torch.int8)
        return (out.detach(), *torch.autograd.grad(out, leaves, d[5]))

    sets = [data(20), data(40)]
    want = [step(d) for d in sets]
    torch.cuda.synchronize()
    for own_stream in (False, True):
        bad, errors = [0, 0], []

        def work(i):
            try:
                s = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
                with torch.cuda.stream(s):
                    got = [step(sets[i]) for _ in range(15)]
                s.synchronize()
                bad[i] = sum(not torch.equal(a, b) for g in got for a, b in zip(g, want[i]))
            except Exception as e:  # noqa: BLE001
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors and bad == [0, 0], (errors, bad)


def test_1024_experts(cuda_device):
    """The most experts there can be, with 0 to 3 rows each: each row against its expert's product alone."""
    g = torch.Generator().manual_seed(11)
    sizes = torch.randint(0, 4, (1024,), generator=g)
    offsets = torch.cat((torch.zeros(1, dtype=torch.long), sizes.cumsum(0))).to(torch.int32).cuda()
    R = int(sizes.sum())
    x, w, dy = randn(12, R, 64, dtype=BF16), randn(13, 1024, 40, 64, dtype=BF16), randn(14, R, 40, dtype=BF16)
    y, (dx, dw) = m.grouped_linear(x, w, offsets), m.grouped_linear_backward(dy, x, w, offsets, dw_dtype=torch.float32)
    e = torch.repeat_interleave(torch.arange(1024), sizes).cuda()
    per_row = torch.arange(R + 1, dtype=torch.int32, device="cuda")
    for lo in range(0, R, 1000):  # a product with a copy of the weights for each row
        hi = min(R, lo + 1000)
        one = per_row[: hi - lo + 1]
        we = w[e[lo:hi]].contiguous()
        assert torch.equal(y[lo:hi], m.grouped_linear(x[lo:hi], we, one))
        assert torch.equal(dx[lo:hi], m.grouped_linear_backward(dy[lo:hi], None, we, one, need_dw=False)[0])
    ref = torch.zeros(1024, 40, 64, dtype=torch.float64, device="cuda").index_add_(0, e, dy.double()[:, :, None] * x.double()[:, None])
    mag = torch.zeros_like(ref).index_add_(0, e, (dy.double()[:, :, None] * x.double()[:, None]).abs())
    assert bool(((dw.double() - ref).abs() <= 2.0 ** -21 * mag).all())  # one step of the tensor core, and the rounding

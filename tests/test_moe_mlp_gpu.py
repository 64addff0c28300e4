"""GPU: moe_mlp, the experts with gradients, bit for bit against the chain of its operators, and against fp64.

The chain is made of the package's public operators (each tested by itself) and torch indexing, with the token's rows added
in fp32 in the order of its routes and rounded once. Against fp64: each rounding between the operators (gate_up, h, rows, sum
in the forward pass; dy is exact, dh, dgate_up, dx rows, their sum or the weights' gradient in the backward pass) moves a
result by at most u = half a step of its norm, and random data do not amplify that by more than 2: 8 u forward, 14 u backward.
"""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
I8, F8 = torch.int8, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def randn(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def make(T, H, I, E, k, dtype, wdt=F32, idt=torch.int32, bad=True, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    ids = torch.rand((T, E), generator=g).topk(k, -1).indices.to(idt)
    if bad and T > 3:
        ids[1, 0], ids[2, :], ids[3, -1] = -1, -1, E
    x, w13, w2 = randn(1, T, H, dtype=dtype), randn(2, E, 2 * I, H, dtype=dtype, scale=H ** -0.5), randn(3, E, H, I, dtype=dtype, scale=I ** -0.5)
    return x, w13, w2, ids.cuda(), torch.rand((T, k), generator=g).to(wdt).cuda(), randn(4, T, H, dtype=dtype)


def chain(x, w13, w2, ids, weights, dout, save):
    """out and the gradients of x, w13, w2 and weights by the operators one after another."""
    T, k = ids.shape
    E, H = w13.shape[0], x.shape[1]
    flat = ids.reshape(-1).long()
    valid = (flat >= 0) & (flat < E)
    order = torch.sort(torch.where(valid, flat, E), stable=True).indices[: int(valid.sum())]
    offsets = torch.bincount(flat[valid], minlength=E).cumsum(0).to(torch.int32)
    offsets = torch.cat((torch.zeros(1, dtype=torch.int32, device="cuda"), offsets))
    token, wr = order // k, weights.reshape(-1)[order].contiguous()

    def combine(rows):
        at = torch.full((T * k,), -1, dtype=torch.long, device="cuda")
        at[order] = torch.arange(order.numel(), device="cuda")
        total = torch.zeros(T, H, device="cuda")
        for j in range(k):
            s = at.view(T, k)[:, j]
            total = total + torch.where((s >= 0)[:, None], rows[s.clamp_min(0)].float() if rows.shape[0] else torch.zeros(T, H, device="cuda"), 0.0)
        return total.to(x.dtype)

    gate_up = m.grouped_linear(x[token], w13, offsets)
    h = m.silu_mul(gate_up, wr)
    out = combine(m.grouped_linear(h, w2, offsets))
    kept = gate_up if save is None else m.save_rows8(gate_up, save, parts=2)
    x_kept = x if save is None else m.restore_rows8(m.save_rows8(x, save))
    dy = dout[token]
    dh, _ = m.grouped_linear_backward(dy, None, w2, offsets, need_dw=False)
    dgu, dwr, h2 = m.silu_mul_backward(dh, kept, wr)
    _, dw2 = m.grouped_linear_backward(dy, h2, w2, offsets, need_dx=False)
    dxs, dw13 = m.grouped_linear_backward(dgu, x_kept[token], w13, offsets)
    dweights = torch.zeros(T * k, dtype=weights.dtype, device="cuda")
    dweights[order] = dwr
    return out, combine(dxs), dw13, dw2, dweights.view(T, k)


def run(x, w13, w2, ids, weights, dout, save):
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2, weights)]
    out = m.moe_mlp(leaves[0], leaves[1], leaves[2], ids, leaves[3], save=save)
    out.backward(dout)
    return (out.detach(), *(t.grad for t in leaves))


@pytest.mark.parametrize("T,H,I,E,k", [(1, 64, 32, 4, 2), (2, 8, 8, 1, 1), (5, 72, 40, 8, 3), (64, 1024, 512, 8, 2), (130, 264, 136, 16, 4),
                                       (300, 256, 192, 64, 8), (37, 520, 1000, 5, 1), (700, 128, 256, 3, 2)])
@pytest.mark.parametrize("dtype,wdt,idt", [(BF16, F32, torch.int32), (F16, F16, torch.int64)])
@pytest.mark.parametrize("save", [None, I8, F8])
def test_chain(cuda_device, T, H, I, E, k, dtype, wdt, idt, save):
    args = make(T, H, I, E, k, dtype, wdt, idt)
    got, want = run(*args, save), chain(*args, save)
    for name, a, b in zip(("out", "dx", "dw13", "dw2", "dweights"), got, want):
        assert a.dtype == b.dtype and torch.equal(a, b), f"{name}: {int((a != b).sum())} of {a.numel()} differ"
    assert torch.equal(m.moe_mlp(*args[:5]), got[0])
    again = run(*args, save)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "not the same bits on a second run"
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_against_fp64(cuda_device, dtype):
    x, w13, w2, ids, weights, dout = make(96, 256, 128, 6, 2, dtype)
    got = run(x, w13, w2, ids, weights, dout, None)
    leaves = [t.double().requires_grad_() for t in (x, w13, w2, weights)]
    rows = []
    for t in range(96):
        total = torch.zeros(256, dtype=torch.float64, device="cuda")
        for j in range(2):
            e = int(ids[t, j])
            if 0 <= e < 6:
                g, u = (leaves[1][e] @ leaves[0][t]).chunk(2)
                total = total + leaves[2][e] @ (torch.nn.functional.silu(g) * u) * leaves[3][t, j]
        rows.append(total)
    out = torch.stack(rows)
    out.backward(dout.double())
    for name, a, b, most in zip(("out", "dx", "dw13", "dw2", "dweights"), got, (out.detach(), *(t.grad for t in leaves)), (8, 14, 14, 14, 14)):
        err = float((a.double() - b).norm() / b.norm())
        assert err <= most * U[dtype], f"{name}: {err}"
    # fused_moe is the same operator: two roundings (h, out) there, four here
    other = m.fused_moe(x, w13, w2, ids, weights)
    assert float((other.double() - out.detach()).norm() / out.detach().norm()) <= 8 * U[dtype]


def test_no_route_and_no_token(cuda_device):
    x, w13, w2, ids, weights, dout = make(6, 64, 32, 4, 2, BF16)
    ids.fill_(-1)
    out, dx, dw13, dw2, dweights = run(x, w13, w2, ids, weights, dout, I8)
    assert all(bool((t == 0).all()) for t in (out, dx, dw13, dw2, dweights))
    out, dx, dw13, dw2, dweights = run(x[:0], w13, w2, ids[:0], weights[:0], dout[:0], None)
    assert out.shape == (0, 64) and bool((dw13 == 0).all()) and bool((dw2 == 0).all()) and dweights.shape == (0, 2)
    out, dx, dw13, dw2, dweights = run(x, w13, w2, ids[:, :0].contiguous(), weights[:, :0].contiguous(), dout, None)
    assert all(bool((t == 0).all()) for t in (out, dx, dw13, dw2)) and dweights.shape == (6, 0)


def test_only_some_gradients(cuda_device):
    args = make(40, 128, 64, 4, 2, BF16)
    want = run(*args, None)
    for which in range(4):
        leaves = [t.clone() for t in (*args[:3], args[4])]
        leaves[which].requires_grad_()
        m.moe_mlp(leaves[0], leaves[1], leaves[2], args[3], leaves[3]).backward(args[5])
        assert torch.equal(leaves[which].grad, want[1 + which])
        assert all(t.grad is None for i, t in enumerate(leaves) if i != which)
    x = args[0].clone().requires_grad_()
    m.moe_mlp(x, *args[1:5]).backward(args[5].t().contiguous().t())  # a gradient with other strides
    assert torch.equal(x.grad, want[1])
    x = args[0].clone().requires_grad_()
    g, = torch.autograd.grad(m.moe_mlp(x, *args[1:5]).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.float().sum().backward()


def test_saved_memory(cuda_device):
    """What a call keeps for its backward pass: with 8-bit copies, half of the 16-bit rows and the scales."""
    args = make(512, 512, 1024, 4, 2, BF16, bad=False)
    kept = {}
    for save in (None, I8):
        x = args[0].clone().requires_grad_()
        m.moe_mlp(x, *args[1:5], save=save)  # whatever the first call allocates
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = m.moe_mlp(x, *args[1:5], save=save)
        kept[save] = torch.cuda.memory_allocated() - before - out.numel() * 2
    rows16, copy = 2 * 1024 * 2048, 512 * 512 + 512 * 16
    metadata = 64 * 1024  # offsets and orders
    assert kept[None] <= rows16 + metadata  # gate_up; x is the caller's
    assert kept[I8] <= rows16 // 2 + rows16 // 64 + copy + metadata


def test_stream_and_graph(cuda_device):
    args = make(48, 256, 128, 8, 2, BF16)
    want = run(*args, I8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [run(*args, I8) for _ in range(2)]
    s.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    x, ids, weights = args[0].clone(), args[3].clone(), args[4].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.moe_mlp(x, args[1], args[2], ids, weights)
    new = make(48, 256, 128, 8, 2, BF16, seed=5)
    x.copy_(new[0] * 0.5), ids.copy_(new[3]), weights.copy_(new[4])
    graph.replay()
    assert torch.equal(out, m.moe_mlp(x, args[1], args[2], ids, weights))


def test_backward_in_a_graph(cuda_device):
    """Forward and backward captured as one graph (leaves without an eager graph that still lives), and replayed on new
    values."""
    args = make(40, 128, 64, 4, 2, BF16)
    static = [t.clone() for t in (*args[:3], args[4], args[5])]
    ids = args[3].clone()

    def step(leaves):
        out = m.moe_mlp(leaves[0], leaves[1], leaves[2], ids, leaves[3], save=I8)
        return torch.autograd.grad(out, leaves, static[4])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step([t.detach().requires_grad_() for t in static[:4]])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step([t.detach().requires_grad_() for t in static[:4]])
    new = make(40, 128, 64, 4, 2, BF16, seed=9)
    ids.copy_(new[3]), static[3].copy_(new[4]), static[0].mul_(-0.5)
    for _ in range(2):
        graph.replay()
    want = run(*static[:3], ids, static[3], static[4], I8)[1:]
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_many_routes_to_one_expert(cuda_device):
    """All 40000 routes to the last of 3 experts, and one row longer than the sorted part of a lane."""
    x, w13, w2, _, _, dout = make(20000, 64, 32, 3, 2, BF16)
    ids = torch.full((20000, 2), 2, dtype=torch.int32, device="cuda")
    ids[777, 1] = 0
    weights = torch.full((20000, 2), 0.5, device="cuda")
    got, want = run(x, w13, w2, ids, weights, dout, None), chain(x, w13, w2, ids, weights, dout, None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_with_the_router_and_the_norm(cuda_device):
    """Norm, routing and experts as one differentiable layer: the gradients of its parts arrive at every parameter."""
    T, H, I, E, k = 80, 256, 128, 8, 2
    x, w13, w2, _, _, dout = make(T, H, I, E, k, BF16)
    norm, gate = torch.ones(H, device="cuda", requires_grad=True), randn(6, E, H, scale=H ** -0.5).requires_grad_()
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    y = m.add_rms_norm(leaves[0], norm)
    weights, ids = m.route_topk(y.float() @ gate.T, k)
    out = m.moe_mlp(y, leaves[1], leaves[2], ids, weights, save=I8)
    (out.float() * dout.float()).sum().backward()
    for t in (norm, gate, *leaves):
        assert t.grad is not None and bool(torch.isfinite(t.grad).all()) and float(t.grad.float().norm()) > 0


def test_refusals(cuda_device):
    x, w13, w2, ids, weights, _ = make(8, 64, 32, 4, 2, BF16)
    for call, msg in (
        (lambda: m.moe_mlp(x.float(), w13, w2, ids, weights), "fp16 or all bf16"),
        (lambda: m.moe_mlp(x, w13, w2.half(), ids, weights), "fp16 or all bf16"),
        (lambda: m.moe_mlp(x, w13[:, :63].contiguous(), w2, ids, weights), "w_gate_up"),
        (lambda: m.moe_mlp(x, w13, w2[:3], ids, weights), "w_down"),
        (lambda: m.moe_mlp(x[:, :56], w13, w2, ids, weights), "hidden_states"),
        (lambda: m.moe_mlp(x[:4], w13, w2, ids, weights), "topk"),
        (lambda: m.moe_mlp(x, w13, w2, ids.float(), weights), "topk_ids"),
        (lambda: m.moe_mlp(x, w13, w2, ids, weights[:, :1]), "topk"),
        (lambda: m.moe_mlp(x, w13, w2, ids, weights.int()), "topk_weights"),
        (lambda: m.moe_mlp(x.t().contiguous().t(), w13, w2, ids, weights), "contiguous"),
        (lambda: m.moe_mlp(x.cpu(), w13, w2, ids, weights), "CUDA|contiguous"),
        (lambda: m.moe_mlp(x, w13, w2, ids, weights, save=torch.uint8), "save"),
        (lambda: m.moe_mlp(x[:, :60].contiguous(), w13[:, :, :60].contiguous(), w2[:, :60].contiguous(), ids, weights), "multiples of 8"),
    ):
        with pytest.raises(ValueError, match=msg):
            call()

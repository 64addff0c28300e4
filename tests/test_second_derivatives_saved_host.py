"""CPU: operators that keep an 8-bit copy for their backward pass say that their gradients cannot be differentiated again, whatever
else needs a gradient. The kernels are replaced by CPU functions that, like them, return tensors without a graph."""
import pytest
import torch

from muxi_race_b200 import grouped, rows8

SAVES = (None, torch.int8, torch.float8_e4m3fn)


def second(out, leaf, square):
    """The derivative of a loss with a penalty on its gradient. Not squared, the gradient that reaches the operator is a constant
    (``pow(1)`` would lead back to the output)."""
    loss = (out.float().square() if square else out.float()).sum()
    g, = torch.autograd.grad(loss, leaf, create_graph=True)
    return torch.autograd.grad(loss + g.float().square().sum(), leaf)


@pytest.mark.parametrize("save", SAVES)
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("weights", [None, "frozen", "trained"])
def test_silu_mul(monkeypatch, save, square, weights):
    def forward(gate_up, w, q_dtype, at=None, valid=None):
        with torch.no_grad():
            g, u = gate_up.float().chunk(2, -1)
            h = (torch.nn.functional.silu(g) * u * (1 if w is None else w[:, None])).to(gate_up.dtype)
            if q_dtype is None:
                return h, None
            return h, rows8.Rows8(torch.zeros(gate_up.shape, dtype=q_dtype), torch.ones(gate_up.shape[0], 2), gate_up.dtype, 2)

    def backward(dh, gate_up, w=None):
        with torch.no_grad():
            return torch.ones(gate_up.shape, dtype=dh.dtype), None if w is None else torch.ones_like(w), dh

    monkeypatch.setattr(rows8, "silu_forward", forward)
    monkeypatch.setattr(rows8, "silu_mul_backward", backward)
    gate_up = torch.randn(3, 16).bfloat16().requires_grad_()
    w = None if weights is None else torch.rand(3).requires_grad_(weights == "trained")
    for leaf in (gate_up,) if weights != "trained" else (gate_up, w):
        with pytest.raises(RuntimeError, match="silu_mul can be differentiated once"):
            second(rows8.silu_mul(gate_up, w, save=save), leaf, square)
    h = rows8.silu_mul(gate_up, w, save=save)
    h.float().sum().backward()
    assert bool((gate_up.grad == 1).all())


@pytest.mark.parametrize("save", SAVES)
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("frozen", [False, True])  # x itself
def test_grouped_linear(monkeypatch, save, square, frozen):
    def product(name, x, x_name, w, offsets, transposed, out=None, zero_rest=True):
        with torch.no_grad():
            return x @ w[0].T

    def backward(dy, x, w, offsets, need_dx=True, need_dw=True):
        with torch.no_grad():
            return dy @ w[0] if need_dx else None, torch.ones_like(w) if need_dw else None

    monkeypatch.setattr(grouped, "_rows_product", product)
    monkeypatch.setattr(grouped, "grouped_linear_backward", backward)
    monkeypatch.setattr(grouped, "save_rows8",
                        lambda x, q_dtype: rows8.Rows8(torch.zeros(x.shape, dtype=q_dtype), torch.ones(x.shape[0], 1), x.dtype))
    source = torch.randn(3, 8, requires_grad=True)  # what x comes from
    w, offsets = torch.randn(1, 8, 8).bfloat16().requires_grad_(), torch.tensor([0, 3])
    for leaf in (w,) if frozen else (source, w):
        x = source.bfloat16().detach() if frozen else source.bfloat16()
        y = grouped.grouped_linear(x, w, offsets, save=save)
        # dw depends on x, dx on w: each derivative through the other one has to be noticed
        g, = torch.autograd.grad((y.float().square() if square else y.float()).sum(), w, create_graph=True)
        if not frozen or square:
            with pytest.raises(RuntimeError, match="grouped_linear can be differentiated once"):
                torch.autograd.grad(g.float().square().sum(), leaf, allow_unused=True)
    x = source.bfloat16()
    grouped.grouped_linear(x, w, offsets, save=save).float().sum().backward()
    assert bool((w.grad == 1).all()) and source.grad is not None


class CpuMlp:
    """The kernels of moe_mlp as CPU functions; one token is one route of one expert."""

    def __init__(self, monkeypatch, T=3, H=8, I=4):
        def half(*shape):
            return torch.randn(shape).bfloat16()

        self.sizes = T, H, I
        self.args = [half(T, H), half(1, 2 * I, H), half(1, H, I), torch.zeros(T, 1, dtype=torch.int32), torch.rand(T, 1)]

        def forward(x, w13, w2, ids, weights, save):
            with torch.no_grad():
                g, u = (x @ w13[0].T).chunk(2, -1)
                out = weights.to(x.dtype) * (torch.nn.functional.silu(g) * u) @ w2[0].T
                gate_up = torch.cat((g, u), -1)
                if save is not None:
                    gate_up = rows8.Rows8(torch.zeros(T, 2 * I, dtype=save), torch.ones(T, 2), x.dtype, 2)
                return out, torch.tensor([0, T], dtype=torch.int32), torch.arange(T), torch.arange(T), gate_up

        def silu_backward(dh, gate_up, weights, dweights, at=None, valid=None):
            if dweights is not None:
                dweights.fill_(1)
            return half(T, 2 * I), half(T, I)

        monkeypatch.setattr(grouped, "_mlp_forward", forward)
        monkeypatch.setattr(grouped, "silu_backward", silu_backward)
        monkeypatch.setattr(grouped, "_gather", lambda x, *a: half(T, H))
        monkeypatch.setattr(grouped, "_combine", lambda y, *a: half(T, H))
        monkeypatch.setattr(grouped, "_rows_product", lambda name, dy, n, w, *a: half(T, w.shape[2]))
        monkeypatch.setattr(grouped, "_grouped_dw", lambda dy, x, shape, offsets, dt: torch.ones(shape, dtype=dt))
        monkeypatch.setattr(grouped, "save_rows8",
                            lambda x, q_dtype: rows8.Rows8(torch.zeros(x.shape, dtype=q_dtype), torch.ones(x.shape[0], 1), x.dtype))


@pytest.mark.parametrize("save", SAVES)
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("trained", [(0,), (0, 1), (0, 2), (0, 4), (1, 4), (0, 1, 2, 4)])  # x, w13, w2, weights
def test_moe_mlp(monkeypatch, save, square, trained):
    cpu = CpuMlp(monkeypatch)
    for leaf in trained:
        args = [t.clone().requires_grad_() if i in trained else t for i, t in enumerate(cpu.args)]
        with pytest.raises(RuntimeError, match="moe_mlp can be differentiated once"):
            second(grouped._moe_mlp_graph(*args, save), args[leaf], square)
    grouped._moe_mlp_graph(*args, save).float().sum().backward()
    assert all(args[i].grad is not None for i in trained)


@pytest.mark.parametrize("save", SAVES)
@pytest.mark.parametrize("trained", [(0,), (2,), (4,), (0, 2, 4), (1,), (0, 1)])
def test_moe_mlp_keeps_tokens_for_their_gradient_only(monkeypatch, save, trained):
    """The tokens, or their copy, are read for the gradient of w_gate_up: without that nothing of their size is kept for them."""
    cpu = CpuMlp(monkeypatch, T=5, H=24, I=4)
    copies = []
    copy = grouped.save_rows8
    monkeypatch.setattr(grouped, "save_rows8", lambda x, q_dtype: copies.append(x) or copy(x, q_dtype))
    args = [t.clone().requires_grad_() if i in trained else t for i, t in enumerate(cpu.args)]
    out = grouped._moe_mlp_graph(*args, save)
    tokens = [t for t in out.grad_fn.saved_tensors if t is not None and t.shape == (5, 24)]
    assert len(tokens) == (1 in trained) and len(copies) == (1 in trained and save is not None)
    out.float().sum().backward()
    assert all(args[i].grad is not None for i in trained)


def test_moe_mlp_tangent_of_the_gradient(monkeypatch):
    """Forward-mode over the backward pass: a tangent of the gradient that reaches the operator would be dropped."""
    cpu = CpuMlp(monkeypatch)
    args = [t.clone().requires_grad_() if t.is_floating_point() else t for t in cpu.args]
    out = grouped._moe_mlp_graph(*args, None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(out, args[0], dual)

"""CPU: operators that keep an 8-bit copy for their backward pass say that their gradients cannot be differentiated again, whatever
else needs a gradient. The kernels are replaced by CPU functions that, like them, return tensors without a graph."""
import pytest
import torch

from muxi_race_b200 import rows8

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

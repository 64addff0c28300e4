"""An MoE layer from the package's operators: norm, router and experts, as a model calls them.

    python examples/moe_layer.py

  decode   the residual's addition and the norm, router logits, routing, 4-bit experts
  int8     the same with 8-bit rows from the norm straight into int8 experts
  train    norm and router with their gradients: one step towards a target distribution of the
           routing weights, and the balance bias moved by the tokens per expert
  experts  a training step of the whole layer, norm, router and 16-bit experts, towards a target output;
           what the experts' backward pass reads again is kept in 8 bits
  dense    an int8 projection beside the experts, fed by the norm's rows
"""
from __future__ import annotations

import os
import sys
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import muxi_race_b200 as m  # noqa: E402


@dataclass
class Layer:
    norm: torch.Tensor   # [H]
    gate: torch.Tensor   # [E, H] router weight
    bias: torch.Tensor   # [E] fp32, for balance
    w13: object          # experts' gate and up: W4Weights, (int8 values, scales) or bf16
    w2: object
    topk: int

    def route(self, y: torch.Tensor, return_counts: bool = False):
        """Sigmoid scores, chosen with the balance bias, renormalised."""
        logits = y.float() @ self.gate.float().T
        return m.route_topk(logits, self.topk, scoring="sigmoid", bias=self.bias, return_counts=return_counts)


def make_layer(H=1024, I=512, E=32, topk=4, kind="w4", seed=0, device="cuda") -> Layer:
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=device)

    w13, w2 = (randn(E, 2 * I, H) * H ** -0.5).bfloat16(), (randn(E, H, I) * I ** -0.5).bfloat16()
    if kind == "w4":
        w13, w2 = m.quantize_w4(w13, gate_up=True), m.quantize_w4(w2)
    elif kind == "int8":
        w13, w2 = m.quantize_rows_int8(w13), m.quantize_rows_int8(w2)
    return Layer((1 + 0.1 * randn(H)).bfloat16(), (randn(E, H) * H ** -0.5).bfloat16(),
                 torch.zeros(E, device=device), w13, w2, topk)


def decode(layer: Layer, x: torch.Tensor, residual: torch.Tensor):
    """(output of the experts, new residual) for a batch of tokens x [T, H]; the residual is updated in place."""
    y, residual = m.add_rms_norm(x, layer.norm, residual, residual_out=residual)
    weights, ids = layer.route(y)
    return m.fused_moe_w4(y, layer.w13, layer.w2, ids, weights), residual


def serve_int8(layer: Layer, x: torch.Tensor, residual: torch.Tensor):
    """The same with int8 experts: the norm writes the 8-bit rows that the experts read."""
    q, scale, residual = m.add_rms_norm_quant(x, layer.norm, residual)
    y = q.float() * scale[:, None]
    weights, ids = layer.route(y)
    return m.fused_moe_int8(q, *layer.w13, *layer.w2, ids, weights, hidden_scale=scale, out_dtype=x.dtype), residual


def train_step(layer: Layer, x: torch.Tensor, residual: torch.Tensor, target: torch.Tensor, lr=0.05, step=1e-3) -> float:
    """One step of the norm's and the router's weights: the routing weights move towards `target` [T, E],
    and the bias by `step` against each expert's surplus of tokens."""
    norm, gate = (t.float().requires_grad_() for t in (layer.norm, layer.gate))
    y, _ = m.add_rms_norm(x.float(), norm, residual.float())
    weights, ids, counts = m.route_topk(y @ gate.T, layer.topk, scoring="sigmoid", bias=layer.bias, return_counts=True)
    loss = (weights - target.gather(1, ids.long())).square().sum(-1).mean()
    loss.backward()
    with torch.no_grad():
        layer.norm.copy_(norm - lr * norm.grad)
        layer.gate.copy_(gate - lr * gate.grad)
        layer.bias += step * torch.sign(counts.float().mean() - counts.float())
    return float(loss.detach())


def layer_loss(x, residual, norm, gate, w13, w2, topk: int, target, save=None):
    """Mean square of what the layer's output, added to the residual stream, is off `target` [T, H]."""
    y, stream = m.add_rms_norm(x, norm, residual)
    weights, ids = m.route_topk(y.float() @ gate.T, topk, scoring="sigmoid")
    return (stream.float() + m.moe_mlp(y, w13, w2, ids, weights, save=save).float() - target.float()).square().mean()


def train_experts(layer: Layer, x: torch.Tensor, residual: torch.Tensor, target: torch.Tensor, lr=2.0, save=torch.int8) -> float:
    """One step of all of the layer's weights (bf16 experts) towards `target`."""
    leaves = [layer.norm.float().requires_grad_(), layer.gate.float().requires_grad_(), layer.w13.detach().requires_grad_(),
              layer.w2.detach().requires_grad_()]
    loss = layer_loss(x, residual, *leaves, layer.topk, target, save)
    loss.backward()
    with torch.no_grad():
        for t, leaf in zip((layer.norm, layer.gate, layer.w13, layer.w2), leaves):
            t.copy_(leaf.detach() - lr * leaf.grad)
    return float(loss.detach())


def dense_int8(layer: Layer, x: torch.Tensor, residual: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor):
    """A projection (int8 weights [N, H] of quantize_rows_int8) of the normalised rows, which leave the norm in 8 bits."""
    q, scale, _ = m.add_rms_norm_quant(x, layer.norm, residual)
    return m.int8_linear(q, scale, w, w_scale, out_dtype=x.dtype)


def main() -> None:
    g = torch.Generator(device="cuda").manual_seed(1)
    x, residual = (torch.randn((16, 1024), generator=g, device="cuda").bfloat16() for _ in range(2))
    layer = make_layer()
    for T in (1, 16):
        out, _ = decode(layer, x[:T], residual[:T].clone())
        print(f"decode   T={T:<3} |out| = {float(out.float().norm()):.3f}")
    out, _ = serve_int8(make_layer(kind="int8"), x, residual)
    print(f"int8     T=16  |out| = {float(out.float().norm()):.3f}")
    target = torch.softmax(torch.randn((16, 32), generator=g, device="cuda") * 3, -1)
    losses = [train_step(layer, x, residual, target) for _ in range(20)]
    print(f"train    loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    layer, target = make_layer(kind="bf16"), torch.randn((16, 1024), generator=g, device="cuda").bfloat16()
    losses = [train_experts(layer, x, residual, target) for _ in range(20)]
    print(f"experts  loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    w = m.quantize_rows_int8((torch.randn((2048, 1024), generator=g, device="cuda") * 1024 ** -0.5).bfloat16())
    print(f"dense    T=16  |out| = {float(dense_int8(layer, x, residual, *w).float().norm()):.3f}")
    assert m.device_status() == 0


if __name__ == "__main__":
    main()

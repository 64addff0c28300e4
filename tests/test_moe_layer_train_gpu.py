"""GPU: the example's training step of a whole layer and its dense int8 projection: they run, and the layer's gradients are
those of the same layer in fp64.

Tolerance of the gradients: the layer's intermediate results are rounded to bf16 (u = 2^-8 of their size) at y, gate_up, h, the
experts' rows, their sum, and backward at dout, dh, dgate_up, the rows' gradients, their sum and the result: eleven, each of which moves a
gradient by at most u of its norm, times 2 for what a product of random data may amplify. With 8-bit copies, two more: an int8
value is off by at most half of amax / 127 of its group, 2^-8 of the largest, and so at most 3 times that of the root mean square
of normal values.
"""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import moe_layer  # noqa: E402
import muxi_race_b200 as m  # noqa: E402

pytestmark = pytest.mark.gpu


def inputs(T, H, seed=1):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return [torch.randn((T, H), generator=g).bfloat16().cuda() for _ in range(3)]


@pytest.mark.parametrize("save", [None, torch.int8])
def test_gradients(cuda_device, save):
    T, H, I, E, k = 64, 256, 128, 8, 2
    layer = moe_layer.make_layer(H, I, E, k, kind="bf16")
    x, residual, target = inputs(T, H)
    leaves = [layer.norm.float().requires_grad_(), layer.gate.float().requires_grad_(), layer.w13.clone().requires_grad_(),
              layer.w2.clone().requires_grad_()]
    moe_layer.layer_loss(x, residual, *leaves, k, target, save).backward()
    with torch.no_grad():
        y, _ = m.add_rms_norm(x, leaves[0], residual)
        _, ids = m.route_topk(y.float() @ leaves[1].T, k, scoring="sigmoid")
    ref = [t.detach().double().requires_grad_() for t in leaves]
    h = x.double() + residual.double()
    y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * ref[0]
    s = torch.sigmoid(y @ ref[1].T).gather(1, ids.long())
    w = s / s.sum(-1, keepdim=True)
    out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for j in range(k):
        gu = torch.einsum("th,toh->to", y, ref[2][ids[:, j].long()])
        a = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
        out = out + torch.einsum("ti,thi->th", a, ref[3][ids[:, j].long()]) * w[:, j:j + 1]
    (h + out - target.double()).square().mean().backward()
    most = 2 * 11 * 2.0 ** -8 + (0 if save is None else 2 * 3 * 2.0 ** -8)
    for name, a, b in zip(("norm", "gate", "w13", "w2"), leaves, ref):
        err = float((a.grad.double() - b.grad).norm() / b.grad.norm())
        assert err <= most, f"{name}: {err}"


def test_training_runs(cuda_device):
    layer = moe_layer.make_layer(256, 128, 8, 2, kind="bf16")
    x, residual, target = inputs(32, 256)
    before = [t.clone() for t in (layer.norm, layer.gate, layer.w13, layer.w2)]
    for save in (None, torch.int8, torch.float8_e4m3fn):
        assert moe_layer.train_experts(layer, x, residual, target, save=save) > 0
    for t, old in zip((layer.norm, layer.gate, layer.w13, layer.w2), before):
        assert bool(torch.isfinite(t.float()).all()) and not torch.equal(t, old)


def test_dense_projection(cuda_device):
    layer = moe_layer.make_layer(256, 128, 8, 2, kind="int8")
    x, residual, _ = inputs(20, 256)
    g = torch.Generator(device="cpu").manual_seed(2)
    w, w_scale = m.quantize_rows_int8((torch.randn((320, 256), generator=g) / 16).bfloat16().cuda())
    y = moe_layer.dense_int8(layer, x, residual, w, w_scale)
    q, scale, _ = m.add_rms_norm_quant(x, layer.norm, residual)
    assert y.dtype == x.dtype and torch.equal(y, m.int8_linear(q, scale, w, w_scale))


def test_main(cuda_device, capsys):
    moe_layer.main()
    said = capsys.readouterr().out
    assert "experts  loss" in said and "dense    T=16" in said

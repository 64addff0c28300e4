"""GPU: the example layer (norm, router, experts) against the same steps in fp64, and its training step.

The layer's intermediates are rounded to bf16 (the norm's output, the experts' h and output: u = 2^-8
each) and its router chooses by them, so the check routes with the layer's own choice; three roundings
of 2^-8 relative to sums of terms of either sign stay within 2 % of the output's norm.
"""
import importlib.util
import os

import pytest
import torch

import muxi_race_b200 as m
from oracle.norm_ref import rms_norm_ref

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "moe_layer.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_layer_example", PATH)
    mod = importlib.util.module_from_spec(spec)
    import sys

    sys.modules["moe_layer_example"] = mod
    spec.loader.exec_module(mod)
    return mod


def inputs(T, H=1024):
    g = torch.Generator(device="cpu").manual_seed(T)
    return (torch.randn((T, H), generator=g).bfloat16().cuda() for _ in range(2))


def experts64(y, w13, w2, ids, weights):
    out = torch.zeros_like(y)
    I = w13.shape[1] // 2
    for e in ids.unique().tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        s = y[t] @ w13[e].double().T
        h = s[:, :I] * torch.sigmoid(s[:, :I]) * s[:, I:]
        out.index_add_(0, t, h @ w2[e].double().T * weights.double()[t, j, None])
    return out


@pytest.mark.parametrize("T", [1, 5, 64])
def test_decode(cuda_device, example, T):
    layer = example.make_layer()
    x, residual = inputs(T)
    kept = residual.clone()
    out, new = example.decode(layer, x, residual)
    assert new is residual
    y, h = rms_norm_ref(x, layer.norm, kept)
    assert float((new.double() - h).norm() / h.norm()) < 2.0 ** -8
    yy, _ = m.add_rms_norm(x, layer.norm, kept)
    weights, ids = layer.route(yy)
    ref = experts64(y, m.dequantize_w4(layer.w13), m.dequantize_w4(layer.w2), ids, weights)
    assert m.device_status() == 0
    assert float((out.double() - ref).norm() / ref.norm()) < 0.02


def test_int8(cuda_device, example):
    """int8 rows and weights: steps of 1/127 of each row's largest value (about 3.5 sigma), a relative
    error of 3.5 / 127 / sqrt(12) = 0.8 % per factor; x, w13, h, w2 are four: under 4 %."""
    layer = example.make_layer(kind="int8")
    x, residual = inputs(48)
    out, _ = example.serve_int8(layer, x, residual)
    q, scale, _ = m.add_rms_norm_quant(x, layer.norm, residual)
    weights, ids = layer.route(q.float() * scale[:, None])
    y, _ = rms_norm_ref(x, layer.norm, residual)
    w13, w2 = (v.double() * s.double()[..., None] for v, s in (layer.w13, layer.w2))
    ref = experts64(y, w13, w2, ids, weights)
    assert m.device_status() == 0
    assert float((out.double() - ref).norm() / ref.norm()) < 0.04


def test_train_step_lowers_the_loss(cuda_device, example):
    layer = example.make_layer()
    x, residual = inputs(64)
    target = torch.softmax(torch.randn(64, 32, generator=torch.Generator(device="cpu").manual_seed(9)).cuda() * 3, -1)
    losses = [example.train_step(layer, x, residual, target) for _ in range(15)]
    assert all(torch.isfinite(torch.tensor(losses))) and losses[-1] < losses[0]
    assert bool((layer.bias != 0).any())


def test_main(cuda_device, example, capsys):
    example.main()
    assert "decode" in capsys.readouterr().out

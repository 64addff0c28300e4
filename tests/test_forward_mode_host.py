"""CPU: no operator has a forward-mode derivative, and each says so where an argument carries a tangent, which its kernel would drop.
Without a tangent the same call inside the same level goes on to the usual checks."""
import pytest
import torch
from torch.autograd import forward_ad

import muxi_race_b200 as m
import muxi_race_b200.torch_ops  # noqa: F401
from muxi_race_b200 import _lib
from muxi_race_b200.ep import ExpertParallelMoE, PeerMemoryEP
from muxi_race_b200.packed import packed_layout

OPS = torch.ops.muxi_race_b200
BF16, I8 = torch.bfloat16, torch.int8


def half(*shape):
    return torch.zeros(shape, dtype=BF16)


IDS, WEIGHTS, OFF = torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, 1), torch.tensor([0, 2, 4])
W, W13, W2 = half(2, 16, 8), half(2, 16, 8), half(2, 8, 8)
X8, SCALE, W8, WSCALE = torch.zeros(4, 16, dtype=I8), torch.ones(4), torch.zeros(3, 16, dtype=I8), torch.ones(3)


def copy_of(scale, parts=1):
    return m.Rows8(torch.zeros(4, 16, dtype=I8), scale, BF16, parts)


# the call, and the floating arguments that may carry a tangent
TRAINING = {
    "grouped_linear": (lambda x, w: m.grouped_linear(x, w, OFF), half(4, 8), W),
    "grouped_linear_backward": (lambda dy, x, w: m.grouped_linear_backward(dy, x, w, OFF), half(4, 16), half(4, 8), W),
    "grouped_linear_backward, copy": (lambda dy, s, w: m.grouped_linear_backward(dy, copy_of(s), w, OFF), half(4, 16), torch.ones(4, 1), W),
    "moe_mlp": (lambda x, w13, w2, w: m.moe_mlp(x, w13, w2, IDS, w), half(4, 8), W13, W2, WEIGHTS),
    "silu_mul": (m.silu_mul, half(4, 16), SCALE),
    "silu_mul_rows8": (m.silu_mul_rows8, half(4, 16), SCALE),
    "silu_mul_backward": (m.silu_mul_backward, half(4, 8), half(4, 16), SCALE),
    "silu_mul_backward, copy": (lambda dh, s, w: m.silu_mul_backward(dh, copy_of(s, 2), w), half(4, 8), torch.ones(4, 2), SCALE),
    "save_rows8": (m.save_rows8, half(4, 16)),
    "restore_rows8": (lambda s: m.restore_rows8(copy_of(s)), torch.ones(4, 1)),
    "torch.ops grouped_linear": (lambda x, w: OPS.grouped_linear(x, w, OFF), half(4, 8), W),
    "torch.ops grouped_linear_backward": (lambda dy, x, w: OPS.grouped_linear_backward(dy, x, w, OFF), half(4, 16), half(4, 8), W),
    "torch.ops silu_mul": (OPS.silu_mul, half(4, 16), SCALE),
    "torch.ops int8_linear": (lambda xs, ws, b: OPS.int8_linear(X8, xs, W8, ws, b, BF16), SCALE, WSCALE, torch.ones(3)),
    "int8_linear": (lambda xs, ws, b: m.int8_linear(X8, xs, W8, ws, b), SCALE, WSCALE, torch.ones(3)),
}


def check(call, args):
    with forward_ad.dual_level():
        with pytest.raises(ValueError):  # not on a GPU
            call(*args)
        for i in range(len(args)):
            for grad in (True, False):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(*dual)
    with pytest.raises(ValueError):
        call(*args)


@pytest.mark.parametrize("name", TRAINING)
def test_training(name):
    call, *args = TRAINING[name]
    check(call, args)


def w4(*shape, gate_up=False):
    """4-bit weights [..., N, K] on the CPU."""
    matrices = 1
    for n in shape[:-2]:
        matrices *= n
    nbytes = _lib.lib().moe_w4_packed_bytes(matrices, *shape[-2:], 128, 0, int(gate_up))
    return m.W4Weights(torch.zeros(nbytes, dtype=torch.uint8), shape, BF16, 128, False, gate_up)


def packed():
    _, total = packed_layout(2, 8, 8, "bf16")
    return m.PackedWeights(torch.zeros(total, dtype=torch.uint8), 2, 8, 8, "bf16")


Q13, Q2 = torch.zeros(2, 16, 8, dtype=I8), torch.zeros(2, 8, 8, dtype=I8)
S13, S2 = torch.ones(2, 16), torch.ones(2, 8)
ROWS8 = torch.zeros(4, 8, dtype=I8)
LOGITS = torch.zeros(4, 2)
META = [torch.zeros(n, dtype=torch.int32) for n in (2, 3, 3, 1)]
OTHERS = {
    "fused_moe": (lambda x, w13, w2, w: m.fused_moe(x, w13, w2, IDS, w), half(4, 8), W13, W2, WEIGHTS),
    "fused_moe_router": (lambda x, w13, w2, g: m.fused_moe_router(x, w13, w2, g, 1), half(4, 8), W13, W2, LOGITS),
    "fused_moe_int8": (lambda x, s13, s2, w: m.fused_moe_int8(x, Q13, s13, Q2, s2, IDS, w), half(4, 8), S13, S2, WEIGHTS),
    "fused_moe_int8, 8-bit rows": (lambda s, s13, s2, w: m.fused_moe_int8(ROWS8, Q13, s13, Q2, s2, IDS, w, hidden_scale=s),
                                   SCALE, S13, S2, WEIGHTS),
    "fused_moe_fp8": (lambda x, s13, s2, w: m.fused_moe_fp8(x, Q13, s13, Q2, s2, IDS, w), half(4, 8), S13, S2, WEIGHTS),
    "fused_moe_packed": (lambda x, w: m.fused_moe_packed(x, packed(), IDS, w), half(4, 8), WEIGHTS),
    "fused_moe_w4": (lambda x, w: m.fused_moe_w4(x, w4(2, 16, 8, gate_up=True), w4(2, 8, 8), IDS, w), half(4, 8), WEIGHTS),
    "pack_weights": (m.pack_weights, half(2, 8, 8), half(2, 8, 8), half(2, 8, 8)),
    "quantize_rows_int8": (m.quantize_rows_int8, half(4, 8)),
    "quantize_rows_fp8": (m.quantize_rows_fp8, half(4, 8)),
    "quantize_w4": (m.quantize_w4, half(4, 8)),
    "pack_w4": (lambda s: m.pack_w4(torch.zeros(4, 4, dtype=torch.uint8), s), half(4, 1)),
    "w4_linear": (lambda x: m.w4_linear(x, w4(3, 8)), half(4, 8)),
    "fused_topk": (lambda g: m.fused_topk(half(4, 8), g, 1), LOGITS),
    "grouped_topk": (lambda g, b: m.grouped_topk(half(4, 8), g, 1, True, 1, 1, b), LOGITS, torch.zeros(2)),
    "route_topk": (lambda g, b: m.route_topk(g, 1, bias=b), LOGITS, torch.zeros(2)),
    "route_topk_backward": (lambda d, g: m.route_topk_backward(d, g, IDS), WEIGHTS, LOGITS),
    "add_rms_norm": (m.add_rms_norm, half(4, 8), half(8), half(4, 8)),
    "add_rms_norm_quant": (m.add_rms_norm_quant, half(4, 8), half(8), half(4, 8)),
    "add_rms_norm_backward": (m.add_rms_norm_backward, half(4, 8), half(4, 8), half(8), half(4, 8)),
    "run_kernel": (lambda x, g, u, d, w: m.run_kernel(x, g, u, d, w, *META, half(4, 8)), half(4, 8), half(2, 8, 8), half(2, 8, 8),
                   half(2, 8, 8), torch.ones(4)),
    "torch.ops add_rms_norm": (lambda x, w, r: OPS.add_rms_norm(x, w, r, 1e-6), half(4, 8), half(8), half(4, 8)),
    "torch.ops route_topk": (lambda g, b: OPS.route_topk(g, 1, "softmax", b, 1, 1, 2, True, 1.0), LOGITS, torch.zeros(2)),
    "torch.ops fused_moe": (lambda x, w13, w2, w: OPS.fused_moe(x, w13, w2, IDS, w), half(4, 8), W13, W2, WEIGHTS),
}


@pytest.mark.parametrize("name", OTHERS)
def test_others(name):
    call, *args = OTHERS[name]
    check(call, args)


@pytest.mark.parametrize("kind", [ExpertParallelMoE, PeerMemoryEP])
def test_expert_parallel(kind):
    layer = kind.__new__(kind)  # a rank without a group: the check comes first
    layer._closed = False
    with forward_ad.dual_level():
        x = forward_ad.make_dual(half(4, 8), half(4, 8))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            layer.forward(x, IDS, WEIGHTS)

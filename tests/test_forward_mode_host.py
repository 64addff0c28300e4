"""CPU: no operator has a forward-mode derivative, and each says so where an argument carries a tangent, which its kernel would drop.
Without a tangent the same call inside the same level goes on to the usual checks."""
import pytest
import torch
from torch.autograd import forward_ad

import muxi_race_b200 as m
import muxi_race_b200.torch_ops  # noqa: F401

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

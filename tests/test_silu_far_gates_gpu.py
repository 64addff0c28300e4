"""GPU: silu_mul and its gradient at gates where s(g) is below fp32's smallest normal number (g < -87.3) and e^-g still finite (g >=
-88.7): with large values beside them the products are ordinary numbers.

Tolerances: F(g) = (16 + 1.2 |g|) 2^-23 of a value's magnitude for exponential, reciprocal and products (tests/test_rows8_gpu.py); a
subnormal s >= 2.9e-39 = 2^-128.04 is off by half of 2^-149 at most, 2^-21.9 of itself; then one rounding to bf16.
"""
import pytest
import torch

import muxi_race_b200 as m
from oracle.train_ref import silu_mul_grad_ref, silu_mul_ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
GATES = [-86.5, -87.0, -87.5, -88.0, -88.5]


@pytest.mark.parametrize("up", [1.0, 3e36, -7e37])
@pytest.mark.parametrize("width", [5, 40])  # single elements, and whole 8s
def test_far_gates(cuda_device, up, width):
    gate = torch.tensor(GATES * (width // 5), dtype=BF16)
    gate_up = torch.cat((gate, torch.full((width,), up, dtype=BF16)))[None].cuda()
    dh = torch.full((1, width), 0.75, dtype=BF16, device="cuda")
    f = (16 + 1.2 * gate.double().abs()) * 2.0 ** -23 + 2.0 ** -21.9
    f = f[None].cuda()

    def near(got, ref, mag, what):
        err = (got.double() - ref).abs()
        tol = 2.0 ** -8 * ref.abs() + f * mag
        assert bool((err <= tol).all()), f"{what}: {got.tolist()} {ref.tolist()}"

    ref = silu_mul_ref(gate_up)
    near(m.silu_mul(gate_up), ref, ref.abs(), "h")
    dgu, _, h = m.silu_mul_backward(dh, gate_up)
    rd, _, mag, _ = silu_mul_grad_ref(dh, gate_up)
    near(dgu[:, :width], rd[:, :width], mag[:, :width], "dgate")
    near(dgu[:, width:], rd[:, width:], mag[:, width:], "dup")
    near(h, ref, ref.abs(), "h again")

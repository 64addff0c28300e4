"""GPU: a buffer that restore_rows8 fills carries no graph, and none from an earlier call."""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_dtype", [torch.int8, torch.float8_e4m3fn])
def test_out_carries_no_graph(cuda_device, q_dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((6, 200), generator=g, device="cuda").bfloat16()
    saved = m.save_rows8(x.clone().requires_grad_(), q_dtype)
    with pytest.raises(RuntimeError, match="not differentiable"):  # a new result does
        m.restore_rows8(saved).float().sum().backward()
    out = torch.empty_like(x)
    assert m.restore_rows8(saved, out=out) is out and not out.requires_grad
    w = torch.ones(200, device="cuda", requires_grad=True)
    other = m.restore_rows8(m.save_rows8(x, q_dtype), out=out)
    (other.float() * w).sum().backward()  # a constant of this graph
    assert torch.equal(w.grad, other.float().sum(0))

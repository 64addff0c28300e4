"""GPU: what the forward pass of moe_mlp holds at once."""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("train", [False, True])
def test_peak(cuda_device, train):
    """The tokens' rows in the experts' order go when the first product has read them, the activation's when the second has: never
    both [R, H] tensors at once."""
    T, H, I, E, k = 2048, 2048, 256, 4, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w13, w2 = (torch.randn(s, generator=g, device="cuda").to(BF16).requires_grad_(train) for s in ((T, H), (E, 2 * I, H), (E, H, I)))
    ids = torch.rand((T, E), generator=g, device="cuda").topk(k, -1).indices.int()
    weights = torch.rand((T, k), generator=g, device="cuda")
    m.moe_mlp(x, w13, w2, ids, weights)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = m.moe_mlp(x, w13, w2, ids, weights)
    peak = torch.cuda.max_memory_allocated() - before
    rows, gate_up, h, result = 2 * T * k * H, 2 * T * k * 2 * I, 2 * T * k * I, 2 * T * H
    assert out.shape == (T, H) and peak <= gate_up + h + rows + result + (1 << 20), peak

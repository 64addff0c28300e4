"""CPU: 4-bit weights that are not on a GPU are refused by name."""
import pytest
import torch

import muxi_race_b200 as m


def test_weights_on_the_cpu_are_refused():
    w = m.W4Weights(torch.zeros(2112, dtype=torch.uint8), (32, 128), torch.float16, 128, False, False)
    with pytest.raises(ValueError, match="CUDA"):
        m.dequantize_w4(w)
    with pytest.raises(ValueError, match="CUDA"):
        m.w4_linear(torch.zeros(1, 128, dtype=torch.float16), w)

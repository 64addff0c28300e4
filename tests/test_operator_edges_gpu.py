"""GPU: edges of the norm, routing and 4-bit operators that their own test files leave out."""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e} over"


def test_w4_linear_refuses_an_output_over_its_rows(cuda_device):
    w = m.quantize_w4(randn(1, 256, 256, dtype=F16))
    big = randn(2, 8, 600, dtype=F16)
    x = big[:, :256]
    ref = m.w4_linear(x, w)
    for out in (x, big[:, 8:264], big[:, 255:511]):
        with pytest.raises(ValueError, match="share memory"):
            m.w4_linear(x, w, out=out)
    beside = big[:, 256:512]  # other columns of the same rows
    kept = x.clone()
    assert torch.equal(m.w4_linear(x, w, out=beside), ref) and torch.equal(x, kept)

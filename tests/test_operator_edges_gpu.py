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


def test_norm_refuses_outputs_over_other_rows(cuda_device):
    """Row t + 1 of x at the place of row t of the output: a row would be written while another reads it."""
    T, H = 64, 256
    big = randn(3, T + 1, H + 32, dtype=F16)
    w, res = randn(4, H, dtype=F16), randn(5, T, H, dtype=F16)
    x = big[1:, :H]
    y, h = m.add_rms_norm(x, w, res)
    for name in ("out", "residual_out"):
        for t in (big[:-1, :H], big[1:, 8:8 + H]):
            with pytest.raises(ValueError, match="share no memory"):
                m.add_rms_norm(x, w, res, **{name: t})
    with pytest.raises(ValueError, match="share no memory"):
        m.add_rms_norm_quant(x, w, res, residual_out=big[:-1, :H])
    both = torch.empty_like(y)
    with pytest.raises(ValueError, match="out and residual_out"):
        m.add_rms_norm(x, w, res, out=both, residual_out=both)
    # x and residual themselves stay allowed, each for either output, and other columns of the same rows
    x1, r1 = x.clone(), res.clone()
    m.add_rms_norm(x1, w, r1, out=r1, residual_out=x1)
    assert torch.equal(r1, y) and torch.equal(x1, h)
    wide = randn(6, T, 3 * H, dtype=F16)
    wide[:, :H], wide[:, H:2 * H] = x, res
    m.add_rms_norm(wide[:, :H], w, wide[:, H:2 * H], out=wide[:, 2 * H:], residual_out=wide[:, H:2 * H])
    assert torch.equal(wide[:, 2 * H:], y) and torch.equal(wide[:, H:2 * H], h) and torch.equal(wide[:, :H], x)

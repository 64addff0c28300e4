"""Oracle of the norm with the residual's addition — TEST INFRASTRUCTURE ONLY.

``add_rms_norm`` and its gradient from their formulas in fp64, on the device of the inputs. The
product (``muxi_race_b200``) never imports it.
"""
from __future__ import annotations

import torch


def rms_norm_ref(x, weight, residual=None, eps=1e-6):
    """(y, h) in fp64: h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight."""
    h = x.double() if residual is None else x.double() + residual.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double(), h


def rms_norm_grad_ref(dy, h, weight, dh=None, eps=1e-6):
    """(dx, dweight, |dx| bound, |dweight| bound) in fp64; the bounds are the same sums with every
    term's magnitude, the scale that fp32 rounding errors of the kernel are relative to."""
    dy, h, w = dy.double(), h.double(), weight.double()
    r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    xh, g = h * r, dy * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    mag = r * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx, mag = dx + dh.double(), mag + dh.double().abs()
    t = (dy * xh).reshape(-1, h.shape[-1])
    return dx, t.sum(0), mag, t.abs().sum(0)

"""Oracle of the 4-bit weights and their products — TEST INFRASTRUCTURE ONLY.

The weights ``s (q - z)`` and the sums from their definition in fp64, on the device of the inputs.
The product (``muxi_race_b200``) never imports it.
"""
from __future__ import annotations

import torch


def w4_values_ref(q, scales, zeros, K, group):
    """fp64 weights [..., N, K] of q [..., N, ceil(K/2)], scales and zeros [..., N, ceil(K/group)]."""
    v = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2)[..., :K].double()
    at = torch.arange(K, device=q.device) // group
    z = 8.0 if zeros is None else zeros.double()[..., at]
    return (v - z) * scales.double()[..., at]


def linear_ref(x, w):
    """(x W^T, |x| |W|^T) in fp64: the result and the scale of its rounding errors."""
    return x.double() @ w.mT, x.double().abs() @ w.abs().mT


def experts_ref(x, w13, w2, ids, weights, u, f32):
    """(out, tolerance) in fp64: out[t] = sum_j weights[t, j] Down(silu(Gate x) * Up x). The
    tolerance follows an error of ``f32`` relative to each sum's magnitude and a rounding ``u`` of h."""
    T, k = ids.shape
    E, H, I = w2.shape
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(out)
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        s, m = linear_ref(x[t], w13[e])
        g, up, dg, du = s[:, :I], s[:, I:], f32 * m[:, :I], f32 * m[:, I:]
        silu = g * torch.sigmoid(g)
        h = silu * up
        dh = 1.1 * dg * (up.abs() + du) + silu.abs() * du + (u + 1e-5) * h.abs()
        y, my = linear_ref(h, w2[e])
        dy = dh @ w2[e].abs().mT + f32 * my
        w = weights.double()[t, j, None]
        out.index_add_(0, t, w * y)
        tol.index_add_(0, t, w.abs() * dy)
    return out, tol + u * out.abs()

"""fp64 restatement of the operators that train the experts: products grouped by expert and their gradients, the
activation and its gradient, and rows in 8 bits (test infrastructure only)."""
import torch

GROUP = 128


def grouped_ref(x, w, offsets):
    """(y, sum of the terms' magnitudes) of y[r] = w[e] x[r]; 0 for rows of no expert."""
    ends = offsets.tolist()
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        xe, we = x[a:b].double(), w[e].double()
        y[a:b], mag[a:b] = xe @ we.T, xe.abs() @ we.abs().T
    return y, mag


def grouped_dw_ref(dy, x, offsets):
    """(dw, sum of the terms' magnitudes) of dw[e] = sum of dy[r] x[r]^T over e's rows."""
    ends = offsets.tolist()
    E = len(ends) - 1
    dw = torch.zeros(E, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(dw)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        d, xe = dy[a:b].double(), x[a:b].double()
        dw[e], mag[e] = d.T @ xe, d.abs().T @ xe.abs()
    return dw, mag


def silu_mul_ref(gate_up, weights=None):
    g, u = gate_up.double().chunk(2, -1)
    h = g * torch.sigmoid(g) * u
    return h if weights is None else h * weights.double()[..., None]


def silu_mul_grad_ref(dh, gate_up, weights=None):
    """(dgate_up, dweights, magnitudes of the two) by the formulas."""
    g, u = gate_up.double().chunk(2, -1)
    d = dh.double()
    s = torch.sigmoid(g)
    t = d if weights is None else d * weights.double()[..., None]
    dg, du = t * u * s * (1 + g * (1 - s)), t * g * s
    mag_g = (t * u).abs() * s * (1 + g.abs() * (1 - s))
    dw = d * g * s * u
    return torch.cat((dg, du), -1), dw.sum(-1), torch.cat((mag_g, du.abs()), -1), dw.abs().sum(-1)


def rows8_ref(x, kind, parts=1):
    """(values, scales) in fp64 that rows x [R, W] stand for in 8 bits; NaN for a group that holds NaN or an infinity."""
    R, W = x.shape
    v = x.double().reshape(R * parts, W // parts)
    pad = -v.shape[1] % GROUP
    v = torch.nn.functional.pad(v, (0, pad)).reshape(R * parts, -1, GROUP)
    amax = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    v, amax = torch.where(bad, 0.0, v), torch.where(bad, 1.0, amax)
    safe = torch.where(amax > 0, amax, 1.0)
    if kind == torch.int8:
        scale = amax / torch.full_like(amax, 127)
        code = v * 127 / safe
        code = torch.sign(code) * torch.floor(code.abs() + 0.5)
    else:
        m, e = torch.frexp(safe)  # 448 = 0.875 * 2^9
        scale = torch.ldexp(torch.ones_like(safe), torch.where(m <= 0.875, e - 9, e - 8))
        code = v / scale
        _, ce = torch.frexp(code)
        step = torch.ldexp(torch.ones_like(code), (ce - 1).clamp_min(-6) - 3)
        code = torch.round(code / step) * step
        # not out of the type's range: 256 scale would be
        out = code.abs() * scale > torch.finfo(x.dtype).max
        code = torch.where(out, torch.sign(code) * 240, code)
        scale = torch.where(amax > 0, scale, 0.0)
    values = torch.where(bad, float("nan"), code * scale).reshape(R * parts, -1)[:, :W // parts].reshape(R, W)
    return values, torch.where(bad, float("nan"), scale).reshape(R, -1)

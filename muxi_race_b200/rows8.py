"""The activation between the experts' two products, and 8-bit copies of rows for the backward pass.

``silu_mul`` is ``h = weight * silu(gate) * up`` with its gradient. What a backward pass reads again, such
as ``gate_up`` or a layer's input, can be kept as :class:`Rows8`: int8 or e4m3 values with one fp32 scale for
each 128 columns of a row, half of the memory of 16-bit rows.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._args import FLOATS, HALVES, IDS, launch, once_differentiable, overlap, pitch, require, rows, without_gradient

GROUP = 128
Q_DTYPES = {torch.int8: _lib.MOE_I8, torch.float8_e4m3fn: _lib.MOE_F8E4M3}


def groups_of(width: int, parts: int) -> int:
    """Scales of a row."""
    return parts * -(-(width // parts) // GROUP)


@dataclass
class Rows8:
    """16-bit rows [..., W] in 8 bits. They stand for ``q * scale`` of their group, rounded to ``dtype``."""

    q: torch.Tensor      # [..., W] int8 or e4m3, contiguous
    scale: torch.Tensor  # [..., parts * ceil(W / parts / 128)] fp32, contiguous
    dtype: torch.dtype   # fp16 or bf16, of the rows that were saved
    parts: int = 1       # equal parts of a row with groups of their own (2: gate and up)

    def __post_init__(self):
        q, scale = self.q, self.scale
        if q.dtype not in Q_DTYPES or not q.is_contiguous() or q.dim() < 1:
            raise ValueError("q must be a contiguous int8 or float8_e4m3fn tensor [..., W]")
        W = q.shape[-1]
        if self.parts < 1 or W % self.parts:
            raise ValueError("parts must divide the row length")
        if (scale.dtype != torch.float32 or not scale.is_contiguous() or scale.device != q.device
                or scale.shape != (*q.shape[:-1], groups_of(W, self.parts))):
            raise ValueError(f"scale must be a contiguous fp32 tensor {(*q.shape[:-1], groups_of(W, self.parts))} on {q.device}")
        require(self.dtype in HALVES, "dtype must be fp16 or bf16")

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    @property
    def device(self) -> torch.device:
        return self.q.device

    def nbytes(self) -> int:
        return self.q.numel() + 4 * self.scale.numel()


def _check_half(t: torch.Tensor, name: str) -> int:
    dt = HALVES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name} must be fp16 or bf16, got {t.dtype}")
    return dt


def _empty_rows8(shape, parts: int, q_dtype: torch.dtype, dtype: torch.dtype, dev: torch.device) -> Rows8:
    require(q_dtype in Q_DTYPES, "q_dtype must be torch.int8 or torch.float8_e4m3fn")
    *lead, W = shape
    return Rows8(torch.empty(shape, dtype=q_dtype, device=dev),
                 torch.empty((*lead, groups_of(W, parts)), dtype=torch.float32, device=dev), dtype, parts)


def save_rows8(x: torch.Tensor, q_dtype: torch.dtype = torch.int8, parts: int = 1) -> Rows8:
    """8-bit copy of rows x [..., W] fp16 / bf16 (of any one pitch).

    ``torch.int8``: scale = amax / 127 of each 128 columns, values rounded to nearest, halves away from zero.
    ``torch.float8_e4m3fn``: the scale is the smallest power of two with 448 scale >= amax. A group that holds NaN
    or an infinity comes back as NaN. Not differentiable: a backward pass that meets the result raises.
    """
    x2 = rows(x, "x")
    dt = _check_half(x, "x")
    R, W = x2.shape
    require(W >= 1, "x must have at least one column")
    require(parts >= 1 and W % parts == 0, "parts must divide the row length")
    r = _empty_rows8(x.shape, parts, q_dtype, x.dtype, x.device)
    launch(x.device, "moe_save_rows8", x2.data_ptr(), pitch(x2), r.q.data_ptr(), Q_DTYPES[q_dtype], r.scale.data_ptr(), R, W,
           parts, dt)
    if torch.is_grad_enabled() and x.requires_grad:
        # the scales carry the node: every use of the copy reads them
        r.scale, = without_gradient("save_rows8", (r.scale,), x)
    return r


def restore_rows8(saved: Rows8, index: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The 16-bit rows that `saved` stands for; with ``index`` [R] int32 / int64, rows ``index[r]`` of a 2-D copy
    (zeros where that is no row). Not differentiable."""
    require(saved.q.is_cuda, "saved rows must be CUDA tensors")
    dev, W = saved.device, saved.shape[-1]
    q = saved.q
    src_rows = q.numel() // W if W else 0
    if index is None:
        shape, R, idx = q.shape, src_rows, (None, _lib.MOE_I32)
    else:
        if q.dim() != 2:
            raise ValueError("index needs rows [T, W]")
        if index.dim() != 1 or index.dtype not in IDS or index.device != dev or not index.is_contiguous():
            raise ValueError(f"index must be a contiguous int32 or int64 tensor [R] on {dev}")
        R = index.shape[0]
        shape, idx = (R, W), (index.data_ptr(), IDS[index.dtype])
    if out is None:
        out = torch.empty(shape, dtype=saved.dtype, device=dev)
    else:
        require(tuple(out.shape) == tuple(shape) and out.dtype == saved.dtype and out.is_contiguous() and out.device == dev,
                f"out must be a contiguous {saved.dtype} tensor {tuple(shape)} on {dev}")
        flat = out.view(1, -1)
        for t in (q, saved.scale, index):
            require(t is None or not overlap(flat, t.view(1, -1)), "out must not share memory with the saved rows or the index")
    launch(dev, "moe_restore_rows", q.data_ptr(), W, Q_DTYPES[q.dtype], saved.scale.data_ptr(), *idx, 1, None, out.data_ptr(),
           R, src_rows, W, saved.parts, HALVES[saved.dtype])
    return without_gradient("restore_rows8", (out,), saved.scale)[0]


# ----------------------------------------------------------------------------- silu(gate) * up
def _weights_args(weights: Optional[torch.Tensor], R: int, dev: torch.device):
    if weights is None:
        return None, 0
    if weights.dtype not in FLOATS or weights.numel() != R or weights.device != dev or not weights.is_contiguous():
        raise ValueError(f"row_weights must be a contiguous fp32, fp16 or bf16 tensor of {R} weights on {dev}")
    return weights.data_ptr(), FLOATS[weights.dtype]


def _check_gate_up(gate_up: torch.Tensor) -> int:
    I = gate_up.shape[-1] // 2
    require(I >= 1 and gate_up.shape[-1] == 2 * I, "gate_up must be [..., 2 I]")
    return I


def silu_forward(gate_up, weights, q_dtype, at=None, valid=None):
    """(h, Rows8 or None) of gate_up [..., 2 I]. at: weights are taken at at[r], valid: pointer to the number of
    rows (rows behind it stay uninitialised)."""
    g2 = rows(gate_up, "gate_up")
    dt = _check_half(gate_up, "gate_up")
    I = _check_gate_up(gate_up)
    R, dev = g2.shape[0], gate_up.device
    w_ptr, w_dt = _weights_args(weights, R, dev) if at is None else (weights.data_ptr(), FLOATS[weights.dtype])
    h = torch.empty((*gate_up.shape[:-1], I), dtype=gate_up.dtype, device=dev)
    saved = None if q_dtype is None else _empty_rows8(gate_up.shape, 2, q_dtype, gate_up.dtype, dev)
    q_args = (None, 0, None) if saved is None else (saved.q.data_ptr(), Q_DTYPES[q_dtype], saved.scale.data_ptr())
    launch(dev, "moe_silu_mul", g2.data_ptr(), pitch(g2), w_ptr, w_dt, None if at is None else at.data_ptr(),
           0 if weights is None else weights.numel(), valid, h.data_ptr(), *q_args, R, I, dt)
    return h, saved


def silu_backward(dh, gate_up, weights, dweights, at=None, valid=None):
    """(dgate_up, h); dweights, if any, is filled in."""
    d2 = rows(dh, "dh")
    dt = _check_half(dh, "dh")
    dev = dh.device
    if isinstance(gate_up, Rows8):
        require(gate_up.parts == 2 and gate_up.dtype == dh.dtype, "saved gate_up must have parts = 2 and the dtype of dh")
        g_args = (gate_up.q.data_ptr(), gate_up.shape[-1], Q_DTYPES[gate_up.q.dtype], gate_up.scale.data_ptr())
    else:
        g2 = rows(gate_up, "gate_up", dev)
        require(gate_up.dtype == dh.dtype, "gate_up must have the dtype of dh")
        g_args = (g2.data_ptr(), pitch(g2), dt, None)
    if gate_up.device != dev:
        raise ValueError(f"gate_up must be on {dev}")
    I = dh.shape[-1]
    if I < 1 or tuple(gate_up.shape) != (*dh.shape[:-1], 2 * I):
        raise ValueError(f"gate_up must be {(*dh.shape[:-1], 2 * I)}, twice as wide as dh")
    R = d2.shape[0]
    w_ptr, w_dt = _weights_args(weights, R, dev) if at is None else (weights.data_ptr(), FLOATS[weights.dtype])
    dgate_up = torch.empty(gate_up.shape, dtype=dh.dtype, device=dev)
    h = torch.empty(dh.shape, dtype=dh.dtype, device=dev)
    launch(dev, "moe_silu_mul_backward", d2.data_ptr(), pitch(d2), *g_args, w_ptr, w_dt, None if at is None else at.data_ptr(),
           0 if weights is None else weights.numel(), valid, dgate_up.data_ptr(), h.data_ptr(),
           None if dweights is None else dweights.data_ptr(), R, I, dt)
    return dgate_up, h


class _SiluMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up, row_weights, q_dtype):
        h, saved = silu_forward(gate_up, row_weights, q_dtype)
        if saved is None:
            ctx.save_for_backward(gate_up, None, row_weights)
        else:
            ctx.save_for_backward(saved.q, saved.scale, row_weights)
        return h

    @staticmethod
    def backward(ctx, dh):
        a, scale, row_weights = ctx.saved_tensors
        gate_up = a if scale is None else Rows8(a, scale, dh.dtype, 2)
        dgate_up, dweights, _ = silu_mul_backward(dh.contiguous(), gate_up, row_weights)
        grads = once_differentiable("silu_mul", (dgate_up,) if dweights is None else (dgate_up, dweights), dh, a, row_weights)
        return grads[0], (grads[1] if dweights is not None else None), None


def silu_mul(gate_up: torch.Tensor, row_weights: Optional[torch.Tensor] = None, save: Optional[torch.dtype] = None) -> torch.Tensor:
    """``h = row_weight * silu(gate) * up`` of gate_up [..., 2 I] fp16 / bf16 (gate columns first; rows of any one pitch).

    row_weights: one per row, fp32 / fp16 / bf16 (the routing weights of the experts' rows), 1 without.
    Differentiable once in gate_up and row_weights. ``save=torch.int8`` or ``torch.float8_e4m3fn``: the backward pass
    works from an 8-bit copy (:func:`save_rows8`, made in the same pass) instead of gate_up itself.
    """
    require(save is None or save in Q_DTYPES, "save must be None, torch.int8 or torch.float8_e4m3fn")
    if torch.is_grad_enabled() and (gate_up.requires_grad or (row_weights is not None and row_weights.requires_grad)):
        return _SiluMul.apply(gate_up, row_weights, save)
    return silu_forward(gate_up, row_weights, None)[0]


def silu_mul_rows8(gate_up: torch.Tensor, row_weights: Optional[torch.Tensor] = None, q_dtype: torch.dtype = torch.int8):
    """:func:`silu_mul` and the 8-bit copy of gate_up that :func:`silu_mul_backward` takes, in one pass: ``(h, Rows8)``.
    Not differentiable (``silu_mul(..., save=)`` is)."""
    require(q_dtype in Q_DTYPES, "q_dtype must be torch.int8 or torch.float8_e4m3fn")
    h, saved = silu_forward(gate_up, row_weights, q_dtype)
    if torch.is_grad_enabled():
        h, saved.scale = without_gradient("silu_mul_rows8", (h, saved.scale), gate_up, row_weights)
    return h, saved


def silu_mul_backward(dh: torch.Tensor, gate_up, row_weights: Optional[torch.Tensor] = None):
    """Gradients of :func:`silu_mul` from dh [..., I] and gate_up [..., 2 I], a tensor or :class:`Rows8` with two parts:
    ``(dgate_up, drow_weights or None, h)``; h is computed again, for the gradient of the product that read it.

    drow_weights has the dtype and shape of row_weights and a fixed summation order.
    """
    dweights = None if row_weights is None else torch.empty_like(row_weights)
    dgate_up, h = silu_backward(dh, gate_up, row_weights, dweights)
    return dgate_up, dweights, h

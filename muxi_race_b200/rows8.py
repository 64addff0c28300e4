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
from ._args import FLOATS, HALVES, IDS, empty_of, graph_link, launch, matrix, no_tangents, once_differentiable, overlap, require, without_gradient

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
    W = shape[-1]
    r = Rows8.__new__(Rows8)  # what __post_init__ checks holds
    r.q = empty_of(shape, q_dtype, dev)
    r.scale = empty_of((*shape[:-1], groups_of(W, parts)), torch.float32, dev)
    r.dtype, r.parts = dtype, parts
    return r


def save_rows8(x: torch.Tensor, q_dtype: torch.dtype = torch.int8, parts: int = 1) -> Rows8:
    """8-bit copy of rows x [..., W] fp16 / bf16 (of any one pitch).

    ``torch.int8``: scale = amax / 127 of each 128 columns, values rounded to nearest, halves away from zero.
    ``torch.float8_e4m3fn``: the scale is the smallest power of two with 448 scale >= amax; values that would round
    beyond x's type stay at 240 scale. A group that holds NaN or an infinity comes back as NaN.
    Not differentiable: a backward pass that meets the result raises.
    """
    no_tangents("save_rows8", x)
    R, W, ld, ptr = matrix(x, "x")
    dt = _check_half(x, "x")
    if W < 1 or parts < 1 or W % parts:
        raise ValueError("x must have at least one column, and parts must divide the row length")
    if q_dtype not in Q_DTYPES:
        raise ValueError("q_dtype must be torch.int8 or torch.float8_e4m3fn")
    dev = x.device
    r = _empty_rows8(x.shape, parts, q_dtype, x.dtype, dev)
    launch(dev, "moe_save_rows8", ptr, ld, r.q.data_ptr(), Q_DTYPES[q_dtype], r.scale.data_ptr(), R, W, parts, dt)
    if torch.is_grad_enabled() and x.requires_grad:
        # the scales carry the node, and restore_rows8 hands it on
        r.scale, = without_gradient("save_rows8", (r.scale,), x)
    return r


def restore_rows8(saved: Rows8, index: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The 16-bit rows that `saved` stands for; with ``index`` [R] int32 / int64, rows ``index[r]`` of a 2-D copy
    (zeros where that is no row). Not differentiable: a backward pass that meets the result of a copy of rows that need a
    gradient raises (``out`` carries no graph)."""
    q, scale, dtype = saved.q, saved.scale, saved.dtype
    no_tangents("restore_rows8", scale)
    if not q.is_cuda:
        raise ValueError("saved rows must be CUDA tensors")
    dev, shape = q.device, q.shape
    W = shape[-1]
    R = src_rows = q.numel() // W if W else 0
    index_ptr, index_dt = None, 0
    if index is not None:
        if len(shape) != 2:
            raise ValueError("index needs rows [T, W]")
        if index.dim() != 1 or index.dtype not in IDS or index.device != dev or not index.is_contiguous():
            raise ValueError(f"index must be a contiguous int32 or int64 tensor [R] on {dev}")
        R = index.shape[0]
        shape, index_ptr, index_dt = (R, W), index.data_ptr(), IDS[index.dtype]
    given = out is not None
    if not given:
        out = empty_of(shape, dtype, dev)
    else:
        require(tuple(out.shape) == tuple(shape) and out.dtype == dtype and out.is_contiguous() and out.device == dev,
                f"out must be a contiguous {dtype} tensor {tuple(shape)} on {dev}")
        flat = out.view(1, -1)
        for t in (q, scale, index):
            require(t is None or not overlap(flat, t.view(1, -1)), "out must not share memory with the saved rows or the index")
    launch(dev, "moe_restore_rows", q.data_ptr(), W, Q_DTYPES[q.dtype], scale.data_ptr(), index_ptr, index_dt, 1, None,
           out.data_ptr(), R, src_rows, W, saved.parts, HALVES[dtype])
    if given or not scale.requires_grad:
        return out
    return without_gradient("restore_rows8", (out,), scale)[0]


# ----------------------------------------------------------------------------- silu(gate) * up
def _weights_args(weights: Optional[torch.Tensor], R: int, dev: torch.device):
    if weights is None:
        return None, 0
    if weights.dtype not in FLOATS or weights.numel() != R or weights.device != dev or not weights.is_contiguous():
        raise ValueError(f"row_weights must be a contiguous fp32, fp16 or bf16 tensor of {R} weights on {dev}")
    return weights.data_ptr(), FLOATS[weights.dtype]


def silu_forward(gate_up, weights, q_dtype, at=None, valid=None):
    """(h, Rows8 or None) of gate_up [..., 2 I]. at: weights are taken at at[r], valid: pointer to the number of
    rows (rows behind it stay uninitialised)."""
    R, W, ld, ptr = matrix(gate_up, "gate_up")
    dt = _check_half(gate_up, "gate_up")
    I = W // 2
    if I < 1 or W != 2 * I:
        raise ValueError("gate_up must be [..., 2 I]")
    dev, shape = gate_up.device, gate_up.shape
    w_ptr, w_dt = _weights_args(weights, R, dev) if at is None else (weights.data_ptr(), FLOATS[weights.dtype])
    h = empty_of((*shape[:-1], I), gate_up.dtype, dev)
    saved, q_args = None, (None, 0, None)
    if q_dtype is not None:
        saved = _empty_rows8(shape, 2, q_dtype, gate_up.dtype, dev)
        q_args = (saved.q.data_ptr(), Q_DTYPES[q_dtype], saved.scale.data_ptr())
    launch(dev, "moe_silu_mul", ptr, ld, w_ptr, w_dt, None if at is None else at.data_ptr(),
           0 if weights is None else weights.numel(), valid, h.data_ptr(), *q_args, R, I, dt)
    return h, saved


def silu_backward(dh, gate_up, weights, dweights, at=None, valid=None):
    """(dgate_up, h); dweights, if any, is filled in."""
    R, I, ld_dh, dh_ptr = matrix(dh, "dh")
    dt = _check_half(dh, "dh")
    dev, dtype, shape = dh.device, dh.dtype, gate_up.shape
    if isinstance(gate_up, Rows8):
        if gate_up.parts != 2 or gate_up.dtype != dtype or gate_up.q.get_device() != dev.index:
            raise ValueError(f"saved gate_up must have parts = 2 and the dtype of dh, and be on {dev}")
        g_args = (gate_up.q.data_ptr(), 2 * I, Q_DTYPES[gate_up.q.dtype], gate_up.scale.data_ptr())
    else:
        _, _, ld, ptr = matrix(gate_up, "gate_up", dev.index)
        if gate_up.dtype != dtype:
            raise ValueError("gate_up must have the dtype of dh")
        g_args = (ptr, ld, dt, None)
    if I < 1 or shape[-1] != 2 * I or shape[:-1] != dh.shape[:-1]:
        raise ValueError(f"gate_up must be {(*dh.shape[:-1], 2 * I)}, twice as wide as dh")
    w_ptr, w_dt = _weights_args(weights, R, dev) if at is None else (weights.data_ptr(), FLOATS[weights.dtype])
    dgate_up = empty_of(shape, dtype, dev)
    h = empty_of(dh.shape, dtype, dev)
    launch(dev, "moe_silu_mul_backward", dh_ptr, ld_dh, *g_args, w_ptr, w_dt, None if at is None else at.data_ptr(),
           0 if weights is None else weights.numel(), valid, dgate_up.data_ptr(), h.data_ptr(),
           None if dweights is None else dweights.data_ptr(), R, I, dt)
    return dgate_up, h


class _SiluMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up, row_weights, q_dtype, link):
        h, saved = silu_forward(gate_up, row_weights, q_dtype)
        if saved is None:
            ctx.save_for_backward(gate_up, None, row_weights, None)
        else:
            ctx.save_for_backward(saved.q, saved.scale, row_weights, link)
        return h

    @staticmethod
    def backward(ctx, dh):
        a, scale, row_weights, link = ctx.saved_tensors
        gate_up = a if scale is None else Rows8(a, scale, dh.dtype, 2)
        dgate_up, dweights, _ = silu_mul_backward(dh.contiguous(), gate_up, row_weights)
        grads = once_differentiable("silu_mul", (dgate_up,) if dweights is None else (dgate_up, dweights), dh, a, row_weights, link)
        return grads[0], (grads[1] if dweights is not None else None), None, None


def silu_mul(gate_up: torch.Tensor, row_weights: Optional[torch.Tensor] = None, save: Optional[torch.dtype] = None) -> torch.Tensor:
    """``h = row_weight * silu(gate) * up`` of gate_up [..., 2 I] fp16 / bf16 (gate columns first; rows of any one pitch).

    row_weights: one per row, fp32 / fp16 / bf16 (the routing weights of the experts' rows), 1 without. fp32 in between: silu
    of a gate below -88.7, where e^-gate is infinite, is 0.
    Differentiable once in gate_up and row_weights. ``save=torch.int8`` or ``torch.float8_e4m3fn``: the backward pass
    works from an 8-bit copy (:func:`save_rows8`, made in the same pass) instead of gate_up itself.
    """
    require(save is None or save in Q_DTYPES, "save must be None, torch.int8 or torch.float8_e4m3fn")
    no_tangents("silu_mul", gate_up, row_weights)
    if torch.is_grad_enabled() and (gate_up.requires_grad or (row_weights is not None and row_weights.requires_grad)):
        return _SiluMul.apply(gate_up, row_weights, save, None if save is None else graph_link(gate_up))
    return silu_forward(gate_up, row_weights, None)[0]


def silu_mul_rows8(gate_up: torch.Tensor, row_weights: Optional[torch.Tensor] = None, q_dtype: torch.dtype = torch.int8):
    """:func:`silu_mul` and the 8-bit copy of gate_up that :func:`silu_mul_backward` takes, in one pass: ``(h, Rows8)``.
    Not differentiable (``silu_mul(..., save=)`` is)."""
    if q_dtype not in Q_DTYPES:
        raise ValueError("q_dtype must be torch.int8 or torch.float8_e4m3fn")
    no_tangents("silu_mul_rows8", gate_up, row_weights)
    h, saved = silu_forward(gate_up, row_weights, q_dtype)
    if torch.is_grad_enabled() and (gate_up.requires_grad or (row_weights is not None and row_weights.requires_grad)):
        h, saved.scale = without_gradient("silu_mul_rows8", (h, saved.scale), gate_up, row_weights)
    return h, saved


def silu_mul_backward(dh: torch.Tensor, gate_up, row_weights: Optional[torch.Tensor] = None):
    """Gradients of :func:`silu_mul` from dh [..., I] and gate_up [..., 2 I], a tensor or :class:`Rows8` with two parts:
    ``(dgate_up, drow_weights or None, h)``; h is computed again, for the gradient of the product that read it.

    drow_weights has the dtype and shape of row_weights and a fixed summation order.
    """
    no_tangents("silu_mul_backward", dh, gate_up.scale if isinstance(gate_up, Rows8) else gate_up, row_weights)
    dweights = None if row_weights is None else empty_of(row_weights.shape, row_weights.dtype, row_weights.device)
    dgate_up, h = silu_backward(dh, gate_up, row_weights, dweights)
    return dgate_up, dweights, h

"""Root-mean-square norm with the residual's addition, optionally with 8-bit output rows.

The step in front of the router and the experts of an MoE layer: ``h = x + residual``,
``y = h / sqrt(mean(h^2) + eps) * weight``. With ``add_rms_norm_quant`` the normalised rows come out
as int8 or e4m3 with one scale per row, the form that ``fused_moe_int8`` / ``fused_moe_fp8`` read.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._args import FLOATS, launch, once_differentiable, overlap_at, pitch, require, rows, without_gradient
from .fused import _workspace

_Q_DTYPES = {torch.int8: _lib.MOE_I8, torch.float8_e4m3fn: _lib.MOE_F8E4M3}


def _check_weight(weight: torch.Tensor, H: int, dtype: torch.dtype, dev: torch.device) -> int:
    if dtype not in FLOATS:
        raise ValueError(f"x must be fp16, bf16 or fp32, got {dtype}")
    if weight.dim() != 1 or weight.shape[0] != H or weight.device != dev or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous tensor [{H}] on {dev}")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise ValueError("weight must have the dtype of x or fp32")
    return FLOATS[weight.dtype]


def _output(t: Optional[torch.Tensor], x: torch.Tensor, name: str, T: int, *others: tuple):
    """`t`, or a new tensor of x's shape and dtype, with its address and row pitch. `t` may be one of
    `others` (address and pitch of as many rows, T), row for row: a row is read before it is written. It
    may not share memory with them in another way, where a row would be written while another is read
    from the same place."""
    if t is None:
        t = torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)
        return t, t.data_ptr(), x.shape[-1]
    require(t.shape == x.shape and t.dtype == x.dtype, f"{name} must have the shape and dtype of x")
    t2 = rows(t, name, x.device)
    here = ptr, ld = t2.data_ptr(), pitch(t2)
    for o in others:
        if o != here and o[0] is not None and _shared(here, o, T, t2):
            raise ValueError(f"{name} must be x or residual itself, or share no memory with them")
    return t, ptr, ld


def _shared(a: tuple, b: tuple, T: int, like: torch.Tensor) -> bool:
    size = like.element_size()
    row = like.shape[1] * size
    return overlap_at(a[0], a[1] * size, row, T, b[0], b[1] * size, row, T)


def _sum_args(x, x_at, T, residual, residual_out):
    """(h, residual's address and pitch, h's address and pitch); no residual: h is None. x_at: x's address
    and pitch."""
    if residual is None:
        require(residual_out is None, "residual_out needs a residual")
        return None, None, 0, None, 0
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError("residual must have the shape and dtype of x")
    r2 = rows(residual, "residual", x.device)
    r_at = r2.data_ptr(), pitch(r2)
    h, h_ptr, h_ld = _output(residual_out, x, "residual_out", T, x_at, r_at)
    return h, *r_at, h_ptr, h_ld


def _forward(x, weight, residual, eps, out, residual_out):
    x2 = rows(x, "x")
    T, H = x2.shape
    dtype, dev = x2.dtype, x2.device
    wdt = _check_weight(weight, H, dtype, dev)
    x_at = x2.data_ptr(), pitch(x2)
    h, r_ptr, r_ld, h_ptr, h_ld = _sum_args(x, x_at, T, residual, residual_out)
    y, y_ptr, y_ld = _output(out, x, "out", T, x_at, (r_ptr, r_ld))
    if out is not None and residual_out is not None and _shared((y_ptr, y_ld), (h_ptr, h_ld), T, x2):
        raise ValueError("out and residual_out share memory")
    dt = FLOATS[dtype]
    launch(dev, "moe_add_rms_norm", *x_at, r_ptr, r_ld, weight.data_ptr(), wdt, y_ptr, y_ld, dt, None,
           h_ptr, h_ld, T, H, eps, dt)
    return y, h


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, h = _forward(x, weight, residual, eps, None, None)
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.eps, ctx.has_residual = eps, h is not None
        return (y, h) if h is not None else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:  # only the sum was used
            dx, dweight = dh, None
        else:
            dx, dweight = once_differentiable("add_rms_norm", add_rms_norm_backward(
                dy.contiguous(), h, weight, None if dh is None else dh.contiguous(), eps=ctx.eps), dy, dh, h, weight)
        return dx, dweight, (dx if ctx.has_residual else None), None


def add_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    out: Optional[torch.Tensor] = None,
    residual_out: Optional[torch.Tensor] = None,
):
    """``y = rms_norm(x + residual) * weight``; returns ``(y, x + residual)``, or ``y`` without a residual.

    x, residual [..., H] fp16 / bf16 / fp32 with contiguous rows of any one pitch; weight [H] in x's
    dtype or fp32. The sum and the statistics are fp32, y is normalised from the unrounded sum.
    ``out`` and ``residual_out`` may be x or residual themselves (updated in place), but share no other memory
    with them or with each other. Differentiable
    once in x, weight and residual when neither is given.
    """
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        require(out is None and residual_out is None, "out and residual_out are not differentiable")
        return _AddRmsNorm.apply(x, weight, residual, eps)
    y, h = _forward(x, weight, residual, eps, out, residual_out)
    return y if residual is None else (y, h)


def add_rms_norm_quant(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    q_dtype: torch.dtype = torch.int8,
    residual_out: Optional[torch.Tensor] = None,
):
    """:func:`add_rms_norm` with 8-bit rows: ``(q [..., H], scale [...] fp32, x + residual or None)``.

    ``scale = max|y| / 127`` and ``q = round(y / scale)`` for ``torch.int8`` (halves away from zero),
    ``/ 448`` and e4m3 rounding for ``torch.float8_e4m3fn``: the scheme of :func:`quantize_rows_int8`
    / :func:`quantize_rows_fp8`, applied to the unrounded y. x must be fp16 or bf16. Not differentiable: a backward pass that meets the
    results raises (a ``residual_out`` carries no graph).
    """
    require(q_dtype in _Q_DTYPES, "q_dtype must be torch.int8 or torch.float8_e4m3fn")
    x2 = rows(x, "x")
    T, H = x2.shape
    dtype, dev = x2.dtype, x2.device
    wdt = _check_weight(weight, H, dtype, dev)
    q = torch.empty_like(x, dtype=q_dtype, memory_format=torch.contiguous_format)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    x_at = x2.data_ptr(), pitch(x2)
    h, r_ptr, r_ld, h_ptr, h_ld = _sum_args(x, x_at, T, residual, residual_out)
    launch(dev, "moe_add_rms_norm", *x_at, r_ptr, r_ld, weight.data_ptr(), wdt, q.data_ptr(), H,
           _Q_DTYPES[q_dtype], scale.data_ptr(), h_ptr, h_ld, T, H, eps, FLOATS[dtype])
    if residual_out is not None:
        return (*without_gradient("add_rms_norm_quant", (q, scale), x, weight, residual), h)
    return without_gradient("add_rms_norm_quant", (q, scale, h), x, weight, residual)


def add_rms_norm_backward(
    dy: torch.Tensor,
    h: torch.Tensor,
    weight: torch.Tensor,
    dh: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
):
    """Gradients of :func:`add_rms_norm`: ``(dx, dweight)``; dx is the gradient of x and of the residual.

    ``h`` is the sum that the forward returned (x itself without a residual), ``dh`` the gradient that
    reaches it from its other uses. dweight has the weight's dtype and a fixed summation order.
    """
    y2 = rows(dy, "dy")
    h2 = rows(h, "h", y2.device)
    require(dy.shape == h.shape and dy.dtype == h.dtype, "dy and h must have one shape and dtype")
    T, H = h2.shape
    dev = h2.device
    wdt = _check_weight(weight, H, h2.dtype, dev)
    dh_args = (None, 0)
    if dh is not None:
        require(dh.shape == h.shape and dh.dtype == h.dtype, "dh must have the shape and dtype of h")
        d2 = rows(dh, "dh", dev)
        dh_args = (d2.data_ptr(), pitch(d2))
    dx = torch.empty_like(h, memory_format=torch.contiguous_format)
    dweight = torch.empty_like(weight)
    nbytes = _lib.lib().moe_add_rms_norm_backward_workspace_bytes(T, H)
    ws = _workspace(nbytes, dev)
    launch(dev, "moe_add_rms_norm_backward", y2.data_ptr(), pitch(y2), h2.data_ptr(), pitch(h2), *dh_args,
           weight.data_ptr(), wdt, dx.data_ptr(), H, dweight.data_ptr(), T, H, eps, FLOATS[h2.dtype], ws.data_ptr(),
           ws.numel())
    return dx, dweight

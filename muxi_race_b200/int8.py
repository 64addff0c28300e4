"""Dense products of int8 rows with a scale for each row of the activations and of the weights.

What stands next to the int8 experts in a model: shared experts and projections. The rows come from
``add_rms_norm_quant`` or ``quantize_rows_int8``, the weights from ``quantize_rows_int8``.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._args import FLOATS, empty2, launch, matrix, no_tangents, overlap, pitch, require, rows, without_gradient
from .fused import _workspace
from .w4 import _workspace_bytes as workspace_bytes


def int8_linear(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    w: torch.Tensor,
    w_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``y = (x @ w.T) * x_scale * w_scale (+ bias)``: x [..., K] int8 with one fp32 scale per row, w [N, K] int8 with one per
    row (output channel), bias [N] fp32; y [..., N] fp16, bf16 or fp32.

    K is a multiple of 16 below 131072, M and N at most 2^31 - 512; x's rows have any pitch that is a multiple of 16. The sum is
    exact in int32; its conversion to fp32 (above 2^24), the two scales and the bias round in fp32, by 4 * 2^-24 in all, and the
    result is rounded once to its type. ``out`` (rows of any pitch) must not share memory with x. Not differentiable: a
    backward pass that meets the result raises (``out`` carries no graph).
    """
    no_tangents("int8_linear", x_scale, w_scale, bias)
    if w.dim() != 2 or w.dtype != torch.int8 or not w.is_cuda or not w.is_contiguous() or w.data_ptr() % 16:
        raise ValueError("w must be a contiguous int8 CUDA tensor [N, K] that starts on 16 bytes")
    N, K = w.shape
    dev = w.device
    if N < 1 or K < 16 or K % 16 or K >= 1 << 17:
        raise ValueError("w needs at least one row, and K a multiple of 16 below 131072")
    M, width, ld, ptr = matrix(x, "x", dev.index)
    if x.dtype != torch.int8 or width != K:
        raise ValueError(f"x must be int8 [..., {K}]")
    if ptr % 16 or (ld % 16 and M > 1):
        raise ValueError("x must start on 16 bytes, with a row pitch that is a multiple of 16")
    if x_scale.dtype != torch.float32 or x_scale.numel() != M or x_scale.get_device() != dev.index or not x_scale.is_contiguous():
        raise ValueError(f"x_scale must be a contiguous fp32 tensor of {M} scales on {dev}")
    if w_scale.dtype != torch.float32 or w_scale.numel() != N or w_scale.get_device() != dev.index or not w_scale.is_contiguous():
        raise ValueError(f"w_scale must be a contiguous fp32 tensor of {N} scales on {dev}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (N,) or bias.device != dev or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous fp32 tensor [{N}] on {dev}")
    given = out is not None
    if not given:
        if out_dtype not in FLOATS:
            raise ValueError("out_dtype must be fp16, bf16 or fp32")
        out = empty2(M, N, out_dtype, dev)
        if x.dim() != 2:
            out = out.view(*x.shape[:-1], N)
        ld_out = N
    else:
        require(tuple(out.shape) == (*x.shape[:-1], N) and out.dtype in FLOATS, f"out must be fp16, bf16 or fp32 [..., {N}]")
        out2 = rows(out, "out", dev)
        ld_out = pitch(out2)
        require(M < 2 or ld_out >= N, "rows of out must not overlap")
        for t in (rows(x, "x"), w, x_scale.view(1, -1), w_scale.view(1, -1), bias if bias is None else bias.view(1, -1)):
            require(t is None or not overlap(out2, t), "out must not share memory with the inputs")
    nbytes = workspace_bytes("moe_int8_linear_workspace_bytes", M, N, K) if M > 16 else 0
    ws = _workspace(nbytes, dev) if nbytes else None  # held until the call has been launched
    launch(dev, "moe_int8_linear", ptr, ld, x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(),
           None if bias is None else bias.data_ptr(), out.data_ptr(), ld_out, FLOATS[out.dtype], M, N, K,
           None if ws is None else ws.data_ptr(), nbytes)
    return out if given else without_gradient("int8_linear", (out,), x_scale, w_scale, bias)[0]

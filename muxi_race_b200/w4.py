"""4-bit weights with group scales: the products of a decode step, dense and per expert.

``W[n, k] = scales[n, g] * (q[n, k] - zeros[n, g])`` with ``g = k // group_size``, q in 0..15 and
zeros in 0..16 (8 where there are none). A weight is laid out once, when the model is loaded
(:func:`pack_w4` from a checkpoint's values, :func:`quantize_w4` from 16-bit weights), as the stream
of tiles that the kernels read.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from ._args import FLOATS, HALVES, IDS, empty2, launch, no_tangents, overlap, pitch, require, rows, without_gradient
from .fused import _workspace


@lru_cache(maxsize=1024)
def _workspace_bytes(name: str, *sizes: int) -> int:
    """What entry point `name` says of these sizes, asked once for each (a call counts its microseconds)."""
    return getattr(_lib.lib(), name)(*sizes)


@dataclass
class W4Weights:
    """4-bit weights of one or more [out_features, in_features] matrices in the kernels' layout."""

    packed: torch.Tensor  # uint8, moe_w4_packed_bytes
    shape: tuple          # (*lead, out_features, in_features)
    dtype: torch.dtype    # of the scales, and of the activations it is used with
    group_size: int
    has_zeros: bool
    gate_up: bool         # gate rows and up rows interleaved, for fused_moe_w4

    def __post_init__(self):
        *lead, N, K = self.shape
        matrices = 1
        for n in lead:
            matrices *= n
        _check_group(self.group_size)
        want = _lib.lib().moe_w4_packed_bytes(matrices, N, K, self.group_size, int(self.has_zeros), int(self.gate_up))
        require(self.packed.dtype == torch.uint8 and self.packed.is_contiguous() and self.packed.numel() == want,
                f"packed must be a contiguous uint8 tensor of {want} bytes for this shape")
        require(self.dtype in HALVES, "dtype must be fp16 or bf16")

    def nbytes(self) -> int:
        return self.packed.numel()


def _check_group(group_size: int) -> None:
    require(group_size in (32, 64, 128), "group_size must be 32, 64 or 128")


def pack_w4(
    q: torch.Tensor,
    scales: torch.Tensor,
    zeros: Optional[torch.Tensor] = None,
    in_features: Optional[int] = None,
    group_size: int = 128,
    gate_up: bool = False,
) -> W4Weights:
    """Lay out 4-bit weights: q [..., N, ceil(K / 2)] uint8 (column 2i in the low half of byte i),
    scales [..., N, ceil(K / group_size)] fp16 / bf16, zeros (optional) uint8 of the scales' shape, 0..16
    (16 comes from checkpoints that store z - 1 in 4 bits; the zero points are checked, which waits for the GPU).

    ``in_features``: K, where it is odd (default: twice q's last dimension). ``gate_up``: the rows are
    gate rows followed by as many up rows, for :func:`fused_moe_w4`.
    """
    no_tangents("pack_w4", scales)
    _check_group(group_size)
    require(q.is_cuda and q.dtype == torch.uint8 and q.is_contiguous() and q.dim() >= 2,
            "q must be a contiguous uint8 CUDA tensor [..., N, ceil(K / 2)]")
    *lead, N, half = q.shape
    K = 2 * half if in_features is None else int(in_features)
    require((K + 1) // 2 == half and K >= 1, f"q holds {2 * half} columns, in_features is {K}")
    want = (*lead, N, -(-K // group_size))
    require(scales.device == q.device and scales.dtype in HALVES and scales.is_contiguous() and tuple(scales.shape) == want,
            f"scales must be a contiguous fp16 or bf16 tensor {want} on {q.device}")
    if zeros is not None:
        require(zeros.device == q.device and zeros.dtype == torch.uint8 and zeros.is_contiguous()
                and tuple(zeros.shape) == want, f"zeros must be a contiguous uint8 tensor {want} on {q.device}")
        require(not bool((zeros > 16).any()), "zeros must be in 0..16")
    return _pack(q, scales, zeros, (*lead, N, K), group_size, gate_up)


def _pack(q, scales, zeros, shape, group_size, gate_up) -> W4Weights:
    *lead, N, K = shape
    matrices = 1
    for n in lead:
        matrices *= n
    nbytes = _lib.lib().moe_w4_packed_bytes(matrices, N, K, group_size, int(zeros is not None), int(gate_up))
    require(nbytes > 0 or matrices == 0, _lib.lib().moe_last_error().decode())
    packed = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    launch(q.device, "moe_w4_pack", q.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), matrices, N,
           K, group_size, int(gate_up), packed.data_ptr(), packed.numel())
    return W4Weights(packed, tuple(shape), scales.dtype, group_size, zeros is not None, gate_up)


def quantize_w4(w: torch.Tensor, group_size: int = 128, symmetric: bool = True, gate_up: bool = False) -> W4Weights:
    """Quantise 16-bit weights [..., N, K] to 4 bits, rounding to nearest.

    Symmetric: scale = amax / 7 of the group, values -8..7. Otherwise scale = (max - min) / 15 with a
    zero point, over the group's range widened to hold 0. A group with NaN or an infinity comes back
    without finite values.
    """
    no_tangents("quantize_w4", w)
    _check_group(group_size)
    require(w.is_cuda and w.dtype in HALVES and w.is_contiguous() and w.dim() >= 2,
            "w must be a contiguous fp16 or bf16 CUDA tensor [..., N, K]")
    *lead, N, K = w.shape
    require(K >= 1, "w must have at least one column")
    q = torch.empty((*lead, N, (K + 1) // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((*lead, N, -(-K // group_size)), dtype=w.dtype, device=w.device)
    zeros = None if symmetric else torch.empty(scales.shape, dtype=torch.uint8, device=w.device)
    launch(w.device, "moe_w4_quantize", w.data_ptr(), HALVES[w.dtype], w.numel() // K, K, group_size, q.data_ptr(),
           scales.data_ptr(), None if symmetric else zeros.data_ptr())
    return _pack(q, scales, zeros, w.shape, group_size, gate_up)


def dequantize_w4(w: W4Weights) -> torch.Tensor:
    """The weights as a 16-bit tensor of ``w.shape``, each ``scale * (q - zero)`` rounded once."""
    require(w.packed.is_cuda, "packed weights must be a CUDA tensor")
    *lead, N, K = w.shape
    matrices = 1
    for n in lead:
        matrices *= n
    out = torch.empty(w.shape, dtype=w.dtype, device=w.packed.device)
    launch(w.packed.device, "moe_w4_unpack", w.packed.data_ptr(), HALVES[w.dtype], matrices, N, K, w.group_size,
           int(w.has_zeros), int(w.gate_up), out.data_ptr())
    return out


def w4_linear(x: torch.Tensor, w: W4Weights, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ W.T`` for a few rows x [..., K] (fp16 / bf16, the dtype of the weight's scales).

    Sums in fp32, rounded once. ``out`` must not share memory with x. The weights are read once for up to 16 rows, and again for every 16
    more: for a prompt, ``torch.matmul`` with :func:`dequantize_w4` is the better call. Not differentiable:
    a backward pass that meets the result raises (``out`` carries no graph).
    """
    no_tangents("w4_linear", x)
    if len(w.shape) != 2 or w.gate_up:
        raise ValueError("w must be one matrix, packed without gate_up")
    N, K = w.shape
    dev = w.packed.device
    x2 = rows(x, "x", dev)
    if x2.dtype != w.dtype or x2.shape[1] != K:
        raise ValueError(f"x must be {w.dtype} [..., {K}]")
    M = x2.shape[0]
    given = out is not None
    if not given:
        out = empty2(M, N, w.dtype, dev)
        if x.dim() != 2:
            out = out.view(*x.shape[:-1], N)
        ld_out = N
    else:
        require(tuple(out.shape) == (*x.shape[:-1], N) and out.dtype == w.dtype, f"out must be {w.dtype} [..., {N}]")
        out2 = rows(out, "out", dev)
        # a block may still read rows of x when another stores its columns of them
        require(not overlap(out2, x2), "out must not share memory with x")
        ld_out = pitch(out2)
    nbytes = _workspace_bytes("moe_w4_linear_workspace_bytes", M, N, K, w.group_size, HALVES[w.dtype])
    ws = _workspace(nbytes, dev) if nbytes else None  # held until the call has been launched
    launch(dev, "moe_w4_linear", x2.data_ptr(), pitch(x2), w.packed.data_ptr(), out.data_ptr(), ld_out, M, N, K,
           w.group_size, w.has_zeros, FLOATS[w.dtype], None if ws is None else ws.data_ptr(), nbytes)
    return out if given else without_gradient("w4_linear", (out,), x)[0]


def fused_moe_w4(
    hidden_states: torch.Tensor,
    w13: W4Weights,
    w2: W4Weights,
    topk_ids: torch.Tensor,
    topk_weights: torch.Tensor,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """:func:`fused_moe` with 4-bit experts: w13 [E, 2I, H] packed with ``gate_up``, w2 [E, H, I].

    hidden_states [T, H] in the dtype of the scales (rows of any pitch); topk_ids [T, k] int32 / int64,
    ids outside [0, E) are skipped; topk_weights [T, k] fp32 / fp16 / bf16. Meant for decode batches:
    each chosen expert's weights are read once for up to 8 of its tokens (16 where the experts have
    more than 4 on average). With 8 experts of H = 4096, I = 14336 it is faster than e4m3 experts up to
    about 15 tokens per expert (8: 210 against 291 us, 16: 300 against 293 us) and than fp16 experts up to 32 (480
    against 485 us). The same bits on every run.

    Sums are fp32; h = silu(gate) * up is rounded to the dtype between the two products, as :func:`fused_moe`
    does (in fp16 an h beyond 65504 becomes infinite). The workspace holds T * k rows of fp32 sums of H for
    each slice of I (1.9 GB a slice at T = 8192, k = 8, H = 7168; one slice up to I = 12544 where an expert's
    tokens are taken 8 at a time, up to 5376 where 16) for the length of the call.

    Not differentiable: a backward pass that meets the result raises (``out``
    carries no graph).
    """
    no_tangents("fused_moe_w4", hidden_states, topk_weights)
    if len(w13.shape) != 3 or not w13.gate_up or len(w2.shape) != 3 or w2.gate_up:
        raise ValueError("w13 must be [E, 2I, H] packed with gate_up, w2 [E, H, I] without")
    E, N13, H = w13.shape
    I = N13 // 2
    dev = w13.packed.device
    if tuple(w2.shape) != (E, H, I) or w2.dtype != w13.dtype or w2.packed.device != dev:
        raise ValueError(f"w2 must be {w13.dtype} [{E}, {H}, {I}] on {dev}")
    if hidden_states.dim() != 2 or hidden_states.shape[1] != H or hidden_states.dtype != w13.dtype:
        raise ValueError(f"hidden_states must be {w13.dtype} [T, {H}]")
    x = rows(hidden_states, "hidden_states", dev)
    T = x.shape[0]
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_ids and topk_weights must both be [T, topk]")
    if topk_ids.dtype not in IDS or topk_weights.dtype not in FLOATS:
        raise ValueError("topk_ids must be int32 or int64, topk_weights fp32, fp16 or bf16")
    if topk_ids.device != dev or topk_weights.device != dev or not topk_ids.is_contiguous() or not topk_weights.is_contiguous():
        raise ValueError(f"topk_ids and topk_weights must be contiguous tensors on {dev}")
    k = topk_ids.shape[1]
    given = out is not None
    if not given:
        out = empty2(T, H, w13.dtype, dev)
    else:
        require(tuple(out.shape) == (T, H) and out.dtype == w13.dtype and out.is_contiguous() and out.device == dev, "bad out")
    if T == 0:
        return out
    nbytes = _workspace_bytes("moe_fused_w4_workspace_bytes", T, k, E, H, I, w13.group_size, w2.group_size,
                              HALVES[w13.dtype])
    ws = _workspace(nbytes, dev)
    launch(dev, "moe_fused_w4", x.data_ptr(), pitch(x), w13.packed.data_ptr(), w13.group_size, w13.has_zeros,
           w2.packed.data_ptr(), w2.group_size, w2.has_zeros, topk_ids.data_ptr(), IDS[topk_ids.dtype],
           topk_weights.data_ptr(), FLOATS[topk_weights.dtype], out.data_ptr(), T, H, I, E, k, FLOATS[w13.dtype],
           ws.data_ptr(), ws.numel())
    return out if given else without_gradient("fused_moe_w4", (out,), hidden_states, topk_weights)[0]

"""Token-major fused MoE: routing alignment, grouped gate/up + SiLU, grouped down + top-k combine.

``fused_moe(hidden_states, w_gate_up, w_down, topk_ids, topk_weights)`` is the north-star call:
it builds the expert-grouped, 128-row-padded layout that the reference's ``run_kernel`` receives
pre-built (初审材料/源代码/benchmark/remote_bench.py:82-101), runs the same two GEMM stages
(初审材料/源代码/submission.py:586-641 and 317-357) and folds the weighted sum over each token's
top-k routes into the Stage2 epilogue. Every step is a CUDA kernel of ``libmoe_b200.so``; block
counts stay on the device, so a call never synchronises the host.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._args import no_tangents, overlap

BLOCK_M = 128
_DTYPES = {torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16}
_W_DTYPES = {torch.float32: _lib.MOE_F32, torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16}
_ID_DTYPES = {torch.int32: _lib.MOE_I32, torch.int64: _lib.MOE_I64}


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Scratch buffer of one call, allocated on the device's current stream. Its block goes back to
    PyTorch's caching allocator when the call has been launched, and the next call on that stream
    gets it again behind this one. Not shared between calls: an entry point launches several kernels
    without the interpreter's lock, so two threads on one stream may interleave theirs; and a buffer that is
    allocated during a graph capture belongs to that graph's memory for as long as the graph lives."""
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def clear_workspace_cache() -> None:
    """Nothing to do: no call keeps its workspace. (``torch.cuda.empty_cache()`` returns the allocator's
    unused memory to the device.)"""


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


# ----------------------------------------------------------------------------- alignment
@dataclass
class Alignment:
    """Routing metadata in the reference's layout (remote_bench.py:82-101) plus the permutation."""

    group_sizes: torch.Tensor            # [E] int32
    group_offsets: torch.Tensor          # [E+1] int32
    group_padded_offsets: torch.Tensor   # [E+1] int32
    group_idx_for_bx: torch.Tensor       # [max_blocks] int32 (first num_blocks valid)
    sorted_route_ids: torch.Tensor       # [max_rows] int32 (first padded_rows valid; pad = R)
    route_slot: torch.Tensor             # [R] int32
    meta: torch.Tensor                   # [4] int32: padded rows, blocks, valid routes, 0

    def padded_rows(self) -> int:
        return int(self.meta[0].item())

    def num_blocks(self) -> int:
        return int(self.meta[1].item())


def max_padded_rows(num_routes: int, num_experts: int, block_m: int = BLOCK_M) -> int:
    return int(_lib.lib().moe_max_padded_rows(num_routes, num_experts, block_m))


def moe_align(topk_ids: torch.Tensor, num_experts: int, block_m: int = BLOCK_M) -> Alignment:
    """Device-side routing alignment of the flat ``topk_ids`` (ids outside [0, E) are skipped)."""
    _check(topk_ids.is_cuda and topk_ids.is_contiguous(), "topk_ids must be a contiguous CUDA tensor")
    _check(topk_ids.dtype in _ID_DTYPES, "topk_ids must be int32 or int64")
    dev = topk_ids.device
    R = topk_ids.numel()
    p_max = max_padded_rows(R, num_experts, block_m)
    i32 = dict(dtype=torch.int32, device=dev)
    al = Alignment(
        group_sizes=torch.empty(num_experts, **i32),
        group_offsets=torch.empty(num_experts + 1, **i32),
        group_padded_offsets=torch.empty(num_experts + 1, **i32),
        group_idx_for_bx=torch.empty(max(p_max // block_m, 1), **i32),
        sorted_route_ids=torch.empty(max(p_max, 1), **i32),
        route_slot=torch.empty(max(R, 1), **i32),
        meta=torch.empty(4, **i32),
    )
    nbytes = _lib.lib().moe_align_workspace_bytes(R, num_experts)
    ws = _workspace(nbytes, dev)
    _lib.call(
        "moe_align", topk_ids.data_ptr(), _ID_DTYPES[topk_ids.dtype], R, num_experts, block_m,
        al.group_sizes.data_ptr(), al.group_offsets.data_ptr(), al.group_padded_offsets.data_ptr(),
        al.group_idx_for_bx.data_ptr(), al.sorted_route_ids.data_ptr(), al.route_slot.data_ptr(),
        al.meta.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev),
    )
    return al


# ----------------------------------------------------------------------------- fused fp16/bf16
def _check_fused(hidden_states, w13, w2, topk_ids, topk_weights, int8, q_dtype=torch.int8):
    _check(hidden_states.dim() == 2, "hidden_states must be [T, H]")
    T, H = hidden_states.shape
    _check(w13.dim() == 3 and w2.dim() == 3, "w_gate_up must be [E, 2I, H] and w_down [E, H, I]")
    E, two_i, h2 = w13.shape
    I = two_i // 2
    _check(two_i == 2 * I and h2 == H, f"w_gate_up shape {tuple(w13.shape)} does not match H={H}")
    _check(tuple(w2.shape) == (E, H, I), f"w_down shape {tuple(w2.shape)} != {(E, H, I)}")
    _check(topk_ids.shape == topk_weights.shape and topk_ids.dim() == 2 and topk_ids.shape[0] == T,
           "topk_ids and topk_weights must both be [T, topk]")
    for t in (hidden_states, w13, w2, topk_ids, topk_weights):
        _check(t.is_cuda and t.is_contiguous() and t.device == hidden_states.device,
               "all tensors must be contiguous CUDA tensors on one device")
    _check(hidden_states.dtype in _DTYPES, f"unsupported activation dtype {hidden_states.dtype}")
    if int8:
        _check(w13.dtype == q_dtype and w2.dtype == q_dtype, f"{q_dtype} weights expected")
    else:
        _check(w13.dtype == hidden_states.dtype and w2.dtype == hidden_states.dtype,
               "weights must have the activation dtype")
    _check(topk_ids.dtype in _ID_DTYPES, "topk_ids must be int32 or int64")
    _check(topk_weights.dtype in _W_DTYPES, "topk_weights must be fp32, fp16 or bf16")
    return int(T), int(H), int(I), int(E), int(topk_ids.shape[1])


def _output(out: Optional[torch.Tensor], x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """`out`, or a new tensor of x's shape in `dtype`. A kernel clears the output while others read x."""
    if out is None:
        return torch.empty(x.shape, dtype=dtype, device=x.device)
    _check(out.shape == x.shape and out.dtype == dtype and out.is_contiguous() and out.device == x.device,
           f"bad out: it must be a contiguous {dtype} tensor {tuple(x.shape)} on {x.device}")
    _check(not overlap(out, x), "out must not share memory with hidden_states")
    return out


def _check_scales(w13_scale: torch.Tensor, w2_scale: torch.Tensor, E: int, H: int, I: int, dev: torch.device) -> None:
    for name, t, n in (("w13_scale", w13_scale, E * 2 * I), ("w2_scale", w2_scale, E * H)):
        _check(t.dtype == torch.float32 and t.numel() == n and t.is_contiguous() and t.device == dev,
               f"{name} must be fp32 [E, {n // E}] on {dev}")


def fused_moe(
    hidden_states: torch.Tensor,
    w_gate_up: torch.Tensor,
    w_down: torch.Tensor,
    topk_ids: torch.Tensor,
    topk_weights: torch.Tensor,
    out: Optional[torch.Tensor] = None,
    deterministic: bool = False,
) -> torch.Tensor:
    """out[t] = sum_j topk_weights[t,j] * W_down[e] (silu(W_gate[e] x_t) * W_up[e] x_t), e = topk_ids[t,j].

    hidden_states [T, H] fp16/bf16; w_gate_up [E, 2I, H] (gate rows first, then up rows);
    w_down [E, H, I]; topk_ids [T, k] int32/int64; topk_weights [T, k] fp32/fp16/bf16.
    ``deterministic``: sum each token's k rows in route order in fp32 (``moe_fused_ordered``),
    so repeated calls give identical bits; the default adds them with atomics in Stage2.
    """
    no_tangents("fused_moe", hidden_states, w_gate_up, w_down, topk_weights)
    T, H, I, E, k = _check_fused(hidden_states, w_gate_up, w_down, topk_ids, topk_weights, False)
    out = _output(out, hidden_states, hidden_states.dtype)
    if T == 0:
        return out
    dev = hidden_states.device
    dt = _DTYPES[hidden_states.dtype]
    fn = "moe_fused_ordered" if deterministic else "moe_fused"
    nbytes = getattr(_lib.lib(), fn + "_workspace_bytes")(T, k, E, H, I, dt)
    ws = _workspace(nbytes, dev)
    _lib.call(
        fn, hidden_states.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(), topk_ids.data_ptr(),
        _ID_DTYPES[topk_ids.dtype], topk_weights.data_ptr(), _W_DTYPES[topk_weights.dtype], out.data_ptr(),
        T, H, I, E, k, dt, ws.data_ptr(), ws.numel(), _stream(dev),
    )
    return out


# ----------------------------------------------------------------------------- router
_LOGIT_DTYPES = {torch.float32: _lib.MOE_F32, torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16}


def _check_logits(gating_output: torch.Tensor, T: int, topk: int) -> int:
    _check(gating_output.dim() == 2 and gating_output.shape[0] == T, "gating_output must be [T, E]")
    _check(gating_output.dtype in _LOGIT_DTYPES, "gating_output must be fp32, fp16 or bf16")
    E = int(gating_output.shape[1])
    _check(1 <= topk <= min(E, 32), "topk must be in [1, min(E, 32)]")
    _check(gating_output.is_cuda and gating_output.is_contiguous(), "gating_output must be a contiguous CUDA tensor")
    return E


def fused_topk(
    hidden_states: torch.Tensor,
    gating_output: torch.Tensor,
    topk: int,
    renormalize: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax top-k routing in one kernel: (topk_weights [T, k] fp32, topk_ids [T, k] int32).

    topk_weights = softmax(gating_output)[topk_ids], renormalised to sum 1 per token when
    ``renormalize``; ids in descending logit order, equal logits by ascending expert id.
    ``hidden_states`` only fixes T (the argument order of the usual fused-MoE router helper).
    """
    no_tangents("fused_topk", gating_output)
    T = int(hidden_states.shape[0])
    E = _check_logits(gating_output, T, topk)
    dev = gating_output.device
    ids = torch.empty((T, topk), dtype=torch.int32, device=dev)
    w = torch.empty((T, topk), dtype=torch.float32, device=dev)
    if T:
        _lib.call("moe_router_topk", gating_output.data_ptr(), _LOGIT_DTYPES[gating_output.dtype], T, E, topk,
                  int(bool(renormalize)), ids.data_ptr(), w.data_ptr(), _stream(dev))
    return w, ids


def grouped_topk(
    hidden_states: torch.Tensor,
    gating_output: torch.Tensor,
    topk: int,
    renormalize: bool,
    num_expert_group: int,
    topk_group: int,
    e_score_correction_bias: Optional[torch.Tensor] = None,
    routed_scaling_factor: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Group-limited sigmoid routing in one kernel (the DeepSeek-V3 router):
    (topk_weights [T, k] fp32, topk_ids [T, k] int32).

    Scores s = sigmoid(gating_output); experts are chosen by s + e_score_correction_bias within the
    topk_group best of num_expert_group groups (group score = sum of its two best); weights are s
    at the chosen ids, renormalised when ``renormalize``, times ``routed_scaling_factor``.
    """
    T = int(hidden_states.shape[0])
    no_tangents("grouped_topk", gating_output, e_score_correction_bias)
    _check(gating_output.dim() == 2 and gating_output.shape[0] == T, "gating_output must be [T, E]")
    _check(gating_output.is_cuda and gating_output.is_contiguous(), "gating_output must be a contiguous CUDA tensor")
    _check(gating_output.dtype in _LOGIT_DTYPES, "gating_output must be fp32, fp16 or bf16")
    E = int(gating_output.shape[1])
    bias_ptr = None
    if e_score_correction_bias is not None:
        b = e_score_correction_bias
        _check(b.device == gating_output.device and b.dtype == torch.float32 and b.is_contiguous() and b.numel() == E,
               "e_score_correction_bias must be a contiguous fp32 tensor [E] on the logits' device")
        bias_ptr = b.data_ptr()
    dev = gating_output.device
    ids = torch.empty((T, topk), dtype=torch.int32, device=dev)
    w = torch.empty((T, topk), dtype=torch.float32, device=dev)
    _lib.call("moe_router_grouped_topk", gating_output.data_ptr(), _LOGIT_DTYPES[gating_output.dtype], bias_ptr, T, E,
              num_expert_group, topk_group, topk, int(bool(renormalize)), float(routed_scaling_factor), ids.data_ptr(),
              w.data_ptr(), _stream(dev))
    return w, ids


def fused_moe_router(
    hidden_states: torch.Tensor,
    w_gate_up: torch.Tensor,
    w_down: torch.Tensor,
    gating_output: torch.Tensor,
    topk: int,
    renormalize: bool = True,
    out: Optional[torch.Tensor] = None,
    return_routing: bool = False,
):
    """``fused_moe`` with the routing computed from router logits on the device.

    Same result as ``fused_moe(hidden_states, w_gate_up, w_down, ids, weights)`` with
    ``weights, ids = fused_topk(hidden_states, gating_output, topk, renormalize)``; the router
    kernel also builds the alignment's expert histogram. Returns ``out`` or, with
    ``return_routing``, ``(out, topk_weights, topk_ids)``.
    """
    no_tangents("fused_moe_router", hidden_states, w_gate_up, w_down, gating_output)
    T = int(hidden_states.shape[0])
    E = _check_logits(gating_output, T, topk)
    dev = hidden_states.device
    ids = torch.empty((T, topk), dtype=torch.int32, device=dev)
    w = torch.empty((T, topk), dtype=torch.float32, device=dev)
    T, H, I, E2, k = _check_fused(hidden_states, w_gate_up, w_down, ids, w, False)
    _check(E2 == E, f"gating_output has {E} experts, the weights {E2}")
    _check(gating_output.device == dev, "gating_output must be on the device of hidden_states")
    out = _output(out, hidden_states, hidden_states.dtype)
    if T:
        dt = _DTYPES[hidden_states.dtype]
        nbytes = _lib.lib().moe_fused_workspace_bytes(T, k, E, H, I, dt)
        ws = _workspace(nbytes, dev)
        _lib.call(
            "moe_fused_router", hidden_states.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(),
            gating_output.data_ptr(), _LOGIT_DTYPES[gating_output.dtype], int(bool(renormalize)), ids.data_ptr(),
            w.data_ptr(), out.data_ptr(), T, H, I, E, k, dt, ws.data_ptr(), ws.numel(), _stream(dev),
        )
    return (out, w, ids) if return_routing else out


# ----------------------------------------------------------------------------- W8A8 int8
def quantize_rows_int8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-row symmetric int8: q = round_half_away(w * 127 / amax_row), scale = amax_row / 127.

    ``w`` [..., K] fp16/bf16 (e.g. stacked weights [E, N, K], one scale per output row).
    Returns (q int8 of w's shape, scale fp32 of shape w.shape[:-1]).
    """
    no_tangents("quantize_rows_int8", w)
    _check(w.is_cuda and w.is_contiguous() and w.dtype in _DTYPES, "w must be a contiguous fp16/bf16 CUDA tensor")
    K = w.shape[-1]
    rows = w.numel() // K if K else 0
    q = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    scale = torch.empty(w.shape[:-1], dtype=torch.float32, device=w.device)
    _lib.call("moe_quantize_rows_int8", w.data_ptr(), _DTYPES[w.dtype], rows, K, q.data_ptr(), scale.data_ptr(),
              _stream(w.device))
    return q, scale


def _fused_q8_rows(x_q, x_scale, q_dtype, w13_q, w13_scale, w2_q, w2_scale, topk_ids, topk_weights, out, out_dtype):
    """fused_moe_int8 / fused_moe_fp8 on rows that are 8-bit already."""
    if out_dtype is None:
        out_dtype = torch.bfloat16 if out is None else out.dtype
    _check(out_dtype in _DTYPES, "out_dtype must be fp16 or bf16")
    _check(out is None or out.dtype == out_dtype, "out must have out_dtype")
    _check(x_q.dim() == 2 and x_q.dtype == q_dtype, f"hidden_states must be {q_dtype} [T, H]")
    T, H = x_q.shape
    _check(x_scale.dtype == torch.float32 and x_scale.numel() == T and x_scale.is_contiguous() and x_scale.device == x_q.device,
           "hidden_scale must be contiguous fp32 [T]")
    _check(x_q.is_cuda and x_q.is_contiguous(), "hidden_states must be a contiguous CUDA tensor")
    out = _output(out, x_q, out_dtype)
    _, _, I, E, k = _check_fused(out, w13_q, w2_q, topk_ids, topk_weights, True, q_dtype)
    _check_scales(w13_scale, w2_scale, E, H, I, x_q.device)
    if T == 0:
        return out
    dev, dt = x_q.device, _DTYPES[out.dtype]
    int8 = q_dtype == torch.int8
    nbytes = getattr(_lib.lib(), "moe_fused_int8_workspace_bytes" if int8 else "moe_fused_fp8_workspace_bytes")(T, k, E, H, I, dt)
    ws = _workspace(nbytes, dev)
    _lib.call(
        "moe_fused_q8_rows", x_q.data_ptr(), x_scale.data_ptr(), _lib.MOE_I8 if int8 else _lib.MOE_F8E4M3, w13_q.data_ptr(),
        w13_scale.data_ptr(), w2_q.data_ptr(), w2_scale.data_ptr(), topk_ids.data_ptr(), _ID_DTYPES[topk_ids.dtype],
        topk_weights.data_ptr(), _W_DTYPES[topk_weights.dtype], out.data_ptr(), T, H, I, E, k, dt, ws.data_ptr(), ws.numel(),
        _stream(dev),
    )
    return out


def fused_moe_int8(
    hidden_states: torch.Tensor,
    w13_q: torch.Tensor,
    w13_scale: torch.Tensor,
    w2_q: torch.Tensor,
    w2_scale: torch.Tensor,
    topk_ids: torch.Tensor,
    topk_weights: torch.Tensor,
    out: Optional[torch.Tensor] = None,
    hidden_scale: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """W8A8 ``fused_moe``: int8 weights with per-output-row scales (from :func:`quantize_rows_int8`),
    activations quantised per token on the device, int32 accumulation, output in the activation dtype.

    With ``hidden_scale`` [T] fp32 the rows are int8 already (:func:`add_rms_norm_quant`) and the output
    is in ``out_dtype`` (default: that of ``out``, or bf16), which is for this form only."""
    no_tangents("fused_moe_int8", hidden_states, hidden_scale, w13_scale, w2_scale, topk_weights)
    if hidden_scale is not None:
        return _fused_q8_rows(hidden_states, hidden_scale, torch.int8, w13_q, w13_scale, w2_q, w2_scale, topk_ids,
                              topk_weights, out, out_dtype)
    _check(out_dtype is None, "out_dtype needs hidden_scale: otherwise the output has the dtype of hidden_states")
    T, H, I, E, k = _check_fused(hidden_states, w13_q, w2_q, topk_ids, topk_weights, True)
    _check_scales(w13_scale, w2_scale, E, H, I, hidden_states.device)
    out = _output(out, hidden_states, hidden_states.dtype)
    if T == 0:
        return out
    dev = hidden_states.device
    dt = _DTYPES[hidden_states.dtype]
    nbytes = _lib.lib().moe_fused_int8_workspace_bytes(T, k, E, H, I, dt)
    ws = _workspace(nbytes, dev)
    _lib.call(
        "moe_fused_int8", hidden_states.data_ptr(), w13_q.data_ptr(), w13_scale.data_ptr(), w2_q.data_ptr(),
        w2_scale.data_ptr(), topk_ids.data_ptr(), _ID_DTYPES[topk_ids.dtype], topk_weights.data_ptr(),
        _W_DTYPES[topk_weights.dtype], out.data_ptr(), T, H, I, E, k, dt, ws.data_ptr(), ws.numel(), _stream(dev),
    )
    return out


# ----------------------------------------------------------------------------- W8A8 fp8 (e4m3)
def quantize_rows_fp8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-row e4m3: scale = amax_row / 448, q = e4m3(w * (448 / amax_row)) (nearest even, saturated).

    ``w`` [..., K] fp16/bf16. Returns (q torch.float8_e4m3fn of w's shape, scale fp32 of shape
    w.shape[:-1]).
    """
    no_tangents("quantize_rows_fp8", w)
    _check(w.is_cuda and w.is_contiguous() and w.dtype in _DTYPES, "w must be a contiguous fp16/bf16 CUDA tensor")
    K = w.shape[-1]
    rows = w.numel() // K if K else 0
    q = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=w.device)
    scale = torch.empty(w.shape[:-1], dtype=torch.float32, device=w.device)
    _lib.call("moe_quantize_rows_fp8", w.data_ptr(), _DTYPES[w.dtype], rows, K, q.data_ptr(), scale.data_ptr(),
              _stream(w.device))
    return q, scale


def fused_moe_fp8(
    hidden_states: torch.Tensor,
    w13_q: torch.Tensor,
    w13_scale: torch.Tensor,
    w2_q: torch.Tensor,
    w2_scale: torch.Tensor,
    topk_ids: torch.Tensor,
    topk_weights: torch.Tensor,
    out: Optional[torch.Tensor] = None,
    hidden_scale: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """fp8 ``fused_moe``: e4m3 weights with per-output-row scales (from :func:`quantize_rows_fp8`),
    activations quantised to e4m3 per token on the device, fp32 accumulation, output in the
    activation dtype.

    With ``hidden_scale`` [T] fp32 the rows are e4m3 already (:func:`add_rms_norm_quant`) and the output
    is in ``out_dtype`` (default: that of ``out``, or bf16), which is for this form only."""
    no_tangents("fused_moe_fp8", hidden_states, hidden_scale, w13_scale, w2_scale, topk_weights)
    if hidden_scale is not None:
        return _fused_q8_rows(hidden_states, hidden_scale, torch.float8_e4m3fn, w13_q, w13_scale, w2_q, w2_scale, topk_ids,
                              topk_weights, out, out_dtype)
    _check(out_dtype is None, "out_dtype needs hidden_scale: otherwise the output has the dtype of hidden_states")
    T, H, I, E, k = _check_fused(hidden_states, w13_q, w2_q, topk_ids, topk_weights, True, torch.float8_e4m3fn)
    _check_scales(w13_scale, w2_scale, E, H, I, hidden_states.device)
    out = _output(out, hidden_states, hidden_states.dtype)
    if T == 0:
        return out
    dev = hidden_states.device
    dt = _DTYPES[hidden_states.dtype]
    nbytes = _lib.lib().moe_fused_fp8_workspace_bytes(T, k, E, H, I, dt)
    ws = _workspace(nbytes, dev)
    _lib.call(
        "moe_fused_fp8", hidden_states.data_ptr(), w13_q.data_ptr(), w13_scale.data_ptr(), w2_q.data_ptr(),
        w2_scale.data_ptr(), topk_ids.data_ptr(), _ID_DTYPES[topk_ids.dtype], topk_weights.data_ptr(),
        _W_DTYPES[topk_weights.dtype], out.data_ptr(), T, H, I, E, k, dt, ws.data_ptr(), ws.numel(), _stream(dev),
    )
    return out


def device_status(clear: bool = True) -> int:
    """Device status word of the current device (0 = every kernel completed normally)."""
    import ctypes

    v = ctypes.c_uint32(0)
    dev = torch.cuda.current_device()
    _lib.call("moe_device_status", _stream(torch.device("cuda", dev)), int(clear), ctypes.byref(v))
    return int(v.value)

"""muxi_race_b200 — a B200-native (sm_100a) fused Mixture-of-Experts operator.

Entry points:
  run_kernel(...)      drop-in for the contest operator's ``run_kernel`` (10 tensors, padded layout)
  fused_moe(...)       token-major fused MoE (routing alignment + both GEMM stages + top-k combine)
  fused_moe_int8(...)  W8A8 variant; weights from quantize_rows_int8()
  fused_moe_fp8(...)   fp8 (e4m3) variant; weights from quantize_rows_fp8()
  moe_align(...)       device-side routing metadata
  fused_topk(...)      softmax top-k routing of router logits; fused_moe_router(...) routes + runs
  grouped_topk(...)    group-limited sigmoid routing (DeepSeek-V3 router)
  route_topk(...)      routing in its general form (softmax / sigmoid, bias, groups, masked experts, counts),
                       differentiable; route_topk_backward(...) its gradient
  add_rms_norm(...)    norm with the residual's addition; add_rms_norm_quant(...) with int8 / e4m3 rows;
                       add_rms_norm_backward(...) its gradient (add_rms_norm is differentiable)
  quantize_w4(...), pack_w4(...)  4-bit weights with group scales -> W4Weights; dequantize_w4(...) back
  w4_linear(...)       product of a few rows with 4-bit weights; fused_moe_w4(...) 4-bit experts
  pack_weights(...)    one-buffer weight format (16-bit, int8 or fp8); fused_moe_packed(...) runs on it
  moe_mlp(...)         fused_moe with gradients (tokens, experts' weights, routing weights), optionally from 8-bit copies
  grouped_linear(...)  products grouped by expert with ragged rows, differentiable; grouped_linear_backward(...)
  silu_mul(...)        weight * silu(gate) * up, differentiable; silu_mul_rows8(...), silu_mul_backward(...)
  save_rows8(...)      8-bit copies of rows for a backward pass -> Rows8; restore_rows8(...) back, in any order
  int8_linear(...)     dense product of int8 rows with scales per row and output channel
  host_pipeline.HostPipeline  host-buffer calls with transfers overlapped across calls
  graphs.GraphedMoE    one call captured into a CUDA graph and replayed
  torch_ops            torch.ops.muxi_race_b200.{fused_moe, fused_moe_int8, fused_moe_fp8, fused_topk,
                       run_kernel} (import to register)
  ep.ExpertParallelMoE expert-parallel fused MoE over torch.distributed (NCCL all-to-all)

All compute runs in hand-written CUDA kernels of ``libmoe_b200.so`` (C ABI in
``include/moe_b200.h``); there is no CPU or library fallback.
"""
from .fused import (Alignment, clear_workspace_cache, device_status, fused_moe, fused_moe_fp8, fused_moe_int8,
                    fused_moe_router, fused_topk, grouped_topk, max_padded_rows, moe_align, quantize_rows_fp8,
                    quantize_rows_int8)
from .grouped import grouped_linear, grouped_linear_backward, moe_mlp
from .int8 import int8_linear
from .norm import add_rms_norm, add_rms_norm_backward, add_rms_norm_quant
from .packed import PackedWeights, fused_moe_packed, pack_weights
from .route import route_topk, route_topk_backward
from .rows8 import Rows8, restore_rows8, save_rows8, silu_mul, silu_mul_backward, silu_mul_rows8
from .submission import run_kernel
from .w4 import W4Weights, dequantize_w4, fused_moe_w4, pack_w4, quantize_w4, w4_linear

__all__ = [
    "Alignment", "clear_workspace_cache", "device_status", "fused_moe", "fused_moe_fp8", "fused_moe_int8",
    "fused_moe_router", "fused_topk", "grouped_topk", "max_padded_rows", "moe_align", "quantize_rows_fp8", "quantize_rows_int8",
    "add_rms_norm", "add_rms_norm_backward", "add_rms_norm_quant",
    "route_topk", "route_topk_backward", "run_kernel", "PackedWeights", "fused_moe_packed", "pack_weights",
    "grouped_linear", "grouped_linear_backward", "moe_mlp", "int8_linear",
    "Rows8", "restore_rows8", "save_rows8", "silu_mul", "silu_mul_backward", "silu_mul_rows8",
    "W4Weights", "dequantize_w4", "fused_moe_w4", "pack_w4", "quantize_w4", "w4_linear",
]

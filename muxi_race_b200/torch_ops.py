"""PyTorch operator registrations of the library's entry points (``torch.ops.muxi_race_b200.*``).

Registered as custom ops with shape functions, so models can call them like built-in operators:
they pass through ``torch.compile`` graphs as opaque nodes (the kernels stay this library's),
through CUDA-graph capture, and through meta / fake-tensor shape propagation.

    import muxi_race_b200.torch_ops  # registers the ops
    out = torch.ops.muxi_race_b200.fused_moe(x, w_gate_up, w_down, topk_ids, topk_weights)
    torch.ops.muxi_race_b200.run_kernel(x, gate_w, up_w, down_w, routed, gs, go, gpo, gidx, out)

The eager implementations are the Python entry points of this package (C ABI underneath).
"""
from typing import Optional

import torch
from torch import Tensor

from . import fused as _fused
from . import grouped as _grouped
from . import int8 as _int8
from . import norm as _norm
from . import route as _route
from . import rows8 as _rows8
from . import submission as _submission
from . import w4 as _w4
from ._args import no_tangents as _no_tangents


@torch.library.custom_op("muxi_race_b200::fused_moe", mutates_args=())
def fused_moe(hidden_states: Tensor, w_gate_up: Tensor, w_down: Tensor, topk_ids: Tensor,
              topk_weights: Tensor) -> Tensor:
    return _fused.fused_moe(hidden_states, w_gate_up, w_down, topk_ids, topk_weights)


@fused_moe.register_fake
def _fused_moe_fake(hidden_states, w_gate_up, w_down, topk_ids, topk_weights):
    return hidden_states.new_empty(hidden_states.shape)


@torch.library.custom_op("muxi_race_b200::fused_moe_int8", mutates_args=())
def fused_moe_int8(hidden_states: Tensor, w13_q: Tensor, w13_scale: Tensor, w2_q: Tensor, w2_scale: Tensor,
                   topk_ids: Tensor, topk_weights: Tensor) -> Tensor:
    return _fused.fused_moe_int8(hidden_states, w13_q, w13_scale, w2_q, w2_scale, topk_ids, topk_weights)


@fused_moe_int8.register_fake
def _fused_moe_int8_fake(hidden_states, w13_q, w13_scale, w2_q, w2_scale, topk_ids, topk_weights):
    return hidden_states.new_empty(hidden_states.shape)


@torch.library.custom_op("muxi_race_b200::fused_moe_fp8", mutates_args=())
def fused_moe_fp8(hidden_states: Tensor, w13_q: Tensor, w13_scale: Tensor, w2_q: Tensor, w2_scale: Tensor,
                  topk_ids: Tensor, topk_weights: Tensor) -> Tensor:
    return _fused.fused_moe_fp8(hidden_states, w13_q, w13_scale, w2_q, w2_scale, topk_ids, topk_weights)


@fused_moe_fp8.register_fake
def _fused_moe_fp8_fake(hidden_states, w13_q, w13_scale, w2_q, w2_scale, topk_ids, topk_weights):
    return hidden_states.new_empty(hidden_states.shape)


@torch.library.custom_op("muxi_race_b200::fused_topk", mutates_args=())
def fused_topk(gating_output: Tensor, topk: int, renormalize: bool) -> tuple[Tensor, Tensor]:
    return _fused.fused_topk(gating_output, gating_output, topk, renormalize)


@fused_topk.register_fake
def _fused_topk_fake(gating_output, topk, renormalize):
    T = gating_output.shape[0]
    return (gating_output.new_empty((T, topk), dtype=torch.float32),
            gating_output.new_empty((T, topk), dtype=torch.int32))


@torch.library.custom_op("muxi_race_b200::grouped_topk", mutates_args=())
def grouped_topk(gating_output: Tensor, topk: int, renormalize: bool, num_expert_group: int, topk_group: int,
                 e_score_correction_bias: Optional[Tensor], routed_scaling_factor: float) -> tuple[Tensor, Tensor]:
    return _fused.grouped_topk(gating_output, gating_output, topk, renormalize, num_expert_group, topk_group,
                               e_score_correction_bias, routed_scaling_factor)


@grouped_topk.register_fake
def _grouped_topk_fake(gating_output, topk, renormalize, num_expert_group, topk_group, e_score_correction_bias,
                       routed_scaling_factor):
    T = gating_output.shape[0]
    return (gating_output.new_empty((T, topk), dtype=torch.float32),
            gating_output.new_empty((T, topk), dtype=torch.int32))


@torch.library.custom_op("muxi_race_b200::run_kernel", mutates_args=("out",))
def run_kernel(stacked_expert_tokens: Tensor, gate_w: Tensor, up_w: Tensor, down_w: Tensor,
               routed_expert_weights: Tensor, group_sizes: Tensor, group_offsets: Tensor,
               group_padded_offsets: Tensor, group_idx_for_bx: Tensor, out: Tensor) -> None:
    _submission.run_kernel(stacked_expert_tokens, gate_w, up_w, down_w, routed_expert_weights, group_sizes,
                           group_offsets, group_padded_offsets, group_idx_for_bx, out)


@run_kernel.register_fake
def _run_kernel_fake(stacked_expert_tokens, gate_w, up_w, down_w, routed_expert_weights, group_sizes,
                     group_offsets, group_padded_offsets, group_idx_for_bx, out):
    return None


@torch.library.custom_op("muxi_race_b200::add_rms_norm", mutates_args=())
def add_rms_norm(x: Tensor, weight: Tensor, residual: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    return _norm._forward(x, weight, residual, eps, None, None)


@add_rms_norm.register_fake
def _add_rms_norm_fake(x, weight, residual, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape)


@torch.library.custom_op("muxi_race_b200::add_rms_norm_backward", mutates_args=())
def add_rms_norm_backward(dy: Tensor, h: Tensor, weight: Tensor, dh: Optional[Tensor], eps: float) -> tuple[Tensor, Tensor]:
    return _norm.add_rms_norm_backward(dy, h, weight, dh, eps)


@add_rms_norm_backward.register_fake
def _add_rms_norm_backward_fake(dy, h, weight, dh, eps):
    return h.new_empty(h.shape), weight.new_empty(weight.shape)


@torch.library.custom_op("muxi_race_b200::route_topk", mutates_args=())
def route_topk(logits: Tensor, topk: int, scoring: str, bias: Optional[Tensor], num_groups: int, topk_groups: int,
               group_top: int, renormalize: bool, scale: float) -> tuple[Tensor, Tensor, Tensor]:
    return _route._forward(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale, True)


@route_topk.register_fake
def _route_topk_fake(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale):
    T, E = logits.shape
    return (logits.new_empty((T, topk), dtype=torch.float32), logits.new_empty((T, topk), dtype=torch.int32),
            logits.new_empty((E,), dtype=torch.int32))


@torch.library.custom_op("muxi_race_b200::w4_linear", mutates_args=())
def w4_linear(x: Tensor, packed: Tensor, out_features: int, group_size: int, has_zeros: bool) -> Tensor:
    return _w4.w4_linear(x, _w4.W4Weights(packed, (out_features, x.shape[-1]), x.dtype, group_size, has_zeros, False))


@w4_linear.register_fake
def _w4_linear_fake(x, packed, out_features, group_size, has_zeros):
    return x.new_empty((*x.shape[:-1], out_features))


@torch.library.custom_op("muxi_race_b200::fused_moe_w4", mutates_args=())
def fused_moe_w4(hidden_states: Tensor, w13: Tensor, w2: Tensor, num_experts: int, intermediate: int, group_size13: int,
                 has_zeros13: bool, group_size2: int, has_zeros2: bool, topk_ids: Tensor, topk_weights: Tensor) -> Tensor:
    H, dt = hidden_states.shape[1], hidden_states.dtype
    return _w4.fused_moe_w4(
        hidden_states, _w4.W4Weights(w13, (num_experts, 2 * intermediate, H), dt, group_size13, has_zeros13, True),
        _w4.W4Weights(w2, (num_experts, H, intermediate), dt, group_size2, has_zeros2, False), topk_ids, topk_weights)


@fused_moe_w4.register_fake
def _fused_moe_w4_fake(hidden_states, w13, w2, num_experts, intermediate, group_size13, has_zeros13, group_size2,
                       has_zeros2, topk_ids, topk_weights):
    return hidden_states.new_empty(hidden_states.shape)


@torch.library.custom_op("muxi_race_b200::grouped_linear", mutates_args=())
def grouped_linear(x: Tensor, w: Tensor, offsets: Tensor) -> Tensor:
    _no_tangents("grouped_linear", x, w)
    return _grouped._rows_product("moe_grouped_linear", x, "x", w, offsets, False)


@grouped_linear.register_fake
def _grouped_linear_fake(x, w, offsets):
    return x.new_empty((x.shape[0], w.shape[1]))


@torch.library.custom_op("muxi_race_b200::grouped_linear_backward", mutates_args=())
def grouped_linear_backward(dy: Tensor, x: Tensor, w: Tensor, offsets: Tensor) -> tuple[Tensor, Tensor]:
    return _grouped.grouped_linear_backward(dy, x, w, offsets)


@grouped_linear_backward.register_fake
def _grouped_linear_backward_fake(dy, x, w, offsets):
    return x.new_empty(x.shape), w.new_empty(w.shape)


@torch.library.custom_op("muxi_race_b200::silu_mul", mutates_args=())
def silu_mul(gate_up: Tensor, row_weights: Optional[Tensor]) -> Tensor:
    _no_tangents("silu_mul", gate_up, row_weights)
    return _rows8.silu_forward(gate_up, row_weights, None)[0]


@silu_mul.register_fake
def _silu_mul_fake(gate_up, row_weights):
    return gate_up.new_empty((*gate_up.shape[:-1], gate_up.shape[-1] // 2))


@torch.library.custom_op("muxi_race_b200::int8_linear", mutates_args=())
def int8_linear(x: Tensor, x_scale: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor], out_dtype: torch.dtype) -> Tensor:
    return _int8.int8_linear(x, x_scale, w, w_scale, bias, out_dtype)


@int8_linear.register_fake
def _int8_linear_fake(x, x_scale, w, w_scale, bias, out_dtype):
    return x.new_empty((*x.shape[:-1], w.shape[0]), dtype=out_dtype)

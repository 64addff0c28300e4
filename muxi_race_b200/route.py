"""Routing of tokens to experts in its general form, differentiable: softmax or sigmoid scores, a
selection bias, groups, experts that are switched off, strided logits, tokens per expert.

``fused_topk`` and ``grouped_topk`` are the two fixed forms of serving (contiguous finite logits, no
gradient); :func:`route_topk` covers what they do, training and masked experts. On a B200 it is the faster one,
called by itself (11 against 15 us up to 4096 tokens) and in a graph: 256 experts, top-8, 128 / 32768 tokens 2.8
/ 20 us (``fused_topk`` 3.6 / 42 us), with sigmoid, bias and groups 4.9 / 44 us (``grouped_topk`` 9.8 / 90 us). Of 8 experts,
top-2, ``fused_topk`` takes less in a graph (2.1 / 9.6 against 2.3 / 11.7 us).
"""
from __future__ import annotations

from typing import Optional

import torch

from ._args import FLOATS, empty2, launch, no_tangents, once_differentiable, pitch, require, rows

_SCORING = {"softmax": 0, "sigmoid": 1}


def _forward(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale, counts):
    no_tangents("route_topk", logits, bias)
    l2 = rows(logits, "logits")
    T, E = l2.shape
    dev, dtype = l2.device, l2.dtype
    if logits.dim() != 2 or dtype not in FLOATS:
        raise ValueError("logits must be fp32, fp16 or bf16 [T, E]")
    if scoring not in _SCORING:
        raise ValueError("scoring must be 'softmax' or 'sigmoid'")
    bias_ptr = None
    if bias is not None:
        if bias.device != dev or bias.dtype != torch.float32 or not bias.is_contiguous() or bias.dim() != 1 or bias.shape[0] != E:
            raise ValueError(f"bias must be a contiguous fp32 tensor [{E}] on {dev}")
        bias_ptr = bias.data_ptr()
    ids = empty2(T, topk, torch.int32, dev)
    weights = empty2(T, topk, torch.float32, dev)
    number = torch.empty_strided((E,), (1,), dtype=torch.int32, device=dev) if counts else None
    launch(dev, "moe_route_topk", l2.data_ptr(), pitch(l2), FLOATS[dtype], bias_ptr, T, E, topk, _SCORING[scoring],
           num_groups, topk_groups, group_top, renormalize, scale, ids.data_ptr(), weights.data_ptr(),
           None if number is None else number.data_ptr())
    return weights, ids, number


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale, counts):
        weights, ids, number = _forward(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale,
                                        counts)
        ctx.save_for_backward(logits, ids)
        ctx.how = scoring, renormalize, scale
        ctx.mark_non_differentiable(ids)
        if number is not None:
            ctx.mark_non_differentiable(number)
        return weights, ids, number

    @staticmethod
    def backward(ctx, dweights, *_):
        logits, ids = ctx.saved_tensors
        scoring, renormalize, scale = ctx.how
        dlogits, = once_differentiable("route_topk", (route_topk_backward(
            dweights, logits, ids, scoring=scoring, renormalize=renormalize, scale=scale),), dweights, logits)
        return (dlogits, *[None] * 9)


def route_topk(
    logits: torch.Tensor,
    topk: int,
    scoring: str = "softmax",
    bias: Optional[torch.Tensor] = None,
    num_groups: int = 1,
    topk_groups: int = 1,
    group_top: int = 2,
    renormalize: bool = True,
    scale: float = 1.0,
    return_counts: bool = False,
):
    """``(topk_weights [T, k] fp32, topk_ids [T, k] int32)``, and with ``return_counts`` the number of
    tokens of each expert ([E] int32).

    logits [T, E] fp32 / fp16 / bf16, rows of any pitch. Scores are ``softmax(logits)`` or
    ``sigmoid(logits)``; the ``topk`` largest ``score + bias`` are chosen (bias [E] fp32, for balance:
    it moves the choice only) among the experts of the ``topk_groups`` best of ``num_groups`` groups,
    a group counting the sum of its ``group_top`` (1 or 2) best (-inf where fewer are eligible). Ids come in descending order, equal
    ones by the lower id (without bias and groups the order is that of the logits, which tells experts apart whose
    scores round to one fp32 value; with a bias, if only of zeros, such experts are equal); weights are the chosen scores,
    divided by their sum when ``renormalize``,
    times ``scale``. An expert whose logit is -inf is never chosen; slots left without one hold id -1
    (which the expert operators skip) and weight 0. (A sigmoid below -88 is 0 in fp32: a token whose chosen scores are
    all 0 has weights 0, renormalised or not.) The weights are differentiable once in
    the logits.
    """
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _RouteTopk.apply(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale,
                               return_counts)
    else:
        out = _forward(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale, return_counts)
    return out if return_counts else out[:2]


def route_topk_backward(
    dweights: torch.Tensor,
    logits: torch.Tensor,
    topk_ids: torch.Tensor,
    scoring: str = "softmax",
    renormalize: bool = True,
    scale: float = 1.0,
) -> torch.Tensor:
    """Gradient of :func:`route_topk`'s weights for the logits ([T, E], the logits' dtype), given the
    ids that it chose (each expert at most once per token)."""
    no_tangents("route_topk_backward", dweights, logits)
    l2 = rows(logits, "logits")
    require(logits.dim() == 2 and l2.dtype in FLOATS, "logits must be fp32, fp16 or bf16 [T, E]")
    require(scoring in _SCORING, "scoring must be 'softmax' or 'sigmoid'")
    T, E = l2.shape
    dev = l2.device
    require(topk_ids.device == dev and topk_ids.dtype == torch.int32 and topk_ids.is_contiguous() and topk_ids.dim() == 2
            and topk_ids.shape[0] == T, "topk_ids must be a contiguous int32 tensor [T, k] on the logits' device")
    require(dweights.shape == topk_ids.shape and dweights.dtype == torch.float32 and dweights.device == dev,
            "dweights must be an fp32 tensor of topk_ids' shape")
    dweights = dweights.contiguous()
    out = empty2(T, E, l2.dtype, dev)
    launch(dev, "moe_route_topk_backward", dweights.data_ptr(), l2.data_ptr(), pitch(l2), FLOATS[l2.dtype],
           topk_ids.data_ptr(), T, E, topk_ids.shape[1], _SCORING[scoring], renormalize, scale, out.data_ptr())
    return out

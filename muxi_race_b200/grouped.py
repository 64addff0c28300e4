"""Matrix products grouped by expert, rows of any number for each, with their gradients; and the expert MLP
made of them, which can be trained.

Rows ``offsets[e] <= r < offsets[e + 1]`` belong to expert e. ``grouped_linear`` multiplies them with that
expert's weights, ``grouped_linear_backward`` gives the gradients of the rows and of the weights.
``moe_mlp`` is :func:`muxi_race_b200.fused_moe` with gradients for the tokens, the experts' weights and the
routing weights.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._args import FLOATS, HALVES, IDS, empty2, graph_link, launch, matrix, no_tangents, once_differentiable, overlap, pitch, require, rows
from .fused import _workspace
from .rows8 import Q_DTYPES, Rows8, restore_rows8, save_rows8, silu_backward, silu_forward
from .w4 import _workspace_bytes as workspace_bytes


_DW_ROWS = 1 << 15  # of which a 16-bit weights' gradient needs no workspace


def _operand(t: torch.Tensor, name: str, dtype: torch.dtype, index: int, width: int, R: Optional[int] = None) -> tuple:
    """(rows, row pitch, address) of an operand [R, width] that is read in 16-byte pieces."""
    if t.dim() != 2 or t.shape[1] != width or (R is not None and t.shape[0] != R) or t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} [{'R' if R is None else R}, {width}]")
    R, _, ld, ptr = matrix(t, name, index)
    if ptr % 16 or (ld % 8 and R > 1):
        raise ValueError(f"{name} must start on 16 bytes, with a row pitch that is a multiple of 8")
    return R, ld, ptr


def _check(w: torch.Tensor, offsets: torch.Tensor):
    """(E, N, K, address of w, its device)"""
    if w.dim() != 3 or w.dtype not in HALVES:
        raise ValueError("w must be fp16 or bf16 [E, N, K]")
    ptr, dev = w.data_ptr(), w.device
    if not w.is_cuda or not w.is_contiguous() or ptr % 16:
        raise ValueError("w must be a contiguous CUDA tensor that starts on 16 bytes")
    E, N, K = w.shape
    if E < 1 or N < 8 or K < 8 or N % 8 or K % 8:
        raise ValueError("w needs at least one expert, and N and K positive multiples of 8")
    if (offsets.dim() != 1 or offsets.shape[0] != E + 1 or offsets.dtype not in IDS or offsets.get_device() != dev.index
            or not offsets.is_contiguous()):
        raise ValueError(f"offsets must be a contiguous int32 or int64 tensor [{E + 1}] on {dev}")
    return E, N, K, ptr, dev


def _rows_product(name: str, x: torch.Tensor, x_name: str, w: torch.Tensor, offsets: torch.Tensor, transposed: bool,
                  out: Optional[torch.Tensor] = None, zero_rest: bool = True) -> torch.Tensor:
    E, N, K, w_ptr, dev = _check(w, offsets)
    red, width = (N, K) if transposed else (K, N)
    dtype = w.dtype
    R, ld, ptr = _operand(x, x_name, dtype, dev.index, red)
    if out is None:
        out, ld_out = empty2(R, width, dtype, dev), width
    else:
        require(tuple(out.shape) == (R, width) and out.dtype == dtype, f"out must be {dtype} [{R}, {width}]")
        rows(out, "out", dev)
        ld_out = pitch(out)
        require(R < 2 or ld_out >= width, "rows of out must not overlap")
        for t in (x, w.view(1, -1), offsets.view(1, -1)):
            require(not overlap(out, t), "out must not share memory with the inputs")
    launch(dev, name, ptr, ld, w_ptr, offsets.data_ptr(), IDS[offsets.dtype], out.data_ptr(), ld_out, R, E, N, K, HALVES[dtype],
           zero_rest)
    return out


def _grouped_dw(dy, x, w_shape, offsets, dw_dtype) -> torch.Tensor:
    E, N, K = w_shape
    dev, dtype = dy.device, dy.dtype
    R, ld_dy, dy_ptr = _operand(dy, "dy", dtype, dev.index, N)
    _, ld_x, x_ptr = _operand(x, "x", dtype, dev.index, K, R)
    dw = torch.empty((E, N, K), dtype=dw_dtype, device=dev)
    args = (dy_ptr, ld_dy, x_ptr, ld_x, offsets.data_ptr(), IDS[offsets.dtype], dw.data_ptr(), FLOATS[dw_dtype], R, E, N, K,
            HALVES[dtype])
    if R > _DW_ROWS and dw_dtype != torch.float32:
        nbytes = workspace_bytes("moe_grouped_linear_dw_workspace_bytes", R, FLOATS[dw_dtype])
        ws = _workspace(nbytes, dev)  # held until the call has been launched
        launch(dev, "moe_grouped_linear_dw_long", *args, ws.data_ptr(), nbytes)
    else:
        launch(dev, "moe_grouped_linear_dw", *args)
    return dw


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """`t` as an operand can be read (gradients come with any strides)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, save, link):
        y = _rows_product("moe_grouped_linear", x, "x", w, offsets, False)
        if save is None or not ctx.needs_input_grad[1]:
            ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, None, w, offsets, None)
        else:
            with torch.no_grad():
                saved = save_rows8(x, save)
            ctx.save_for_backward(saved.q, saved.scale, w, offsets, link)
        return y

    @staticmethod
    def backward(ctx, dy):
        a, scale, w, offsets, link = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        with torch.no_grad():
            x = a if scale is None else Rows8(a, scale, w.dtype)
            grads = grouped_linear_backward(_aligned(dy), x, w, offsets, need_dx=need_dx, need_dw=need_dw)
        done = iter(once_differentiable("grouped_linear", tuple(g for g in grads if g is not None), dy, a, w, link))
        return tuple(None if g is None else next(done) for g in grads) + (None, None, None)


def grouped_linear(
    x: torch.Tensor,
    w: torch.Tensor,
    offsets: torch.Tensor,
    out: Optional[torch.Tensor] = None,
    save: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``y[r] = w[e] @ x[r]`` for the rows ``offsets[e] <= r < offsets[e + 1]`` of each expert e.

    x [R, K] fp16 / bf16 with rows of any pitch that is a multiple of 8, w [E, N, K] (N and K multiples of 8,
    E <= 1024, R, N at most 2^31 - 512, K at most 2^27), offsets [E + 1] int32 / int64, not falling (``moe_align(ids, E, 1).group_offsets``). Rows of no
    expert, before offsets[0] or from offsets[E] on, are 0 in a new result and left as they are in ``out``; what they
    hold in x is not used. Sums in fp32, which the tensor core cuts towards zero, by up to 2^-23 for each 16 terms (K = 14336: at
    most 7e-5 of a sum), then rounded once; the same bits on every run, and for a row whatever the others are
    and however many.

    Differentiable once in x and w (``out`` is not). ``save=torch.int8`` or ``torch.float8_e4m3fn``: x is kept for the
    gradient of w as an 8-bit copy (:func:`save_rows8`).
    """
    require(save is None or save in Q_DTYPES, "save must be None, torch.int8 or torch.float8_e4m3fn")
    no_tangents("grouped_linear", x, w)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        require(out is None, "out is not differentiable")
        return _GroupedLinear.apply(x, w, offsets, save, None if save is None else graph_link(x))
    return _rows_product("moe_grouped_linear", x, "x", w, offsets, False, out, out is None)


def grouped_linear_backward(
    dy: torch.Tensor,
    x,
    w: torch.Tensor,
    offsets: torch.Tensor,
    dw_dtype: Optional[torch.dtype] = None,
    need_dx: bool = True,
    need_dw: bool = True,
):
    """Gradients of :func:`grouped_linear`: ``dx[r] = w[e].T @ dy[r]`` and ``dw[e] = sum of dy[r] x[r].T`` over e's rows.

    Returns ``(dx, dw)``, None for what is not asked for. x [R, K] or its :class:`Rows8` (not needed without dw); dw in
    w's dtype or ``torch.float32``, 0 for an expert without rows. Rows of no expert take no part, and their dx is 0. Plain
    tensors: the results carry no graph.

    The tensor core cuts its fp32 sums towards zero. dw's rows are therefore taken in parts that are added with rounding, of
    768 rows for ``torch.float32`` and of 32768 for 16 bits (which takes a workspace of 39 MB where there are more).
    """
    no_tangents("grouped_linear_backward", dy, x.scale if isinstance(x, Rows8) else x, w)
    E, N, K, _, dev = _check(w, offsets)
    if dw_dtype is None:
        dw_dtype = w.dtype
    elif dw_dtype != w.dtype and dw_dtype != torch.float32:
        raise ValueError("dw_dtype must be the dtype of w or torch.float32")
    _operand(dy, "dy", w.dtype, dev.index, N)
    dx = _rows_product("moe_grouped_linear_dx", dy, "dy", w, offsets, True) if need_dx else None
    dw = None
    if need_dw:
        if isinstance(x, Rows8):
            require(x.shape == (dy.shape[0], K) and x.dtype == w.dtype and x.device == dev,
                    f"saved x must be {w.dtype} [{dy.shape[0]}, {K}] on {dev}")
            x = restore_rows8(x)
        dw = _grouped_dw(dy, x, (E, N, K), offsets, dw_dtype)
    return dx, dw


# ----------------------------------------------------------------------------- the expert MLP
def _gather(x, order, topk: int, valid: int, R: int) -> torch.Tensor:
    """Rows order[r] // topk of tokens x [T, H] or Rows8, for r below *valid."""
    T, H = x.shape
    if isinstance(x, Rows8):
        src = (x.q.data_ptr(), H, Q_DTYPES[x.q.dtype], x.scale.data_ptr())
    else:
        src = (x.data_ptr(), pitch(x), HALVES[x.dtype], None)
    out = empty2(R, H, x.dtype, x.device)
    launch(x.device, "moe_restore_rows", *src, order.data_ptr(), _lib.MOE_I32, max(topk, 1), valid, out.data_ptr(), R, T, H, 1,
           HALVES[x.dtype])
    return out


def _combine(y: torch.Tensor, slot: torch.Tensor, T: int, topk: int) -> torch.Tensor:
    out = empty2(T, y.shape[1], y.dtype, y.device)
    launch(y.device, "moe_combine_rows", y.data_ptr(), slot.data_ptr(), out.data_ptr(), T, topk, y.shape[0], y.shape[1],
           HALVES[y.dtype])
    return out


def _sort_routes(ids: torch.Tensor, E: int) -> tuple:
    """(offsets [E + 1], the routes in the experts' order, each route's place there or -1): ``moe_align`` without padding."""
    R, dev = ids.numel(), ids.device
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    rest = torch.empty(2 * E + 1 + 4, dtype=torch.int32, device=dev)  # sizes, padded offsets (the same), totals
    order, slot = (torch.empty(max(R, 1), dtype=torch.int32, device=dev) for _ in range(2))
    ws = _workspace(_lib.lib().moe_align_workspace_bytes(R, E), dev)
    at = rest.data_ptr()
    launch(dev, "moe_align", ids.data_ptr(), IDS[ids.dtype], R, E, 1, at, offsets.data_ptr(), at + 4 * E, None, order.data_ptr(),
           slot.data_ptr(), at + 4 * (2 * E + 1), ws.data_ptr(), ws.numel())
    return offsets, order, slot


def _mlp_forward(x, w13, w2, ids, weights, save):
    """(out, offsets, order, slot, gate_up or its Rows8)."""
    T, topk = ids.shape
    R, E = T * topk, w13.shape[0]
    offsets, order, slot = _sort_routes(ids, E)
    valid = offsets.data_ptr() + 4 * E
    xs = _gather(x, order, topk, valid, R)
    gate_up = _rows_product("moe_grouped_linear", xs, "x", w13, offsets, False, None, False)
    del xs
    h, saved = silu_forward(gate_up, weights, save, order, valid)
    y = _rows_product("moe_grouped_linear", h, "h", w2, offsets, False, None, False)
    del h
    return _combine(y, slot, T, topk), offsets, order, slot, (gate_up if saved is None else saved)


class _MoeMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, ids, weights, save, link):
        out, offsets, order, slot, gate_up = _mlp_forward(x, w13, w2, ids, weights, save)
        kept = None, None  # x is read for w13's gradient only
        if ctx.needs_input_grad[1]:
            if save is None:
                kept = x, None
            else:
                with torch.no_grad():
                    x8 = save_rows8(x, save)
                kept = x8.q, x8.scale
        kept += (gate_up, None) if save is None else (gate_up.q, gate_up.scale)
        ctx.save_for_backward(*kept, w13, w2, weights, offsets, order, slot, link)
        ctx.topk = ids.shape[1]
        return out

    @staticmethod
    def backward(ctx, dout):
        x, x_scale, gate_up, scale, w13, w2, weights, offsets, order, slot, link = ctx.saved_tensors
        need_x, need_w13, need_w2, _, need_weights, *_ = ctx.needs_input_grad
        no_tangents("moe_mlp's gradient", dout)
        grads = [None] * 7
        with torch.no_grad():
            kept = x
            if x_scale is not None:
                x = Rows8(x, x_scale, w13.dtype)
            if scale is not None:
                gate_up = Rows8(gate_up, scale, w13.dtype, 2)
            T, topk, E = dout.shape[0], ctx.topk, w13.shape[0]
            R, valid = T * topk, offsets.data_ptr() + 4 * E
            dy = _gather(_aligned(dout), order, topk, valid, R)
            dh = _rows_product("moe_grouped_linear_dx", dy, "dy", w2, offsets, True, None, False)
            dweights = torch.zeros_like(weights) if need_weights else None  # routes to no expert: 0
            dgate_up, h = silu_backward(dh, gate_up, weights, dweights, order, valid)
            if need_w2:
                grads[2] = _grouped_dw(dy, h, w2.shape, offsets, w2.dtype)
            del dy, dh, h
            if need_x:
                dxs = _rows_product("moe_grouped_linear_dx", dgate_up, "dgate_up", w13, offsets, True, None, False)
                grads[0] = _combine(dxs, slot, T, topk)
                del dxs
            if need_w13:
                grads[1] = _grouped_dw(dgate_up, _gather(x, order, topk, valid, R), w13.shape, offsets, w13.dtype)
            grads[4] = dweights
        done = iter(once_differentiable("moe_mlp", tuple(g for g in grads if g is not None), dout, kept, w13, w2, weights, link))
        return tuple(None if g is None else next(done) for g in grads)


def _moe_mlp_graph(x, w13, w2, ids, weights, save):
    link = None if save is None and w13.requires_grad else graph_link(x)  # None: x itself is kept
    return _MoeMlp.apply(x, w13, w2, ids, weights, save, link)


def moe_mlp(
    hidden_states: torch.Tensor,
    w_gate_up: torch.Tensor,
    w_down: torch.Tensor,
    topk_ids: torch.Tensor,
    topk_weights: torch.Tensor,
    save: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """:func:`muxi_race_b200.fused_moe` for training: differentiable once in hidden_states, w_gate_up, w_down and topk_weights.

    ``out[t] = sum_j topk_weights[t, j] * w_down[e] (silu(gate_e x_t) * up_e x_t)``, e = topk_ids[t, j]; ids outside
    [0, E) are skipped (their weights' gradient is 0). hidden_states [T, H] fp16 / bf16, w_gate_up [E, 2 I, H] (gate rows
    first), w_down [E, H, I], H and I multiples of 8, E <= 1024; topk_ids [T, k] int32 / int64, topk_weights [T, k] fp32 / fp16 /
    bf16. The same bits on every run, forward and backward.

    For the backward pass the call keeps gate_up [T k, 2 I] and, for w_gate_up's gradient, hidden_states; with ``save=torch.int8`` or
    ``torch.float8_e4m3fn`` as 8-bit copies (half the memory), from which the gradients of the weights and of the activation
    are then taken. The rows between the products are rounded to the dtype (in fp16 values beyond 65504 become
    infinite); the routing weight is applied in front of the down product.
    """
    require(save is None or save in Q_DTYPES, "save must be None, torch.int8 or torch.float8_e4m3fn")
    no_tangents("moe_mlp", hidden_states, w_gate_up, w_down, topk_weights)
    if w_gate_up.dim() != 3 or w_down.dim() != 3 or hidden_states.dim() != 2:
        raise ValueError("hidden_states must be [T, H], w_gate_up [E, 2I, H] and w_down [E, H, I]")
    E, two_i, H = w_gate_up.shape
    I, dt, dev = two_i // 2, hidden_states.dtype, hidden_states.device
    T = hidden_states.shape[0]
    if two_i != 2 * I or tuple(w_down.shape) != (E, H, I) or hidden_states.shape[1] != H:
        raise ValueError("hidden_states must be [T, H], w_gate_up [E, 2I, H] and w_down [E, H, I]")
    if dt not in HALVES or w_gate_up.dtype != dt or w_down.dtype != dt:
        raise ValueError("hidden_states, w_gate_up and w_down must all be fp16 or all bf16")
    if E < 1 or E > 1024 or H < 8 or I < 8 or H % 8 or I % 8:
        raise ValueError("need 1 to 1024 experts, and H and I positive multiples of 8")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_ids and topk_weights must both be [T, topk]")
    if topk_ids.dtype not in IDS or topk_weights.dtype not in FLOATS:
        raise ValueError("topk_ids must be int32 or int64, topk_weights fp32, fp16 or bf16")
    for name, t in (("hidden_states", hidden_states), ("w_gate_up", w_gate_up), ("w_down", w_down), ("topk_ids", topk_ids),
                    ("topk_weights", topk_weights)):
        if not t.is_cuda or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous CUDA tensor on {dev}")
    if w_gate_up.data_ptr() % 16 or w_down.data_ptr() % 16:
        raise ValueError("w_gate_up and w_down must start on 16 bytes")
    tensors = (hidden_states, w_gate_up, w_down, topk_weights)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return _moe_mlp_graph(hidden_states, w_gate_up, w_down, topk_ids, topk_weights, save)
    return _mlp_forward(hidden_states, w_gate_up, w_down, topk_ids, topk_weights, None)[0]

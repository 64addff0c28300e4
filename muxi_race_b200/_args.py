"""Argument helpers of the operators that are called many times per step (small calls, where the
host time of a call counts)."""
from __future__ import annotations

import torch

from . import _lib

FLOATS = {torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16, torch.float32: _lib.MOE_F32}
HALVES = {torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16}
IDS = {torch.int32: _lib.MOE_I32, torch.int64: _lib.MOE_I64}

#: handle of the current stream of a device ordinal, without building a Stream object; None in a torch
#: without CUDA, where the package can be imported and its argument checks work, but no call gets as far
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_functions: dict = {}


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def rows(t: torch.Tensor, name: str, device: torch.device | None = None) -> torch.Tensor:
    """`t` [..., H] as a 2-D view whose rows are contiguous; raises if there is none."""
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be a CUDA tensor" + (f" on {device}" if device is not None else ""))
    if t.dim() != 2:
        require(t.dim() >= 1, f"{name} must have at least one dimension")
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name} must have one row pitch: its leading dimensions cannot be viewed as one") from None
    if not t.is_contiguous() and t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    return t


def pitch(t: torch.Tensor) -> int:
    """Row pitch of a 2-D tensor in elements (a single row has whatever pitch suits)."""
    return t.shape[1] if t.is_contiguous() or t.shape[0] == 1 else t.stride(0)


def overlap_at(a: int, step_a: int, row_a: int, rows_a: int, b: int, step_b: int, row_b: int, rows_b: int) -> bool:
    """Whether two blocks of rows share memory: their addresses, and in bytes from row to row and the rows
    themselves. Column ranges of one wider tensor are told apart; rows of different pitches that interleave
    count as shared."""
    if a + (rows_a - 1) * step_a + row_a <= b or b + (rows_b - 1) * step_b + row_b <= a or rows_a == 0 or rows_b == 0:
        return False
    if step_a != step_b or step_a == 0 or rows_a == 1 or rows_b == 1:
        return True
    at = (b - a) % step_a  # where a row of b starts from the last start of a row of a
    return at < row_a or at + row_b > step_a


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """:func:`overlap_at` of two 2-D tensors with contiguous rows."""
    size_a, size_b = a.element_size(), b.element_size()
    return overlap_at(a.data_ptr(), pitch(a) * size_a, a.shape[1] * size_a, a.shape[0],
                      b.data_ptr(), pitch(b) * size_b, b.shape[1] * size_b, b.shape[0])


def empty2(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """An uninitialised contiguous [rows, cols] tensor (the cheapest way to one)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


class _NoGraph(torch.autograd.Function):
    @staticmethod
    def forward(ctx, message, results, *sources):
        ctx.message = message
        return results

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(ctx.message)


def once_differentiable(name: str, grads: tuple, *sources):
    """The gradients that a kernel made of `sources`, as a backward function returns them. Where a graph of
    them is being built (``create_graph=True``), differentiating them for whatever the sources come from
    raises instead of passing them for constants. (``torch.autograd.function.once_differentiable`` sees the
    incoming gradient only, and is passed over by ``torch.autograd.grad``, whose inputs it does not lead to.)"""
    if not torch.is_grad_enabled():
        return grads
    return _NoGraph.apply(f"{name} can be differentiated once: its gradient comes from a kernel without a graph", grads,
                          *sources)


def without_gradient(name: str, results: tuple, *sources):
    """The results of an operator that has no gradient. Where `sources` ask for one, going back through the
    results raises instead of leaving its part out."""
    if not torch.is_grad_enabled() or not any(s is not None and s.requires_grad for s in sources):
        return results
    return _NoGraph.apply(f"{name} is not differentiable", results, *sources)


def launch(device: torch.device, name: str, *args) -> None:
    """Call entry point `name` with the current stream of `device` appended, that device current."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.lib(), name)
    index = device.index
    if _current_device() == index:
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        _lib.check(name, code)

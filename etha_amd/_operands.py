"""Checks and addressing shared by the operators on local shards (:mod:`etha_amd.embedding`, :mod:`etha_amd.int8`,
:mod:`etha_amd.experts`): device tensors in, one call of the C ABI out."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _native

DTYPE_CODES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
TOKEN_CODES = {torch.int32: _native.I32, torch.int64: _native.I64}


def check_device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """Index of the one GPU that all operands live on."""
    index = first.get_device()
    if index < 0:
        raise RuntimeError(f"{what}: tensors live on {first.device}; this operator only runs on a GPU (there is no CPU path)")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: operands live on {first.device} and {t.device}")
    return index


def code_of(what: str, dtype: torch.dtype) -> int:
    code = DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError(f"{what}: element type {dtype}; float32, bfloat16 and float16 are supported")
    return code


def row_stride(t: torch.Tensor) -> int | None:
    """Distance, in elements, between consecutive rows (all leading dims flattened) of a tensor whose last dim is
    contiguous; None if the rows do not lie at one distance."""
    dim = t.dim()
    if dim == 2:  # the usual case first
        return t.stride(0) if t.stride(1) == 1 or t.shape[1] <= 1 else None
    if dim == 0 or (t.stride(-1) != 1 and t.shape[-1] > 1):
        return None
    stride, expect = None, None
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = step
        elif step != expect:
            return None
        expect = step * size
    return t.shape[-1] if stride is None else stride


MOST_STRIDE = 1 << 23  # bytes between the rows of a product's operand


def readable_rows(t: torch.Tensor, most: int | None = None) -> tuple[torch.Tensor, int]:
    """``t`` or, where its rows do not lie at one distance (of at most ``most`` bytes), a contiguous copy; and that
    distance in elements."""
    stride = row_stride(t)
    if stride is None or (most is not None and stride * t.element_size() > most):
        return t.contiguous(), t.shape[-1]  # a single row counts as contiguous, whatever its stride says
    return t, stride


def _byte_range(t: torch.Tensor) -> tuple[int, int]:
    """First byte and the byte behind the last that the elements of ``t`` lie in."""
    if t.is_contiguous():
        at = t.data_ptr()
        return at, at + t.numel() * t.element_size()
    lo = hi = 0
    for size, step in zip(t.shape, t.stride()):
        lo += min(0, (size - 1) * step)
        hi += max(0, (size - 1) * step)
    es = t.element_size()
    return t.data_ptr() + lo * es, t.data_ptr() + (hi + 1) * es


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``a`` and ``b`` are columns of their own of rows that lie at one distance, as those of one wide buffer: modulo
    that distance, no byte of one then lies where one of the other does."""
    if not a.dim() or not b.dim():
        return False
    step_a, step_b = row_stride(a), row_stride(b)
    if not step_a or not step_b or step_a * a.element_size() != step_b * b.element_size():
        return False
    apart = step_a * a.element_size()
    behind = (b.data_ptr() - a.data_ptr()) % apart
    return a.shape[-1] * a.element_size() <= behind and behind + b.shape[-1] * b.element_size() <= apart


def check_out(what: str, out: torch.Tensor, shape, dtypes, *inputs: torch.Tensor | None) -> int:
    """Checks an output that the caller passes; returns its row stride."""
    if out.shape != shape:
        raise ValueError(f"{what}: out has shape {tuple(out.shape)}, not {tuple(shape)}")
    if out.dtype not in dtypes:
        raise ValueError(f"{what}: out is {out.dtype}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: out requires a gradient")
    refuse_tangent(what, out)
    if out.dim() and out.is_contiguous():
        stride = shape[-1]
    else:
        stride = row_stride(out)
        rows = out.numel() // out.shape[-1] if out.dim() and out.shape[-1] else 0
        if stride is None or (rows > 1 and stride < out.shape[-1]):
            raise ValueError(f"{what}: the rows of out have to be contiguous, apart and at one distance")
    if out.numel():
        lo, hi = _byte_range(out)
        for t in inputs:
            if t is not None and t.numel():
                a, b = _byte_range(t)
                if a < hi and lo < b and not _interleaved(t, out):
                    raise ValueError(f"{what}: out overlaps an input")
    return stride


def written(out: torch.Tensor) -> None:
    """Tells autograd that a tensor of the caller's was written: kernels write by address, which it cannot see, and a graph that
    saved it earlier would go on with the new values."""
    increment_version(out)


def refuse_tangent(what: str, *tensors: torch.Tensor | None) -> None:
    """No operator has a forward-mode derivative, and a result without a tangent would stand for one of zero."""
    if forward_ad._current_level < 0:  # outside of forward-mode differentiation no tensor has a tangent
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative: pass the primal of its operands")


def refuse_grad(what: str, *inputs: torch.Tensor | None) -> None:
    """For operators without a gradient: a silent cut of the graph would train on nothing."""
    if forward_ad._current_level >= 0:
        refuse_tangent(what, *inputs)
    for t in inputs:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or detach its inputs")


def refuse_captured_backward(what: str) -> None:
    """Autograd's accumulation into a leaf runs on the stream of the leaf's first graph; under capture on another stream
    that ends the process, so a backward pass is captured by calling the gradient functions themselves."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"the backward pass of {what} cannot be captured into a graph: capture a call of its gradient function")


_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_entry_points: dict = {}


def call(index: int, name: str, *args) -> None:
    """Entry point ``name`` with ``args`` and the current stream of GPU ``index``, which is the current device for the call.

    Where a kernel takes a few microseconds the host is what a call costs: stream and device are asked for without the
    objects that ``torch.cuda`` wraps them in.
    """
    func = _entry_points.get(name)
    if func is None:
        func = _entry_points[name] = getattr(_native.lib(), name)
    if index == _current_device():
        rc = func(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = func(*args, _current_stream(index))
    if rc != 0:
        _native._check(name, rc)

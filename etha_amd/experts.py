"""Products grouped by expert, over expert shards as a redistribute delivers them.

``weight`` is ``[experts, out, in]``; rows ``offsets[e] .. offsets[e + 1]`` of ``x`` (sorted by expert) belong to expert ``e``.
``offsets`` stays on the device: sizes of a batch are never waited for.  A rank that holds a range of the experts
(``Shard(0)``) passes that range of the offsets; column- and row-parallel shards (``Shard(1)``, ``Shard(2)``) pass their own
part of ``out`` or ``in``, the latter's results being the members of a ``Partial("sum")`` (rounded to the type of ``x``; fp32
members come by an ``out`` of that type).
"""

from __future__ import annotations

import torch

from . import _native
from ._operands import (DTYPE_CODES, MOST_STRIDE, call, check_device, check_out, code_of, readable_rows, refuse_captured_backward,
                        refuse_grad, refuse_tangent, written)

_OPERANDS = {torch.bfloat16: _native.BF16, torch.float16: _native.F16}


def _check(what: str, weight: torch.Tensor | None, offsets: torch.Tensor, *rows: torch.Tensor) -> None:
    refuse_tangent(what, weight, *rows)
    if offsets.dim() != 1 or offsets.dtype != torch.int32 or offsets.numel() < 1:
        raise ValueError(f"{what}: offsets are {offsets.dtype} {tuple(offsets.shape)}, not int32 [experts + 1]")
    dtype = rows[0].dtype
    same = dtype in _OPERANDS
    if weight is not None:
        if weight.dim() != 3:
            raise ValueError(f"{what}: weight has {weight.dim()} dims, not [experts, out, in]")
        if weight.shape[0] != offsets.numel() - 1:
            raise ValueError(f"{what}: {weight.shape[0]} experts and {offsets.numel()} offsets")
        same = same and weight.dtype == dtype
    for t in rows:
        if t.dim() != 2:
            raise ValueError(f"{what}: rows have {t.dim()} dims, not 2")
        same = same and t.dtype == dtype
    if not same:
        dtypes = {str(t.dtype) for t in (*rows, *(() if weight is None else (weight,)))}
        raise ValueError(f"{what}: operands are {', '.join(sorted(dtypes))}; all bfloat16 or all float16 are supported")


def _matrices(what: str, weight: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """Row and matrix stride of a weight whose rows are contiguous."""
    if weight.stride(2) != 1 and weight.shape[2] > 1:
        raise ValueError(f"{what}: the rows of weight have to be contiguous")
    if weight.stride(1) * 2 > MOST_STRIDE:
        return weight.contiguous(), weight.shape[2], weight.shape[1] * weight.shape[2]
    return weight, weight.stride(1), weight.stride(0)


def _product(what, x, weight, offsets, transposed, out):
    """Rows of ``x`` times their expert's matrix (``transposed``: ``[in, out]`` instead of ``[out, in]``)."""
    experts, n, k = weight.shape
    cols, red = (k, n) if transposed else (n, k)
    if x.shape[1] != red:
        raise ValueError(f"{what}: rows of {x.shape[1]} elements and a weight of {tuple(weight.shape)}")
    source, stride = readable_rows(x, MOST_STRIDE)
    weight, w_stride, w_group = _matrices(what, weight)
    offsets = offsets if offsets.is_contiguous() else offsets.contiguous()
    rows = x.shape[0]
    given, fresh = out, out is None
    if not fresh:
        out_stride = check_out(what, out, (rows, cols), DTYPE_CODES, x, weight, offsets)
    device = check_device(what, x, weight, offsets, out)
    if fresh:
        out, out_stride = x.new_empty((rows, cols)), cols
    call(device, "etha_grouped_matmul", source.data_ptr(), _OPERANDS[x.dtype], rows, stride,
         weight.data_ptr(), experts, cols, red, w_stride, w_group, int(transposed), offsets.data_ptr(), out.data_ptr(),
         DTYPE_CODES[out.dtype], out_stride, int(fresh))
    if given is not None:
        written(given)
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return _product("grouped_linear", x, weight, offsets, False, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        refuse_captured_backward("grouped_linear")
        x, weight, offsets = ctx.saved_tensors
        rows = grouped_linear_grad_rows(grad, weight, offsets) if ctx.needs_input_grad[0] else None
        matrices = grouped_linear_grad_weight(grad, x, offsets) if ctx.needs_input_grad[1] else None
        return rows, matrices, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = weight[e] @ x[t]`` for the expert ``e`` of row ``t``: ``[rows, out]`` in the type of ``x`` (bf16 or fp16).

    Rows of no expert (before ``offsets[0]``, from ``offsets[-1]`` on) are zeros, or left as they are in a given ``out``
    (which may be fp32).  Sums are held in fp32.  Differentiable in ``x`` and ``weight`` (in reverse mode; not with
    ``out``).
    """
    _check("grouped_linear", weight, offsets, x)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        if out is not None:
            raise ValueError("grouped_linear: out cannot be given where an input requires a gradient")
        return _GroupedLinear.apply(x, weight, offsets)
    return _product("grouped_linear", x, weight, offsets, False, out)


def grouped_linear_grad_rows(grad: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of :func:`grouped_linear` with respect to ``x``: ``grad[t] @ weight[e]``; rows of no expert as there."""
    refuse_grad("grouped_linear_grad_rows", grad, weight)
    _check("grouped_linear_grad_rows", weight, offsets, grad)
    return _product("grouped_linear_grad_rows", grad, weight, offsets, True, out)


def grouped_linear_grad_weight(grad: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, *, dtype: torch.dtype | None = None,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of :func:`grouped_linear` with respect to ``weight``: ``grad[rows of e].T @ x[rows of e]`` for each expert, zeros
    for an expert without rows; in ``dtype`` (default: that of ``x``)."""
    what = "grouped_linear_grad_weight"
    refuse_grad(what, grad, x)
    _check(what, None, offsets, grad, x)
    if grad.shape[0] != x.shape[0]:
        raise ValueError(f"{what}: {grad.shape[0]} rows of grad and {x.shape[0]} of x")
    experts, n, k = offsets.numel() - 1, grad.shape[1], x.shape[1]
    g, g_stride = readable_rows(grad, MOST_STRIDE)
    r, r_stride = readable_rows(x, MOST_STRIDE)
    offsets = offsets if offsets.is_contiguous() else offsets.contiguous()
    given = out
    if out is None:
        dtype = dtype or x.dtype
        code_of(what, dtype)
    else:
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"{what}: dtype {dtype} and an out of {out.dtype}")
        check_out(what, out, (experts, n, k), DTYPE_CODES, grad, x, offsets)
    device = check_device(what, x, grad, offsets, out)
    if out is None:
        out = x.new_empty((experts, n, k), dtype=dtype)
    nbytes = _native.grouped_matmul_reduce_workspace(x.shape[0], experts, n, k)
    workspace = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    call(device, "etha_grouped_matmul_reduce", g.data_ptr(), r.data_ptr(), _OPERANDS[x.dtype], x.shape[0], g_stride, r_stride, experts,
         n, k, offsets.data_ptr(), out.data_ptr(), DTYPE_CODES[out.dtype], out.stride(1), out.stride(0),
         workspace.data_ptr() if nbytes else None, nbytes)
    if given is not None:
        written(given)
    return out


def grouped_linear_grad(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *,
                        weight_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Both gradients of :func:`grouped_linear`: of ``x``, and of ``weight`` in ``weight_dtype`` (default: the weight's).  Neither
    is part of a graph, so inputs that require a gradient are refused, as by either of the two: call them under
    ``torch.no_grad()`` or detach their inputs."""
    refuse_grad("grouped_linear_grad", grad, x, weight)
    return (grouped_linear_grad_rows(grad, weight, offsets),
            grouped_linear_grad_weight(grad, x, offsets, dtype=weight_dtype or weight.dtype))

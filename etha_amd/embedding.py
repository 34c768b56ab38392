"""Embedding lookup in a shard of a vocabulary, and its gradient.

A redistribute delivers an embedding as row shards (``Shard(0)``, possibly uneven) or column shards (``Shard(1)``).
:func:`embedding` reads either: with ``first_row`` set to the global index of the shard's first row, tokens of other shards
give zero rows, and the results of all shards are the members of a ``Partial("sum")``, which the framework's reduction
collapses.  :func:`embedding_grad` is the gradient of that shard: each row's tokens are summed in fp32, in their order.
"""

from __future__ import annotations

import operator

import torch

from . import _native
from ._operands import (DTYPE_CODES, TOKEN_CODES, call, check_device, check_out, code_of, readable_rows, refuse_captured_backward,
                        refuse_grad, refuse_tangent, row_stride, written)


def _token_operand(what: str, tokens: torch.Tensor) -> tuple[torch.Tensor, int]:
    code = TOKEN_CODES.get(tokens.dtype)
    if code is None:
        raise ValueError(f"{what}: tokens are {tokens.dtype}; int32 and int64 are supported")
    return (tokens if tokens.is_contiguous() else tokens.contiguous()), code


def _first_row(what: str, first_row) -> int:
    if type(first_row) is not int:
        first_row = operator.index(first_row)
    if not -(1 << 63) <= first_row < 1 << 63:
        raise ValueError(f"{what}: first_row {first_row} has more than 64 bits")
    return first_row


def _lookup(tokens, weight, scale, first_row, dtype, out):
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight has {weight.dim()} dims, not [rows, width]")
    rows, width = weight.shape
    stride = row_stride(weight)
    if stride is None:
        raise ValueError("embedding: the rows of weight have to be contiguous")
    weight_code = code_of("embedding", weight.dtype)
    source, token_code = _token_operand("embedding", tokens)
    given = out
    if out is None:
        dtype = dtype or weight.dtype
        out_code = code_of("embedding", dtype)
        device = check_device("embedding", weight, tokens)
        out = weight.new_empty((*tokens.shape, width), dtype=dtype)
        out_stride = width
    else:
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"embedding: dtype {dtype} and an out of {out.dtype}")
        out_stride = check_out("embedding", out, (*tokens.shape, width), DTYPE_CODES, tokens, weight)
        out_code = DTYPE_CODES[out.dtype]
        device = check_device("embedding", weight, tokens, out)
    call(device, "etha_embedding", source.data_ptr(), token_code, tokens.numel(), weight.data_ptr(),
         weight_code, rows, width, stride, first_row, scale, out.data_ptr(), out_code, out_stride)
    if given is not None:
        written(given)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, first_row, dtype):
        ctx.save_for_backward(tokens)
        ctx.rest = (weight.shape[0], scale, first_row, weight.dtype)
        return _lookup(tokens, weight, scale, first_row, dtype, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        refuse_captured_backward("embedding")
        (tokens,) = ctx.saved_tensors
        rows, scale, first_row, dtype = ctx.rest
        return None, embedding_grad(grad, tokens, rows, scale=scale, first_row=first_row, dtype=dtype), None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, first_row: int = 0,
              dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * weight[tokens - first_row]`` in ``dtype`` (default: the weight's), zeros for tokens outside the shard.

    ``tokens``: int32 or int64, any shape; ``weight``: ``[rows, width]`` in fp32, bf16 or fp16 with contiguous rows.  The
    product with ``scale`` is formed in fp32 and rounded once.  Differentiable in ``weight`` (in reverse mode; not with ``out``).
    """
    refuse_tangent("embedding", weight)
    if weight.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("embedding: out cannot be given where weight requires a gradient")
        return _Embedding.apply(tokens, weight, float(scale), _first_row("embedding", first_row), dtype)
    return _lookup(tokens, weight, float(scale), _first_row("embedding", first_row), dtype, out)


def embedding_grad(grad: torch.Tensor, tokens: torch.Tensor, n_rows: int, *, scale: float = 1.0, first_row: int = 0,
                   dtype: torch.dtype | None = None, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of :func:`embedding` with respect to its weight: ``[n_rows, width]`` in ``dtype`` (default: the gradient's).

    ``grad``: the gradient of the result, ``tokens.shape + (width,)``.  Rows without a token become zeros.  With ``out`` and
    ``accumulate=True`` the sums are added to ``out`` (micro-batches into one gradient) and rows without a token are not
    touched.  The same inputs give the same bits.  The result is not part of a graph, so a ``grad`` that requires a
    gradient is refused.
    """
    refuse_grad("embedding_grad", grad)
    if grad.dim() != tokens.dim() + 1 or grad.shape[:-1] != tokens.shape:
        raise ValueError(f"embedding_grad: grad has shape {tuple(grad.shape)} for tokens of {tuple(tokens.shape)}")
    if n_rows < 0:
        raise ValueError(f"embedding_grad: {n_rows} rows")
    if accumulate and out is None:
        raise ValueError("embedding_grad: accumulate needs an out")
    scale, first_row = float(scale), _first_row("embedding_grad", first_row)
    width, n_tokens = grad.shape[-1], tokens.numel()
    grad_code = code_of("embedding_grad", grad.dtype)
    grad, grad_stride = readable_rows(grad)
    source, token_code = _token_operand("embedding_grad", tokens)
    given = out
    if out is None:
        dtype = dtype or grad.dtype
        out_code = code_of("embedding_grad", dtype)
        device = check_device("embedding_grad", grad, tokens)
        out = grad.new_empty((n_rows, width), dtype=dtype)
        out_stride = width
    else:
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"embedding_grad: dtype {dtype} and an out of {out.dtype}")
        out_stride = check_out("embedding_grad", out, (n_rows, width), DTYPE_CODES, grad, tokens)
        out_code = DTYPE_CODES[out.dtype]
        device = check_device("embedding_grad", grad, tokens, out)
    nbytes = _native.embedding_grad_workspace(n_tokens, n_rows, width, grad_code)
    workspace = grad.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    call(device, "etha_embedding_grad", grad.data_ptr(), grad_code, grad_stride, source.data_ptr(),
         token_code, n_tokens, n_rows, width, first_row, scale, out.data_ptr(), out_code, out_stride, int(accumulate),
         workspace.data_ptr() if nbytes else None, nbytes)
    if given is not None:
        written(given)
    return out

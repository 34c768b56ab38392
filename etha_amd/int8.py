"""Weights in 8 bits: rows with a scale each, and the product of 8-bit rows.

An inference job that holds its projections in 8 bits turns every weight shard that a redistribute delivers into integers
with one scale for each output channel (:func:`quantize_rows`), and multiplies tokens, converted the same way with one scale
for each token, with them (:func:`int8_linear`).
"""

from __future__ import annotations

import torch

from . import _native
from ._operands import DTYPE_CODES, call, check_device, check_out, code_of, readable_rows, refuse_grad

INT8_MAX_WIDTH = 131071  # ETHA_INT8_MAX_WIDTH


def quantize_rows(x: torch.Tensor, *, values: torch.Tensor | None = None,
                  scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``x`` (its last dim) in 8 bits: ``(values int8, scales fp32)`` with ``x ~ values * scales[..., None]``.

    ``scales`` is the row's largest magnitude times 1 / 127 in fp32; values are rounded half to even and lie within +-127.  A row of
    zeros has scale 0; a row that holds a NaN or an infinity has that as its scale and zeros as values.  ``values`` and
    ``scales`` may be given to be written.
    """
    if x.dim() == 0:
        raise ValueError("quantize_rows: x has no rows")
    refuse_grad("quantize_rows", x)
    code = code_of("quantize_rows", x.dtype)
    if values is not None:
        values_stride = check_out("quantize_rows", values, x.shape, (torch.int8,), x, scales)
    if scales is not None:
        check_out("quantize_rows", scales, x.shape[:-1], (torch.float32,), x)
        if not scales.is_contiguous():
            raise ValueError("quantize_rows: scales have to be contiguous")
    device = check_device("quantize_rows", x, values, scales)
    width = x.shape[-1]
    rows = x.numel() // width if width else x.shape[:-1].numel()
    source, stride = readable_rows(x)
    if values is None:
        values, values_stride = torch.empty(x.shape, dtype=torch.int8, device=device), width
    if scales is None:
        scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    call(device, _native.lib().etha_quantize_rows, "etha_quantize_rows", source.data_ptr(), code, rows, width, stride,
         values.data_ptr(), values_stride, scales.data_ptr())
    return values, scales


def _check_scales(what: str, name: str, scales: torch.Tensor, shape) -> torch.Tensor:
    if scales.dtype != torch.float32 or tuple(scales.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} is {scales.dtype} {tuple(scales.shape)}, not float32 {tuple(shape)}")
    return scales if scales.is_contiguous() else scales.contiguous()


def int8_matmul(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """``(x * x_scales[..., None]) @ (weight * weight_scales[:, None]).T + bias`` of 8-bit operands, in ``dtype``.

    ``x``: int8 ``[..., width]``; ``weight``: int8 ``[channels, width]``; scales and ``bias`` fp32.  The sum over the integers
    is exact (``width`` up to 131071); scales and bias are applied in fp32 and rounded once.
    """
    if x.dtype != torch.int8 or weight.dtype != torch.int8:
        raise ValueError(f"int8_matmul: operands are {x.dtype} and {weight.dtype}, not int8")
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"int8_matmul: {tuple(x.shape)} times {tuple(weight.shape)} (channels, width)")
    refuse_grad("int8_matmul", x_scales, weight_scales, bias)
    channels, width = weight.shape
    rows = x.numel() // width if width else x.shape[:-1].numel()
    x_scales = _check_scales("int8_matmul", "x_scales", x_scales, x.shape[:-1])
    weight_scales = _check_scales("int8_matmul", "weight_scales", weight_scales, (channels,))
    if bias is not None:
        bias = _check_scales("int8_matmul", "bias", bias, (channels,))
    if width > INT8_MAX_WIDTH:
        raise ValueError(f"int8_matmul: width {width}; a sum over more than {INT8_MAX_WIDTH} products may leave 32 bits")
    source, stride = readable_rows(x)
    weight, weight_stride = readable_rows(weight)
    device = check_device("int8_matmul", x, x_scales, weight, weight_scales, bias, out)
    if out is None:
        out_code = code_of("int8_matmul", dtype)
        out, out_stride = torch.empty((*x.shape[:-1], channels), dtype=dtype, device=device), channels
    else:
        out_stride = check_out("int8_matmul", out, (*x.shape[:-1], channels), DTYPE_CODES, x, x_scales, weight, weight_scales, bias)
        out_code = DTYPE_CODES[out.dtype]
    call(device, _native.lib().etha_int8_matmul, "etha_int8_matmul", source.data_ptr(), x_scales.data_ptr(), rows, stride,
         weight.data_ptr(), weight_scales.data_ptr(), channels, weight_stride, width, None if bias is None else bias.data_ptr(),
         out.data_ptr(), out_code, out_stride)
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """A linear layer over an 8-bit weight: ``x`` (fp32, bf16 or fp16) is converted with a scale for each token
    (:func:`quantize_rows`) and multiplied (:func:`int8_matmul`); the result is in ``dtype`` (default: that of ``x``)."""
    refuse_grad("int8_linear", x)
    if out is None and dtype is None:
        dtype = x.dtype
    values, scales = quantize_rows(x)
    return int8_matmul(values, scales, weight, weight_scales, bias=bias, dtype=dtype, out=out)

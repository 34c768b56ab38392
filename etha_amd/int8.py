"""Weights in 8 bits: rows with a scale each, and the product of 8-bit rows.

An inference job that holds its projections in 8 bits turns every weight shard that a redistribute delivers into integers
with one scale for each output channel (:func:`quantize_rows`), and multiplies tokens, converted the same way with one scale
for each token, with them (:func:`int8_linear`).  :class:`Int8Weight` is such a weight as the target of a transfer:
``ReshardJob`` (``TensorSpec.target_int8``) and ``TensorBusClient.register_tensors`` convert it when its values have arrived.
"""

from __future__ import annotations

import torch

from . import _native
from ._operands import DTYPE_CODES, MOST_STRIDE, call, check_device, check_out, code_of, readable_rows, refuse_grad, written

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
        check_out("quantize_rows", scales.unsqueeze(-1), (*x.shape[:-1], 1), (torch.float32,), x)
        if not scales.is_contiguous():
            raise ValueError("quantize_rows: scales have to be contiguous")
    device = check_device("quantize_rows", x, values, scales)
    width = x.shape[-1]
    rows = x.numel() // width if width else x.shape[:-1].numel()
    source, stride = readable_rows(x)
    given = values, scales
    if values is None:
        values, values_stride = x.new_empty(x.shape, dtype=torch.int8), width
    if scales is None:
        scales = x.new_empty(x.shape[:-1], dtype=torch.float32)
    call(device, "etha_quantize_rows", source.data_ptr(), code, rows, width, stride,
         values.data_ptr(), values_stride, scales.data_ptr())
    for out in given:
        if out is not None:
            written(out)
    return values, scales


def _check_scales(what: str, name: str, scales: torch.Tensor, shape) -> torch.Tensor:
    if scales.dtype != torch.float32 or tuple(scales.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} is {scales.dtype} {tuple(scales.shape)}, not float32 {tuple(shape)}")
    return scales if scales.is_contiguous() else scales.contiguous()


def _weight_operands(what, x, weight, weight_scales, bias):
    if weight.dtype != torch.int8:
        raise ValueError(f"{what}: the weight is {weight.dtype}, not int8")
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: {tuple(x.shape)} times {tuple(weight.shape)} (channels, width)")
    channels, width = weight.shape
    if width > INT8_MAX_WIDTH:
        raise ValueError(f"{what}: width {width}; a sum over more than {INT8_MAX_WIDTH} products may leave 32 bits")
    weight_scales = _check_scales(what, "weight_scales", weight_scales, (channels,))
    if bias is not None:
        bias = _check_scales(what, "bias", bias, (channels,))
    weight, stride = readable_rows(weight, MOST_STRIDE)
    rows = x.numel() // width if width else x.shape[:-1].numel()
    return weight, stride, weight_scales, bias, channels, width, rows


def int8_matmul(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """``(x * x_scales[..., None]) @ (weight * weight_scales[:, None]).T + bias`` of 8-bit operands, in ``dtype``.

    ``x``: int8 ``[..., width]``; ``weight``: int8 ``[channels, width]``; scales and ``bias`` fp32.  The sum over the integers
    is exact (``width`` up to 131071).  The rest is fp32: the sum is rounded to it, the two scales are multiplied, and their
    product is applied to the sum, with the bias in one fused operation; then comes the result's type.
    """
    what = "int8_matmul"
    if x.dtype != torch.int8:
        raise ValueError(f"{what}: x is {x.dtype}, not int8")
    refuse_grad(what, x_scales, weight_scales, bias)
    weight, w_stride, weight_scales, bias, channels, width, rows = _weight_operands(what, x, weight, weight_scales, bias)
    x_scales = _check_scales(what, "x_scales", x_scales, x.shape[:-1])
    source, stride = readable_rows(x, MOST_STRIDE)
    if out is not None:
        out_stride = check_out(what, out, (*x.shape[:-1], channels), DTYPE_CODES, x, x_scales, weight, weight_scales, bias)
    device = check_device(what, x, x_scales, weight, weight_scales, bias, out)
    given = out
    if out is None:
        code_of(what, dtype)
        out, out_stride = x.new_empty((*x.shape[:-1], channels), dtype=dtype), channels
    call(device, "etha_int8_matmul", source.data_ptr(), x_scales.data_ptr(), rows, stride,
         weight.data_ptr(), weight_scales.data_ptr(), channels, w_stride, width, None if bias is None else bias.data_ptr(),
         out.data_ptr(), DTYPE_CODES[out.dtype], out_stride)
    if given is not None:
        written(given)
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """A linear layer over an 8-bit weight: ``x`` (fp32, bf16 or fp16) is converted with a scale for each token, as
    :func:`quantize_rows` does it, and multiplied, as :func:`int8_matmul` does it, with the same bits; the result is in
    ``dtype`` (default: that of ``x``)."""
    what = "int8_linear"
    refuse_grad(what, x, weight_scales, bias)
    x_code = code_of(what, x.dtype)
    weight, w_stride, weight_scales, bias, channels, width, rows = _weight_operands(what, x, weight, weight_scales, bias)
    source, stride = readable_rows(x)
    if out is not None:
        out_stride = check_out(what, out, (*x.shape[:-1], channels), DTYPE_CODES, x, weight, weight_scales, bias)
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"{what}: dtype {dtype} and an out of {out.dtype}")
    device = check_device(what, x, weight, weight_scales, bias, out)
    given = out
    if out is None:
        dtype = dtype or x.dtype
        code_of(what, dtype)
        out, out_stride = x.new_empty((*x.shape[:-1], channels), dtype=dtype), channels
    nbytes = _native.int8_linear_workspace(rows, channels, width)
    workspace = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    call(device, "etha_int8_linear", source.data_ptr(), x_code, rows, stride, weight.data_ptr(),
         weight_scales.data_ptr(), channels, w_stride, width, None if bias is None else bias.data_ptr(), out.data_ptr(),
         DTYPE_CODES[out.dtype], out_stride, workspace.data_ptr() if nbytes else None, nbytes)
    if given is not None:
        written(given)
    return out


class Int8Weight:
    """A weight in 8 bits that a transfer fills: the transfer writes ``landing`` (``[..., channels, width]`` in fp32, bf16 or
    fp16), :meth:`refresh` converts it into ``values`` (int8) and ``scales`` (fp32, one for each channel), which keep their
    addresses, so that captured graphs read the new weights.

    The landing stays for the next transfer, whose plan holds its address: such a weight needs 3 or 5 bytes an element.  What
    it saves is what a product reads.
    """

    def __init__(self, landing: torch.Tensor):
        if landing.dim() < 2:
            raise ValueError(f"Int8Weight: a weight of {landing.dim()} dims has no channels")
        code_of("Int8Weight", landing.dtype)
        self.landing = landing
        self.values = torch.zeros(landing.shape, dtype=torch.int8, device=landing.device)
        self.scales = torch.zeros(landing.shape[:-1], dtype=torch.float32, device=landing.device)

    def refresh(self) -> "Int8Weight":
        """Convert what lies in ``landing``, on the current stream."""
        with torch.no_grad():
            quantize_rows(self.landing, values=self.values, scales=self.scales)
        return self

    def linear(self, x: torch.Tensor, *, bias: torch.Tensor | None = None, dtype: torch.dtype | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """:func:`int8_linear` over this weight (two dims)."""
        return int8_linear(x, self.values, self.scales, bias=bias, dtype=dtype, out=out)

"""Outputs beside their inputs in one buffer: columns of their own are no overlap, shared bytes are refused."""

import pytest
import torch

from etha_amd._operands import check_out
from etha_amd.embedding import embedding, embedding_grad
from etha_amd.experts import grouped_linear, grouped_linear_grad_rows, grouped_linear_grad_weight
from etha_amd.int8 import int8_linear, int8_matmul, quantize_rows


def bytes_of(t):
    """The bytes that the elements of ``t`` lie in."""
    at = torch.tensor([t.data_ptr()])
    for size, step in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(size)[None] * step * t.element_size()).reshape(-1)
    return {int(a) + k for a in at for k in range(t.element_size())}


def test_what_is_an_overlap():
    """Against the bytes themselves: nothing that shares one is taken, and columns of one buffer are."""
    gen = torch.Generator().manual_seed(3)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (), generator=gen))
    taken = 0
    for _ in range(3000):
        memory = torch.zeros(400, dtype=torch.uint8)
        views = []
        for _ in range(2):
            dtype = (torch.float32, torch.bfloat16, torch.int8)[pick(0, 2)]
            typed = memory.view(dtype)
            rows, width = pick(1, 5), pick(1, 6)
            step = pick(0, 1) * (24 // typed.element_size()) or pick(width, 14)
            if step < width:
                continue
            room = typed.numel() - (rows - 1) * step - width
            shape, strides = ((rows, width), (step, 1)) if rows != 4 or pick(0, 1) else ((2, 2, width), (2 * step, step, 1))
            views.append(typed.as_strided(shape, strides, pick(0, min(room, 40))))
        if len(views) < 2:
            continue
        a, out = views
        shared = bool(bytes_of(a) & bytes_of(out))
        try:
            check_out("it", out, tuple(out.shape), (out.dtype,), a)
            assert not shared
            taken += 1
        except ValueError as e:
            assert "overlaps" in str(e)
    assert taken > 100
    wide = torch.zeros(7, 20)
    assert check_out("it", wide[:, 9:], (7, 11), (torch.float32,), wide[:, :9]) == 20
    assert check_out("it", wide[:, :9], (7, 9), (torch.float32,), wide[:, 9:]) == 20
    for other in (wide[:, 8:], wide[1:, 3:9], wide[:, ::2], wide.t()[:9]):
        with pytest.raises(ValueError, match="overlaps"):
            check_out("it", wide[:, :9], (7, 9), (torch.float32,), other)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_outputs_beside_their_inputs(gpu_device, rows):
    gen = torch.Generator(device=gpu_device).manual_seed(rows)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=gpu_device)

    def beside(values, width, call, dtype=None):
        """``call(x, out)`` with x and out in one buffer gives what it gives with an out of its own, and leaves the rest."""
        dtype = dtype or values.dtype
        for first in (True, False):  # the input before its output, and behind it
            es, eo = values.element_size(), torch.empty(0, dtype=dtype).element_size()
            n, k = values.numel() // values.shape[-1], values.shape[-1]
            left, right = (k * es, width * eo) if first else (width * eo, k * es)
            cut = -(-left // 16) * 16
            wide = torch.full((n, cut + -(-right // 16) * 16 + 16), 77, dtype=torch.uint8, device=gpu_device)
            lo, hi = wide[:, :left], wide[:, cut:cut + right]
            x, out = (lo.view(values.dtype), hi.view(dtype)) if first else (hi.view(values.dtype), lo.view(dtype))
            x.copy_(values.reshape(n, k))
            apart = torch.full((n, width), 3, dtype=dtype, device=gpu_device)
            call(x, apart)
            call(x, out)
            assert torch.equal(out, apart) and torch.equal(x, values.reshape(n, k))
            assert bool((wide[:, left:cut] == 77).all()) and bool((wide[:, cut + right:] == 77).all())

    offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=gpu_device)
    weight = rand(2, 90, 136).bfloat16()
    beside(rand(rows, 136).bfloat16(), 90, lambda x, out: grouped_linear(x, weight, offsets, out=out))
    beside(rand(rows, 90).bfloat16(), 136, lambda g, out: grouped_linear_grad_rows(g, weight, offsets, out=out), torch.float32)
    ids = torch.randint(0, rows, (rows,), generator=gen, device=gpu_device)
    beside(rand(rows, 72).bfloat16(), 72, lambda w, out: embedding(ids, w, out=out), torch.float32)
    beside(rand(rows, 72).bfloat16(), 72, lambda g, out: embedding_grad(g, ids, rows, out=out), torch.float32)
    beside(rand(rows, 500), 500, lambda x, out: quantize_rows(x, values=out), torch.int8)
    w, ws, xs = torch.randint(-127, 128, (33, 260), generator=gen, device=gpu_device, dtype=torch.int8), rand(33).abs(), rand(rows).abs()
    beside(torch.randint(-127, 128, (rows, 260), generator=gen, device=gpu_device, dtype=torch.int8), 33,
           lambda x, out: int8_matmul(x, xs, w, ws, out=out), torch.bfloat16)
    beside(rand(rows, 260).bfloat16(), 33, lambda x, out: int8_linear(x, w, ws, out=out))
    # the gradient of the matrices lies beside rows of as many as it has itself
    n = 24
    x = rand(2 * n, 64).bfloat16()
    grad, cuts = rand(2 * n, n).bfloat16(), torch.tensor([0, 30, 2 * n], dtype=torch.int32, device=gpu_device)
    wide = torch.zeros(2 * n, 128, dtype=torch.bfloat16, device=gpu_device)
    wide[:, :64] = x
    grouped_linear_grad_weight(grad, wide[:, :64], cuts, out=wide.view(2, n, 128)[..., 64:])
    assert torch.equal(wide.view(2, n, 128)[..., 64:], grouped_linear_grad_weight(grad, x, cuts)) and torch.equal(wide[:, :64], x)

"""Rows in 8 bits and the product of 8-bit rows, against plain forms in 64 bits.

Tolerances.  Values in 8 bits are integers and compared as such; a scale is one fp32 product.  The product's
integer sum is exact; fp32 rounds it, the product of the two scales, their product and the sum with the bias: four
roundings of at most 2^-24 of |product| + |bias|, then half a step of the result's type.
"""

import pytest
import torch

from etha_amd import _native as nat
from etha_amd.int8 import int8_linear, int8_matmul, quantize_rows

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain_rows(x):
    x = x.cpu()
    scale = x.abs().amax(-1).float() * (torch.ones(()) / 127)
    fine = scale.isfinite() & (scale > 0)
    quotient = x.double() / torch.where(fine, scale, torch.ones(())).double()[..., None]
    q = torch.where(fine[..., None], quotient.nan_to_num().round().clamp(-127, 127), 0.0)
    return q.to(torch.int8), scale


def check_rows(x, values, scales):
    q, s = plain_rows(x)
    assert values.dtype == torch.int8 and scales.dtype == torch.float32
    assert torch.equal(scales.cpu().nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))
    assert torch.equal(values.cpu(), q)


def check_product(got, x, xs, w, ws, bias):
    total = (x.cpu().double() @ w.cpu().double().t()) * xs.cpu().double()[..., None] * ws.cpu().double()
    want = total if bias is None else total + bias.cpu().double()
    size = total.abs() + (0 if bias is None else bias.cpu().double().abs())
    bound = 4 * 2.0 ** -24 * size
    bound = bound + (want.abs() + bound) * torch.finfo(got.dtype).eps / 2
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} more than the bound"


# ---- refusals (no GPU needed) -------------------------------------------------------------------------------------

def test_refusals():
    x, w, s = torch.zeros(3, 8), torch.zeros(5, 8, dtype=torch.int8), torch.zeros(5)
    q, qs = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        quantize_rows(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        int8_matmul(q, qs, w, s)
    with pytest.raises(ValueError, match="no rows"):
        quantize_rows(torch.zeros(()))
    with pytest.raises(ValueError, match="element type"):
        quantize_rows(x.double())
    with pytest.raises(ValueError, match="values|out is"):
        quantize_rows(x, values=torch.zeros(3, 8))
    with pytest.raises(ValueError, match="shape"):
        quantize_rows(x, values=torch.zeros(3, 7, dtype=torch.int8))
    with pytest.raises(ValueError, match="shape"):
        quantize_rows(x, scales=torch.zeros(4))
    with pytest.raises(ValueError, match="contiguous"):
        quantize_rows(x, scales=torch.zeros(6)[::2])
    with pytest.raises(ValueError, match="overlaps"):
        quantize_rows(x, values=x.view(torch.int8)[:, :8])
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize_rows(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_linear(x.clone().requires_grad_(), w, s)
    with pytest.raises(ValueError, match="not int8"):
        int8_matmul(x, qs, w, s)
    with pytest.raises(ValueError, match="channels, width"):
        int8_matmul(q, qs, w[:, :7], s)
    with pytest.raises(ValueError, match="x_scales"):
        int8_matmul(q, qs[:2], w, s)
    with pytest.raises(ValueError, match="weight_scales"):
        int8_matmul(q, qs, w, s.double())
    with pytest.raises(ValueError, match="bias"):
        int8_matmul(q, qs, w, s, bias=torch.zeros(4))
    with pytest.raises(ValueError, match="width"):
        int8_matmul(torch.zeros(1, 131072, dtype=torch.int8), qs[:1], torch.zeros(5, 131072, dtype=torch.int8), s)


def test_entry_points_refuse_what_they_cannot_take():
    lib = nat.lib()
    rows = lambda **k: lib.etha_quantize_rows(*{**dict(x=0x1000, d=nat.F32, r=4, w=4, xs=4, v=0x1000, vs=4, s=0x1000, st=None), **k}.values())
    assert rows(d=nat.I8) == nat.ERR_UNSUPPORTED
    assert rows(x=None) == nat.ERR_INVALID and rows(v=None) == nat.ERR_INVALID and rows(s=None) == nat.ERR_INVALID
    assert rows(r=1 << 31) == nat.ERR_UNSUPPORTED
    assert rows(r=0) == 0
    mul = lambda **k: lib.etha_int8_matmul(*{**dict(x=0x1000, xs=0x1000, m=4, xp=16, w=0x1000, ws=0x1000, n=4, wp=16, k=16, b=None, o=0x1000,
                                                    od=nat.BF16, op=4, st=None), **k}.values())
    assert mul(k=131072) == nat.ERR_UNSUPPORTED
    assert mul(od=nat.I8) == nat.ERR_UNSUPPORTED
    assert mul(m=1 << 31) == nat.ERR_UNSUPPORTED
    assert mul(x=None) == nat.ERR_INVALID and mul(ws=None) == nat.ERR_INVALID and mul(o=None) == nat.ERR_INVALID
    assert mul(m=0) == 0 and mul(n=0) == 0
    lin = lambda **k: lib.etha_int8_linear(*{**dict(x=0x1000, d=nat.BF16, m=40, xp=16, w=0x1000, ws=0x1000, n=4, wp=16, k=16, b=None, o=0x1000,
                                                    od=nat.BF16, op=4, wk=0x1000, wb=1 << 20, st=None), **k}.values())
    assert lin(k=131072) == nat.ERR_UNSUPPORTED and lin(d=nat.I8) == nat.ERR_UNSUPPORTED and lin(od=nat.F64) == nat.ERR_UNSUPPORTED
    assert lin(x=None) == nat.ERR_INVALID and lin(ws=None) == nat.ERR_INVALID and lin(o=None) == nat.ERR_INVALID
    assert lin(wk=None) == nat.ERR_INVALID and lin(wb=16) == nat.ERR_INVALID and lin(wk=0x1008) == nat.ERR_INVALID
    assert lin(m=0) == 0 and lin(n=0) == 0
    assert nat.int8_linear_workspace(0, 8, 100) == 0 and nat.int8_linear_workspace(40, 8, 100) == 40 * 112 + 160
    with pytest.raises(nat.EthaNativeError):
        nat.int8_linear_workspace(1, 8, 131072)


# ---- rows -------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 7), (3, 64), (70, 511), (9, 1001), (6, 2048), (4, 2056), (130, 4096), (5, 8191),
                                        (4, 8200), (3, 32768), (2, 33001), (37, 700), (33, 1024), (11, 2300), (9, 2560), (7, 2561), (6, 3584),
                                        (5, 3585), (32769, 3600)])
def test_rows(gpu_device, rows, width, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(rows * width)
    x = (torch.randn(rows, width, generator=gen, device=gpu_device) * 3).to(dtype)
    check_rows(x, *quantize_rows(x))


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes(gpu_device):
    x = torch.randn((1 << 21) + 5, 9, dtype=torch.bfloat16, device=gpu_device)[:, :8]  # 18 bytes between rows
    values, scales = quantize_rows(x)
    for part in (slice(0, 4), slice((1 << 21) - 4, None)):
        check_rows(x[part], values[part], scales[part])


@pytest.mark.gpu
def test_one_row_into_a_given_scale(gpu_device):
    x = torch.randn(77, device=gpu_device)
    scale = torch.empty((), device=gpu_device)
    values, got = quantize_rows(x, scales=scale)
    assert got is scale
    check_rows(x[None], values[None], got[None])


@pytest.mark.gpu
def test_rounding_of_halves(gpu_device):
    """Quotients at and next to a half: with a scale that is a power of two halves are exact, with others they are near."""
    for top in (127.0, 254.0, 63.5, 127.0 * 1.0009765625, 100.0, 3e-37, 127 * 2.0 ** -126, 3e-40, 127 * 2.0 ** -149, 2.0 ** -149, 3e38):
        scale = torch.tensor(top, dtype=torch.float32) * (torch.ones(()) / 127)
        n = torch.arange(-127, 127, dtype=torch.float64) + 0.5
        near = (n * scale.double()).float()
        x = torch.cat([near, torch.nextafter(near, torch.tensor(1e30)), torch.nextafter(near, torch.tensor(-1e30)), torch.tensor([top, -top])])
        x = x.clamp(-top, top)[None].to(gpu_device)
        check_rows(x, *quantize_rows(x))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,power", [(torch.float16, 0), *((torch.float32, p) for p in (-127, -126, -125, -100, 0, 100))], ids=str)
def test_rounding_next_to_halves(gpu_device, dtype, power):
    """Quotients within a few units of the last place of every half, and on it where it is a number; the last column is the
    row's largest magnitude and sets its scale."""
    gen = torch.Generator().manual_seed(4)
    top = (torch.rand(64, 1, generator=gen).double() + 1) * 100 * 2.0 ** power
    scale = (top.float() * (torch.ones(()) / 127)).double()
    x = ((torch.arange(-126, 126).double() + 0.5) * scale).to(dtype)
    bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    nudged = [(bits + k).view(dtype) for k in (-2, -1, 0, 1, 2)]
    x = torch.cat([*nudged, top.to(dtype)], 1)
    assert bool((x.abs().amax(1) == x[:, -1].abs()).all())
    for columns in (slice(None), slice(0, None, 5), slice(4, None, 41)):  # alone in their waves, or together
        part = torch.cat([x[:, columns], x[:, -1:]], 1).to(gpu_device)
        check_rows(part, *quantize_rows(part))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [40, 3000, 9000, 40000])
def test_rows_with_zeros_infinities_and_nan(gpu_device, width):
    x = torch.randn(8, width, device=gpu_device)
    x[0], x[1] = 0.0, -0.0
    x[2, width // 2], x[3, 0], x[4, -1], x[5, 1] = float("inf"), float("-inf"), float("nan"), torch.finfo(torch.float32).max
    values, scales = quantize_rows(x)
    check_rows(x, values, scales)
    assert scales[0] == 0 and scales[2].isinf() and scales[3].isinf() and scales[4].isnan()
    assert not bool(values[[0, 1, 2, 3, 4]].any())
    low = torch.full((1, width), torch.finfo(torch.bfloat16).min, device=gpu_device, dtype=torch.bfloat16)
    check_rows(low, *quantize_rows(low))


@pytest.mark.gpu
def test_rows_of_views_into_views(gpu_device):
    base = torch.randn(2, 6, 300, device=gpu_device).half()
    x = base[:, ::2, 1:200]  # two distances between rows: a copy is made
    values, scales = quantize_rows(x)
    assert values.shape == (2, 3, 199) and scales.shape == (2, 3)
    check_rows(x, values, scales)
    wide = torch.full((6, 310), 5, dtype=torch.int8, device=gpu_device)
    s = torch.zeros(6, device=gpu_device)
    got = quantize_rows(base[0, :, 3:], values=wide[:, 7:304], scales=s)
    assert got[0].data_ptr() == wide[:, 7:].data_ptr() and got[1] is s
    check_rows(base[0, :, 3:], wide[:, 7:304], s)
    assert bool((wide[:, :7] == 5).all()) and bool((wide[:, 304:] == 5).all())
    assert quantize_rows(base[0, :0])[0].shape == (0, 300)
    values, scales = quantize_rows(base[0, :, :0])
    assert values.shape == (6, 0) and not bool(scales.any())


# ---- product ----------------------------------------------------------------------------------------------------------

def operands(gen, m, n, k, device, low=-127):
    return (torch.randint(low, 128, (m, k), generator=gen, device=device, dtype=torch.int8), torch.rand(m, generator=gen, device=device) * 0.1,
            torch.randint(low, 128, (n, k), generator=gen, device=device, dtype=torch.int8), torch.rand(n, generator=gen, device=device) * 0.1)


PRODUCTS = [(1, 1, 1), (1, 14336 // 4, 4096), (2, 65, 130), (3, 300, 64), (7, 128, 128), (16, 1000, 500), (17, 129, 127), (33, 72, 1001),
            (64, 640, 4096), (65, 257, 256), (128, 128, 4099), (200, 130, 96), (255, 512, 384), (300, 771, 640), (513, 300, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(gpu_device, m, n, k, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(m + n + k)
    x, xs, w, ws = operands(gen, m, n, k, gpu_device, low=-128)
    bias = torch.randn(n, generator=gen, device=gpu_device) if (m + n) % 2 else None
    got = int8_matmul(x, xs, w, ws, bias=bias, dtype=dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    check_product(got, x, xs, w, ws, bias)
    assert torch.equal(got, int8_matmul(x, xs, w, ws, bias=bias, dtype=dtype))


@pytest.mark.gpu
def test_product_at_the_end_of_32_bits(gpu_device):
    k = 131071
    x = torch.full((2, k), -128, dtype=torch.int8, device=gpu_device)
    one = torch.ones(2, device=gpu_device)
    got = int8_matmul(x, one, x, one, dtype=torch.float32)
    assert bool((got == float(128 * 128 * k)).all())
    x[1] = 127
    got = int8_matmul(x, one, x, one, dtype=torch.float32)
    check_product(got, x, one, x, one, None)


@pytest.mark.gpu
def test_a_single_row_whatever_its_stride(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(10)
    x, xs, w, ws = operands(gen, 1, 1, 200, gpu_device)
    far = lambda t: torch.as_strided(t, t.shape, (1 << 30, 1))
    check_product(int8_matmul(far(x), xs, far(w), ws), x, xs, w, ws, None)


@pytest.mark.gpu
def test_product_of_views(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    for m in (3, 70, 300):
        x, xs, w, ws = operands(gen, 2 * m, 210, 333, gpu_device)
        a, b = x[::2, 5:300], w[10:, 7:302]  # unaligned starts, widths and distances
        out = torch.full((m, 220), 9.0, device=gpu_device)
        got = int8_matmul(a, xs[::2], b, ws[10:], out=out[:, 3:203])
        check_product(got, a, xs[::2], b, ws[10:], None)
        assert bool((out[:, :3] == 9).all()) and bool((out[:, 203:] == 9).all())
        stacked = int8_matmul(x.view(2, m, 333), xs.view(2, m), w, ws, dtype=torch.float32)
        assert stacked.shape == (2, m, 210)
        check_product(stacked.view(2 * m, 210), x, xs, w, ws, None)
    assert int8_matmul(x[:0], xs[:0], w, ws).shape == (0, 210)
    assert int8_matmul(x, xs, w[:0], ws[:0]).shape == (600, 0)
    bias = torch.randn(210, device=gpu_device)
    assert torch.equal(int8_matmul(x[:, :0], xs, w[:, :0], ws, bias=bias, dtype=torch.float32), bias.expand(600, 210))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 515, 4096), (1, 64, 77), (1, 40, 33001), (2, 300, 4100), (4, 9000, 256), (3, 1000, 1001), (8, 512, 2048), (40, 200, 512), (300, 400, 640),
                                   (5, 70, 200), (7, 33, 4096), (9, 8200, 1000), (12, 9000, 1030), (16, 130, 2048), (16, 100, 2049), (16, 17, 5),
                                   (17, 130, 512)])
def test_linear(gpu_device, m, n, k, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(m * n + k)
    _, _, w, ws = operands(gen, 1, n, k, gpu_device)
    x = torch.randn(m, k, generator=gen, device=gpu_device).to(dtype)
    if m > 2:
        x[1] = 0
    bias = torch.randn(n, generator=gen, device=gpu_device) if m % 2 else None
    got = int8_linear(x, w, ws, bias=bias)
    assert got.dtype == dtype
    q, s = plain_rows(x)
    check_product(got, q, s, w, ws, bias)
    values, scales = quantize_rows(x)
    assert torch.equal(got, int8_matmul(values, scales, w, ws, bias=bias, dtype=dtype)), "the two steps give the same bits"
    assert torch.equal(int8_linear(x[None], w, ws, bias=bias)[0], got)


@pytest.mark.gpu
def test_a_poisoned_token_poisons_its_row_alone(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(5)
    for m in (4, 12, 100):
        _, _, w, ws = operands(gen, 1, 70, 200, gpu_device)
        x = torch.randn(m, 200, generator=gen, device=gpu_device)
        x[2, 7] = float("nan")
        x[3, 8] = float("inf")
        got = int8_linear(x, w, ws)
        assert bool(got[2].isnan().all()) and bool(got[3].isnan().all())
        assert bool(got[:2].isfinite().all()) and bool(got[4:].isfinite().all())


@pytest.mark.gpu
def test_capture(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(6)
    _, _, w, ws = operands(gen, 1, 300, 512, gpu_device)
    for m in (1, 9, 200):
        x = torch.randn(m, 512, generator=gen, device=gpu_device).bfloat16()
        graph = torch.cuda.CUDAGraph()
        int8_linear(x, w, ws)
        with torch.cuda.graph(graph):
            y = int8_linear(x, w, ws)
        for _ in range(4):
            x.copy_(torch.randn(m, 512, generator=gen, device=gpu_device))
            graph.replay()
            eager = int8_linear(x, w, ws)
            torch.cuda.synchronize()
            assert torch.equal(y, eager)

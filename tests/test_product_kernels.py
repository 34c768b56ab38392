"""Every kernel that a product may take: which sizes take it, and its values there.

The rule that chooses among the kernels is asked on the host (``etha_product_kernel``), so that a change of the rule cannot
leave a kernel without a test.  Values are compared with products in 64 bits, within the bounds that tests/test_experts.py
and tests/test_int8.py derive.
"""

import pytest
import torch

from etha_amd import _native as nat
from etha_amd.experts import grouped_linear, grouped_linear_grad_rows, grouped_linear_grad_weight
from etha_amd.int8 import int8_matmul

from test_experts import bounds_of
from test_int8 import check_product

CODES = {torch.int8: nat.I8, torch.bfloat16: nat.BF16, torch.float16: nat.F16}

# product, kernel, rows, columns of the result, length of the sum, experts; for the reduction: rows and columns of the
# matrices, rows of the operands.  None of them is a whole number of tiles.
CASES = [
    (nat.PRODUCT_INT8, "few 16", 11, 1000, 400, 0),
    (nat.PRODUCT_INT8, "few 32", 20, 2603, 80, 0),
    (nat.PRODUCT_INT8, "few 64", 43, 2600, 336, 0),
    (nat.PRODUCT_INT8, "tile 32", 515, 517, 336, 0),
    (nat.PRODUCT_INT8, "tile 128", 1030, 1029, 336, 0),
    (nat.PRODUCT_INT8, "tile 256", 2600, 4101, 1040, 0),
    (nat.PRODUCT_ROWS, "few 16", 20, 515, 328, 3),
    (nat.PRODUCT_ROWS, "few 32", 66, 515, 72, 8),
    (nat.PRODUCT_ROWS, "few 64", 130, 1029, 72, 3),
    (nat.PRODUCT_ROWS, "tile 32", 700, 701, 72, 8),
    (nat.PRODUCT_ROWS, "tile 128", 1029, 2053, 328, 8),
    (nat.PRODUCT_ROWS, "tile 256", 1537, 4101, 328, 8),
    (nat.PRODUCT_ROWS_T, "few 16", 20, 515, 328, 3),
    (nat.PRODUCT_ROWS_T, "tile 32", 700, 701, 72, 8),
    (nat.PRODUCT_ROWS_T, "tile 128", 1029, 2053, 328, 8),
    (nat.PRODUCT_ROWS_T, "tile 256", 1537, 4101, 328, 8),
    (nat.PRODUCT_REDUCE, "tile 128", 131, 333, 1100, 3),  # the sum is cut into parts
    (nat.PRODUCT_REDUCE, "tile 128", 700, 701, 600, 8),
    (nat.PRODUCT_REDUCE, "tile 256", 2051, 2053, 600, 3),
]


def memory_of(product, rows, cols, red, experts):
    """Shapes of the two operands in memory."""
    if product == nat.PRODUCT_REDUCE:
        return (red, rows), (red, cols)
    if product == nat.PRODUCT_INT8:
        return (rows, red), (cols, red)
    return (rows, red), ((experts, red, cols) if product == nat.PRODUCT_ROWS_T else (experts, cols, red))


def kernel_of(product, p, q, rows, cols, red, experts):
    return nat.product_kernel(product, CODES[p.dtype], (p.data_ptr(), p.stride(0)), (q.data_ptr(), q.stride(-2), q.stride(0)),
                              rows, cols, red, experts)


def ceil_to(n, to):
    return (n + to - 1) // to * to


@pytest.mark.parametrize("product,kernel,rows,cols,red,experts", CASES)
def test_sizes_take_the_kernel(product, kernel, rows, cols, red, experts):
    p, q = memory_of(product, rows, cols, red, experts)
    dtype = nat.I8 if product == nat.PRODUCT_INT8 else nat.BF16
    whole = 16 if product == nat.PRODUCT_INT8 else 8
    pitch = [ceil_to(t[-1], whole) for t in (p, q)]
    assert nat.product_kernel(product, dtype, (0, pitch[0]), (0, pitch[1], q[-2] * pitch[1]), rows, cols, red, experts) == (kernel, True)
    assert nat.product_kernel(product, dtype, (0, pitch[0] + 1), (0, pitch[1] + 1, q[-2] * (pitch[1] + 1)), rows, cols, red, experts) == (kernel, False)


def test_the_rule_covers_every_kernel():
    rows = {"few 16", "few 32", "few 64", "tile 32", "tile 128", "tile 256"}
    reached = {p: {c[1] for c in CASES if c[0] == p} for p in range(4)}
    assert reached[nat.PRODUCT_INT8] == reached[nat.PRODUCT_ROWS] == rows
    assert reached[nat.PRODUCT_ROWS_T] == rows - {"few 32", "few 64"}
    assert reached[nat.PRODUCT_REDUCE] == {"tile 128", "tile 256"}
    for p in range(4):  # rows shorter than 16 bytes that do not start at 16-byte addresses
        short = (7, 5, 300, 3) if p == nat.PRODUCT_REDUCE else (5, 5, 7, 3)
        assert nat.product_kernel(p, nat.I8 if p == nat.PRODUCT_INT8 else nat.F16, (2, 7), (2, 7, 35), *short) == ("short", False)


def test_a_product_takes_a_kernel_that_fits_a_launch():
    """A launch has fewer than 2^22 workgroups: where the cheapest tile would need more, a larger one is taken."""
    aligned = (0x1000, 16), (0x1000, 16, 256)
    for rows, cols in (((1 << 29) + 5, 1), (1, (1 << 29) + 5), ((1 << 30) - 2048, 1)):
        assert nat.product_kernel(nat.PRODUCT_INT8, nat.I8, *aligned, rows, cols, 16) == ("tile 256", True)
        assert nat.product_kernel(nat.PRODUCT_ROWS, nat.BF16, *aligned, rows, cols, 8, 2) == ("tile 256", True)
    assert nat.product_kernel(nat.PRODUCT_INT8, nat.I8, *aligned, 1 << 28, 1, 16)[0] == "tile 128"
    lib = nat.lib()
    assert lib.etha_int8_matmul(0x1000, 0x1000, 1 << 30, 16, 0x1000, 0x1000, 1, 16, 16, None, 0x1000, nat.BF16, 1, None) == nat.ERR_UNSUPPORTED
    assert b"too large" in lib.etha_last_error()
    # one row whose conversion would be a part of the product, if its columns fitted a launch
    assert nat.int8_linear_workspace(1, (1 << 26) - 16, 16) == 0 and nat.int8_linear_workspace(1, 1 << 26, 16) == 16 + 4


def test_inspection_refuses_what_is_no_product():
    good = dict(product=nat.PRODUCT_ROWS, dtype=nat.BF16, p=(0, 8), q=(0, 8, 64), rows=4, cols=8, red=8, n_groups=2)
    assert nat.product_kernel(**good) == ("few 16", True)
    for change in (dict(product=4), dict(dtype=nat.I8), dict(product=nat.PRODUCT_INT8), dict(n_groups=(1 << 16) + 1), dict(rows=0),
                   dict(rows=1 << 31), dict(red=1 << 31)):
        with pytest.raises(nat.EthaNativeError):
            nat.product_kernel(**{**good, **change})


# ---- values -----------------------------------------------------------------------------------------------------------

def placed(gen, shape, dtype, pitch, start, device):
    """Normal values in rows that lie ``pitch`` elements apart from element ``start`` on; NaN around them (127 for int8)."""
    lead = shape[:-1]
    size = start + pitch * torch.Size(lead).numel() + 64
    memory = torch.full((size,), 127 if dtype == torch.int8 else float("nan"), dtype=dtype, device=device)
    strides = [pitch, 1] if len(shape) == 2 else [shape[1] * pitch, pitch, 1]
    t = memory.as_strided(shape, strides, start)
    if dtype == torch.int8:
        t.copy_(torch.randint(-128, 128, shape, generator=gen, device=device, dtype=torch.int8))
    else:
        t.copy_(torch.randn(shape, generator=gen, device=device))
    return t


def offsets_of(rows, experts, device):
    """Uneven groups, the second one empty, a row before the first and two behind the last."""
    cuts = [1, 1 + rows // (2 * experts)]
    for e in range(1, experts):
        cuts.append(cuts[1] + (rows - 2 - cuts[1]) * (e - 1) // max(1, experts - 2) if experts > 2 else rows - 2)
    return torch.tensor(cuts[: experts + 1], dtype=torch.int32, device=device)


def check(got, want, size, n):
    info = torch.finfo(got.dtype)
    bound = (n + 4) * 2.0 ** -23 * size
    bound = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} more than the bound"


def check_values(gen, device, product, kernel, rows, cols, red, experts, dtype, pitch, start, direct):
    """One product of operands whose rows lie ``pitch(width)`` elements apart from element ``start`` on."""
    ps, qs = memory_of(product, rows, cols, red, experts)
    p, q = (placed(gen, s, dtype, pitch(s[-1]), start, device) for s in (ps, qs))
    assert kernel_of(product, p, q, rows, cols, red, experts) == (kernel, direct)
    if product == nat.PRODUCT_INT8:
        xs, ws = (torch.rand(n, generator=gen, device=device) * 0.1 for n in (rows, cols))
        check_product(int8_matmul(p, xs, q, ws, dtype=torch.float32), p, xs, q, ws, None)
        return
    offsets = offsets_of(red if product == nat.PRODUCT_REDUCE else rows, experts, device)
    ends = bounds_of(offsets, p.shape[0])
    assert len(set(ends)) == experts  # one group is empty
    a, b = p.double(), q.double()
    if product == nat.PRODUCT_REDUCE:
        got = grouped_linear_grad_weight(p, q, offsets, dtype=torch.float32)
        for e in range(experts):
            g, x = a[ends[e]:ends[e + 1]].t(), b[ends[e]:ends[e + 1]]
            check(got[e], torch.mm(g, x), torch.mm(g.abs(), x.abs()), ends[e + 1] - ends[e])
        return
    got = grouped_linear_grad_rows(p, q, offsets) if product == nat.PRODUCT_ROWS_T else grouped_linear(p, q, offsets)
    for e in range(experts):
        x, w = a[ends[e]:ends[e + 1]], b[e] if product == nat.PRODUCT_ROWS_T else b[e].t()
        check(got[ends[e]:ends[e + 1]], torch.mm(x, w), torch.mm(x.abs(), w.abs()), red)
    assert bool((got[: ends[0]] == 0).all()) and bool((got[ends[-1]:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("staging", ["direct", "registers"])
@pytest.mark.parametrize("product,kernel,rows,cols,red,experts", CASES)
def test_values(gpu_device, product, kernel, rows, cols, red, experts, staging):
    gen = torch.Generator(device=gpu_device).manual_seed(rows + cols)
    dtype, whole = (torch.int8, 16) if product == nat.PRODUCT_INT8 else (torch.bfloat16 if rows % 2 else torch.float16, 8)
    if staging == "direct":  # rows at 16-byte addresses; widths that matter to it are whole pieces of 16 bytes
        if product == nat.PRODUCT_REDUCE:
            rows, cols = ceil_to(rows, 8), ceil_to(cols, 8)
        elif product == nat.PRODUCT_ROWS_T:
            cols = ceil_to(cols, 8)
        check_values(gen, gpu_device, product, kernel, rows, cols, red, experts, dtype, lambda n: ceil_to(n, whole), 0, True)
    else:  # odd distances and starts; where the sum is along a row, an odd length
        red = red if product == nat.PRODUCT_REDUCE else red - 3
        check_values(gen, gpu_device, product, kernel, rows, cols, red, experts, dtype, lambda n: ceil_to(n, whole) + 1, 3, False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [((1 << 29) + 5, 1), (1, (1 << 29) + 5)])
def test_a_product_of_very_many_rows_or_columns(gpu_device, rows, cols):
    many = torch.randint(-127, 128, (max(rows, cols), 16), device=gpu_device, dtype=torch.int8)
    scales = torch.rand(max(rows, cols), device=gpu_device)
    x, w, xs, ws = (many, many[-1:], scales, scales[-1:]) if rows > 1 else (many[-1:], many, scales[-1:], scales)
    got = int8_matmul(x, xs, w, ws)
    for at in (0, 1 << 28, max(rows, cols) - 700):
        part = slice(at, at + 700)
        if rows > 1:
            check_product(got[part], x[part], xs[part], w, ws, None)
        else:
            check_product(got[:, part], x, xs, w[part], ws[part], None)


@pytest.mark.gpu
@pytest.mark.parametrize("over", range(1, 8))
@pytest.mark.parametrize("product,kernel,rows,cols,red,experts", [c for c in CASES if c[0] >= nat.PRODUCT_ROWS_T and c[1] != "few 16"])
def test_widths_that_are_no_whole_pieces(gpu_device, product, kernel, rows, cols, red, experts, over):
    """Operands that lie transposed go straight into LDS also where their rows end within a piece of 16 bytes, or within 4:
    the last row's last piece reaches over the operand's end."""
    gen = torch.Generator(device=gpu_device).manual_seed(over)
    rows = rows // 8 * 8 + over if product == nat.PRODUCT_REDUCE else rows
    cols = cols // 8 * 8 + over
    check_values(gen, gpu_device, product, kernel, rows, cols, red, experts, torch.bfloat16, lambda n: ceil_to(n, 8), 0, True)

"""Products grouped by expert, against plain forms in 64 bits.

Tolerance.  Products of two 16-bit values are exact in fp32 (22 bits at most).  A sum over K of them in fp32, in whatever
grouping and with at most one unit (2^-23) lost at each addition, is off by at most (K + 4) 2^-23 of the sum of their
magnitudes (the 4: joins of partial sums); the result's type adds half a step, of a subnormal value where it is that small.
"""

import pytest
import torch

from etha_amd import _native as nat
from etha_amd.experts import grouped_linear, grouped_linear_grad, grouped_linear_grad_rows, grouped_linear_grad_weight

HALVES = [torch.bfloat16, torch.float16]


def bounds_of(offsets, rows):
    """Offsets as the operators take them: each the largest of itself and those before it, within [0, rows]."""
    out, top = [], 0
    for v in offsets.tolist():
        top = max(top, min(max(v, 0), rows))
        out.append(top)
    return out


def check(got, want, size, n):
    info = torch.finfo(got.dtype)
    bound = (n + 4) * 2.0 ** -23 * size
    bound = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} more than the bound"


def check_rows(got, x, weight, offsets, transposed=False):
    x, weight = x.cpu().double(), weight.cpu().double()
    ends = bounds_of(offsets, x.shape[0])
    cols = weight.shape[2] if transposed else weight.shape[1]
    want, size = torch.zeros(x.shape[0], cols, dtype=torch.float64), torch.zeros(x.shape[0], cols, dtype=torch.float64)
    for e in range(weight.shape[0]):
        rows, w = slice(ends[e], ends[e + 1]), weight[e] if transposed else weight[e].t()
        want[rows] = x[rows] @ w
        size[rows] = x[rows].abs() @ w.abs()
    check(got, want, size, x.shape[1])
    assert bool((got[: ends[0]] == 0).all()) and bool((got[ends[-1]:] == 0).all())


def check_weight(got, grad, x, offsets):
    grad, x = grad.cpu().double(), x.cpu().double()
    ends = bounds_of(offsets, x.shape[0])
    for e in range(got.shape[0]):
        rows = slice(ends[e], ends[e + 1])
        check(got[e], grad[rows].t() @ x[rows], grad[rows].abs().t() @ x[rows].abs(), ends[e + 1] - ends[e])


def case(gen, sizes, n, k, dtype, device, before=0, behind=0):
    ends = [before]
    for s in sizes:
        ends.append(ends[-1] + s)
    rows = ends[-1] + behind
    rand = lambda *s: torch.randn(*s, generator=gen, device=device).to(dtype)
    return rand(rows, k), rand(len(sizes), n, k), torch.tensor(ends, dtype=torch.int32, device=device), rand(rows, n)


# ---- refusals (no GPU needed) -------------------------------------------------------------------------------------

def test_refusals():
    x, w, off, g = torch.zeros(6, 8).bfloat16(), torch.zeros(2, 5, 8).bfloat16(), torch.zeros(3, dtype=torch.int32), torch.zeros(6, 5).bfloat16()
    with pytest.raises(RuntimeError, match="no CPU path"):
        grouped_linear(x, w, off)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grouped_linear_grad_weight(g, x, off)
    with pytest.raises(ValueError, match="offsets"):
        grouped_linear(x, w, off.long())
    with pytest.raises(ValueError, match="experts"):
        grouped_linear(x, w, off[:2])
    with pytest.raises(ValueError, match="dims"):
        grouped_linear(x, w[0], off)
    with pytest.raises(ValueError, match="dims"):
        grouped_linear(x[None], w, off)
    with pytest.raises(ValueError, match="operands are"):
        grouped_linear(x.float(), w.float(), off)
    with pytest.raises(ValueError, match="operands are"):
        grouped_linear(x.half(), w, off)
    with pytest.raises(ValueError, match="rows of"):
        grouped_linear(x[:, :7], w, off)
    with pytest.raises(ValueError, match="rows of weight"):
        grouped_linear(g, w.transpose(1, 2), off)
    with pytest.raises(ValueError, match="rows of"):
        grouped_linear_grad_rows(x, w, off)
    with pytest.raises(ValueError, match="rows of grad"):
        grouped_linear_grad_weight(g[:4], x, off)
    with pytest.raises(ValueError, match="element type"):
        grouped_linear_grad_weight(g, x, off, dtype=torch.float64)
    with pytest.raises(ValueError, match="requires a gradient"):
        grouped_linear(x.clone().requires_grad_(), w, off, out=g)
    with pytest.raises(ValueError, match="overlaps"):
        grouped_linear(x, torch.zeros(2, 8, 8).bfloat16(), off, out=x)


def test_entry_points_refuse_what_they_cannot_take():
    lib = nat.lib()
    mul = lambda **k: lib.etha_grouped_matmul(*{**dict(x=0x1000, d=nat.BF16, m=4, xs=8, w=0x1000, e=2, n=8, k=8, ws=8, wg=64, t=0, off=0x1000,
                                                       o=0x1000, od=nat.BF16, os=8, z=1, st=None), **k}.values())
    assert mul(d=nat.F32) == nat.ERR_UNSUPPORTED
    assert mul(od=nat.I8) == nat.ERR_UNSUPPORTED
    assert mul(e=(1 << 16) + 1) == nat.ERR_UNSUPPORTED
    assert mul(m=1 << 31) == nat.ERR_UNSUPPORTED
    for name in ("x", "w", "off", "o"):
        assert mul(**{name: None}) == nat.ERR_INVALID
    assert mul(xs=(1 << 22) + 8) == nat.ERR_UNSUPPORTED and mul(ws=-8) == nat.ERR_UNSUPPORTED
    assert mul(m=0) == 0 and mul(n=0) == 0
    red = lambda **k: lib.etha_grouped_matmul_reduce(*{**dict(g=0x1000, x=0x1000, d=nat.F16, m=4, gs=8, xs=8, e=2, n=8, k=8, off=0x1000,
                                                              o=0x1000, od=nat.F32, os=8, og=64, wk=None, wb=0, st=None), **k}.values())
    assert red(m=4096) == nat.ERR_INVALID and b"workspace" in lib.etha_last_error()
    assert red(m=4096, wk=0x1004, wb=1 << 30) == nat.ERR_INVALID and red(m=4096, wk=0x1000, wb=64) == nat.ERR_INVALID
    assert nat.grouped_matmul_reduce_workspace(4, 2, 8, 8) == 0 and nat.grouped_matmul_reduce_workspace(4096, 2, 8, 8) % (2 * 8 * 8 * 4) == 0
    assert red(d=nat.I8) == nat.ERR_UNSUPPORTED and red(od=nat.F64) == nat.ERR_UNSUPPORTED
    for name in ("g", "x", "off", "o"):
        assert red(**{name: None}) == nat.ERR_INVALID
    assert red(e=0) == 0 and red(n=0) == 0


# ---- values -----------------------------------------------------------------------------------------------------------

CASES = [  # sizes of the groups, out, in, rows before the first and behind the last group
    ([1], 1, 1, 0, 0),
    ([1], 3, 9, 2, 3),
    ([0, 0, 0], 64, 64, 0, 5),
    ([16, 0, 1, 3], 96, 200, 0, 0),
    ([5, 12, 0, 130], 129, 65, 1, 0),
    ([300], 515, 258, 0, 0),
    ([127, 128, 129, 1, 0, 255], 130, 136, 0, 7),
    ([2] * 70, 40, 72, 3, 3),
    ([0] * 64 + [33] + [0] * 70 + [2], 64, 128, 0, 0),
    ([257, 600], 256, 512, 0, 0),
    ([40, 70, 10], 768, 1024, 0, 0),
    ([700, 1, 323], 384, 320, 0, 256),
    ([3000], 130, 72, 2, 1),      # few tiles and many rows: the sum over the rows is cut
    ([5, 1500, 0, 2600], 33, 47, 0, 9),
    ([1, 0, 6, 2], 700, 330, 0, 0),  # few rows, a long sum for the gradient of the rows
    ([16, 17], 1029, 65, 1, 0),
    ([9], 12, 7, 0, 0),           # rows shorter than 16 bytes
    ([140, 30], 5, 300, 0, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES, ids=str)
@pytest.mark.parametrize("sizes,n,k,before,behind", CASES)
def test_products(gpu_device, sizes, n, k, before, behind, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(sum(sizes) + n + k)
    x, weight, offsets, grad = case(gen, sizes, n, k, dtype, gpu_device, before, behind)
    y = grouped_linear(x, weight, offsets)
    assert y.dtype == dtype
    check_rows(y, x, weight, offsets)
    rows, matrices = grouped_linear_grad(grad, x, weight, offsets, weight_dtype=torch.float32)
    assert rows.dtype == dtype and matrices.dtype == torch.float32
    check_rows(rows, grad, weight, offsets, transposed=True)
    check_weight(matrices, grad, x, offsets)
    assert grouped_linear_grad_weight(grad, x, offsets).dtype == dtype
    check_weight(grouped_linear_grad_weight(grad, x, offsets), grad, x, offsets)
    for a, b in ((y, grouped_linear(x, weight, offsets)), (rows, grouped_linear_grad_rows(grad, weight, offsets)),
                 (matrices, grouped_linear_grad_weight(grad, x, offsets, dtype=torch.float32))):
        assert torch.equal(a, b), "the same call gives the same bits"


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[-5, 10, 4, 30, 99], [40, 30, 20, 10, 0], [0, 2 ** 31 - 1, -2 ** 31, 5, 7], [3, 3, 3, 3, 3]])
def test_offsets_that_are_no_offsets(gpu_device, offsets):
    """Entries outside the rows or out of order are taken as the nearest that are not; nothing outside is touched."""
    gen = torch.Generator(device=gpu_device).manual_seed(3)
    x, weight, _, grad = case(gen, [10, 10, 10, 4], 24, 40, torch.bfloat16, gpu_device)
    off = torch.tensor(offsets, dtype=torch.int32, device=gpu_device)
    check_rows(grouped_linear(x, weight, off), x, weight, off)
    rows, matrices = grouped_linear_grad(grad, x, weight, off)
    check_rows(rows, grad, weight, off, transposed=True)
    check_weight(matrices, grad, x, off)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32, torch.float16], ids=str)
def test_rows_of_no_expert_are_left_in_a_given_out(gpu_device, out):
    gen = torch.Generator(device=gpu_device).manual_seed(4)
    x, weight, offsets, grad = case(gen, [3, 0, 200], 70, 90, torch.bfloat16, gpu_device, 5, 150)
    wide = torch.full((x.shape[0], 80), 3.0, device=gpu_device, dtype=out)
    grouped_linear(x, weight, offsets, out=wide[:, 1:71])
    inside = wide[5:208, 1:71].clone()
    wide[5:208, 1:71] = 3.0
    assert bool((wide == 3).all())
    whole = torch.zeros(x.shape[0], 70, dtype=out, device=gpu_device)
    whole[5:208] = inside
    check_rows(whole, x, weight, offsets)
    own = torch.full((3, 70, 90), 3.0, device=gpu_device, dtype=out)
    grouped_linear_grad_weight(grad, x, offsets, out=own)
    check_weight(own, grad, x, offsets)


@pytest.mark.gpu
def test_views(gpu_device):
    """Odd starts and distances, an expert range of a larger set, a column- and a row-parallel part of a weight."""
    gen = torch.Generator(device=gpu_device).manual_seed(5)
    for sizes in ([3, 4, 0, 2, 1], [100, 3, 40, 200, 7]):
        x, weight, offsets, grad = case(gen, sizes, 150, 210, torch.float16, gpu_device)
        xs, ws = x[:, 3:180], weight[1:4, 5:100, 3:180]
        y = grouped_linear(xs, ws, offsets[1:5])
        check_rows(y, xs, ws, offsets[1:5])
        gs = grad[:, 5:100]
        rows, matrices = grouped_linear_grad(gs, xs, ws, offsets[1:5], weight_dtype=torch.float32)
        check_rows(rows, gs, ws, offsets[1:5], transposed=True)
        check_weight(matrices, gs, xs, offsets[1:5])
        one = grad[:1, :1].expand(x.shape[0], 95)  # a broadcast gradient
        check_rows(grouped_linear_grad_rows(one, ws, offsets[1:5]), one, ws, offsets[1:5], transposed=True)
    for rows in (5, 70, 300):  # one row for all: its stride is zero
        x, weight, offsets, grad = case(gen, [rows, 3], 128, 256, torch.bfloat16, gpu_device)
        one, many = grad[:1].expand(rows + 3, 128), x[:1].expand(rows + 3, 256)
        check_weight(grouped_linear_grad_weight(one, x, offsets), one, x, offsets)
        check_weight(grouped_linear_grad_weight(grad, many, offsets), grad, many, offsets)
        check_rows(grouped_linear_grad_rows(one, weight, offsets), one, weight, offsets, transposed=True)
        check_rows(grouped_linear(many, weight, offsets), many, weight, offsets)
        same = weight[:1].expand(2, 128, 256)  # one matrix for all experts
        check_rows(grouped_linear(x, same, offsets), x, same, offsets)


@pytest.mark.gpu
def test_rows_far_apart(gpu_device):
    """Rows 8 MiB apart are read where they lie, rows further apart are copied first."""
    gen = torch.Generator(device=gpu_device).manual_seed(15)
    x, weight, offsets, grad = case(gen, [130, 0, 140], 72, 96, torch.bfloat16, gpu_device)
    for apart in (1 << 22, (1 << 22) + 8):
        far = torch.empty(270, apart, dtype=torch.bfloat16, device=gpu_device)[:, 3:99]
        far.copy_(x)
        check_rows(grouped_linear(far, weight, offsets), x, weight, offsets)
        check_weight(grouped_linear_grad_weight(grad, far, offsets), grad, x, offsets)
        del far


@pytest.mark.gpu
def test_a_single_row_whatever_its_stride(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(16)
    x, weight, offsets, grad = case(gen, [0, 1], 1, 96, torch.bfloat16, gpu_device)
    far = torch.as_strided(x, x.shape, (1 << 30, 1))
    check_rows(grouped_linear(far, weight, offsets), x, weight, offsets)
    check_weight(grouped_linear_grad_weight(grad, far, offsets), grad, x, offsets)
    matrices = torch.as_strided(weight, weight.shape, (96, 1 << 30, 1))  # one row each
    check_rows(grouped_linear(x, matrices, offsets), x, weight, offsets)


@pytest.mark.gpu
def test_nan_stays_in_its_group(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(6)
    for sizes in ([3, 5, 2], [130, 70, 40]):
        x, weight, offsets, grad = case(gen, sizes, 100, 72, torch.bfloat16, gpu_device, 2, 9)
        lo, hi = 2 + sizes[0], 2 + sizes[0] + sizes[1]
        for t in (x, grad):
            t[:2], t[-9:], t[lo:hi] = float("nan"), float("inf"), float("nan")
        y = grouped_linear(x, weight, offsets)
        rows, matrices = grouped_linear_grad(grad, x, weight, offsets)
        for t in (y, rows):
            assert bool(t[lo:hi].isnan().all()) and bool(t[:lo].isfinite().all()) and bool(t[hi:].isfinite().all())
        assert bool(matrices[1].isnan().all()) and bool(matrices[0].isfinite().all()) and bool(matrices[2].isfinite().all())
        weight[0] = float("nan")
        y = grouped_linear(x, weight, offsets)
        assert bool(y[2:lo].isnan().all()) and bool(y[hi:].isfinite().all())


@pytest.mark.gpu
def test_empty(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(7)
    x, weight, offsets, grad = case(gen, [4, 3], 20, 24, torch.bfloat16, gpu_device)
    assert grouped_linear(x[:0], weight, offsets).shape == (0, 20)
    assert grouped_linear(x, weight[:, :0], offsets).shape == (7, 0)
    assert bool((grouped_linear(x[:, :0], weight[:, :, :0], offsets) == 0).all())
    assert bool((grouped_linear(x, weight[:0], offsets[:1]) == 0).all())
    assert grouped_linear_grad_weight(grad, x, offsets[:1]).shape == (0, 20, 24)
    assert bool((grouped_linear_grad_weight(grad[:0], x[:0], offsets) == 0).all())


@pytest.mark.gpu
def test_autograd_gives_the_formulas(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(8)
    x, weight, offsets, grad = case(gen, [30, 0, 41], 66, 50, torch.bfloat16, gpu_device, 2, 3)
    x.requires_grad_()
    weight.requires_grad_()
    y = grouped_linear(x, weight, offsets)
    check_rows(y.detach(), x.detach(), weight.detach(), offsets)
    y.backward(grad)
    check_rows(x.grad, grad, weight.detach(), offsets, transposed=True)
    check_weight(weight.grad, grad, x.detach(), offsets)
    # against differences: y is linear in each input, so a step of any length has no error but the roundings: of y (half a
    # step of bf16 of |y|), of the gradient (half a step of bf16) and of the sums
    for t, other in ((x, weight), (weight, x)):
        step = torch.randn(t.shape, generator=gen, device=gpu_device).bfloat16()
        with torch.no_grad():
            moved = grouped_linear(step, other, offsets) if t is x else grouped_linear(other, step, offsets)
        change = moved.double() * grad.double()
        slope = t.grad.double() * step.double()
        allowed = (2.0 ** -8 + 80 * 2.0 ** -23) * float(change.abs().sum() + slope.abs().sum())
        with torch.no_grad():  # the sums behind a small result may be much larger than it: their own roundings
            size = grouped_linear(step.abs(), other.abs(), offsets) if t is x else grouped_linear(other.abs(), step.abs(), offsets)
        allowed += 2 * 80 * 2.0 ** -23 * float((size.double() * grad.double().abs()).sum()) * (1 + 2.0 ** -7)
        assert abs(float(change.sum() - slope.sum())) <= allowed
    # shared inputs: the gradients of two uses add up in autograd
    x.grad = None
    (grouped_linear(x, weight, offsets).float().sum() + grouped_linear(x, weight, offsets).float().sum()).backward()
    ones = torch.ones_like(grad)
    once = grouped_linear_grad_rows(ones, weight.detach(), offsets)
    assert torch.equal(x.grad, once + once)


@pytest.mark.gpu
def test_capture(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    for sizes in ([3, 0, 2, 4], [200, 10, 0, 300]):
        x, weight, offsets, grad = case(gen, sizes, 256, 192, torch.bfloat16, gpu_device)
        grouped_linear(x, weight, offsets)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = grouped_linear(x, weight, offsets)
            rows, matrices = grouped_linear_grad(grad, x, weight, offsets)
        for k in range(4):
            x.mul_(-0.5)
            grad.add_(1)
            offsets[1:-1] = torch.randint(0, x.shape[0], (3,), generator=gen, device=gpu_device).sort().values.int()  # other sizes
            graph.replay()
            eager = (grouped_linear(x, weight, offsets), *grouped_linear_grad(grad, x, weight, offsets))
            torch.cuda.synchronize()
            for a, b in zip((y, rows, matrices), eager):
                assert torch.equal(a, b)

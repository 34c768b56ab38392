"""Embedding lookup in vocabulary shards and its gradient, against plain forms.

Tolerances.  The lookup is one fp32 product and one rounding: compared bit for bit.  A gradient sums n values in fp32, in
some grouping: each of its n additions rounds a partial sum that is at most A = sum |values|, by at most 2^-24 A; the
products with scale and the value added to (accumulate) add one rounding of 2^-24 each, the result's type half a step.
"""

import numpy as np
import pytest
import torch

from etha_amd import _native as nat
from etha_amd.embedding import embedding, embedding_grad

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain_lookup(tokens, weight, scale, first, dtype):
    local = tokens.long() - first
    here = (local >= 0) & (local < weight.shape[0])
    rows = weight.float()[local.clamp(0, max(weight.shape[0] - 1, 0))] * scale if weight.shape[0] else \
        torch.zeros(*tokens.shape, weight.shape[1], device=weight.device)
    return torch.where(here[..., None], rows, torch.zeros((), device=weight.device)).to(dtype)


def check_gradient(got, grad, tokens, rows, scale, first, before=None):
    """Against sums in 64 bits on the host, with the bound of the module's first lines."""
    g, t = grad.double().cpu().reshape(-1, grad.shape[-1]), tokens.long().cpu().reshape(-1) - first
    here = (t >= 0) & (t < rows)
    width = grad.shape[-1]
    want, size = torch.zeros(rows, width, dtype=torch.float64), torch.zeros(rows, width, dtype=torch.float64)
    count = torch.zeros(rows, dtype=torch.float64)
    want.index_add_(0, t[here], g[here])
    size.index_add_(0, t[here], g[here].abs())
    count.index_add_(0, t[here], torch.ones_like(t[here], dtype=torch.float64))
    want, size = want * scale, size * abs(scale)
    bound = size * (count[:, None] + 2) * 2.0 ** -24
    if before is not None:
        want = want + before.double().cpu()
        bound = bound + (size + before.double().cpu().abs()) * 2.0 ** -24
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # half a step of a subnormal result
    bound = bound + (want.abs() + bound) * torch.finfo(got.dtype).eps / 2 + tiny
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} more than the bound"
    if before is None:
        assert bool((got.cpu()[count == 0] == 0).all())


# ---- refusals (no GPU needed) -------------------------------------------------------------------------------------

def test_refusals():
    w, t = torch.zeros(8, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding(t, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding_grad(torch.zeros(3, 4), t, 8)
    with pytest.raises(ValueError, match="dims"):
        embedding(t, torch.zeros(8))
    with pytest.raises(ValueError, match="int32 and int64"):
        embedding(t.to(torch.int16), w)
    with pytest.raises(ValueError, match="element type"):
        embedding(t, w.double())
    with pytest.raises(ValueError, match="element type"):
        embedding(t, w, dtype=torch.int8)
    with pytest.raises(ValueError, match="contiguous"):
        embedding(t, torch.zeros(4, 8).t())
    with pytest.raises(ValueError, match="shape"):
        embedding(t, w, out=torch.zeros(3, 5))
    with pytest.raises(ValueError, match="an out of"):
        embedding(t, w, out=torch.zeros(3, 4), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="apart"):
        embedding(t, w, out=torch.zeros(4).expand(3, 4))
    with pytest.raises(ValueError, match="overlaps"):
        embedding(t, w, out=w[2:5])
    with pytest.raises(ValueError, match="requires a gradient"):
        embedding(t, w.clone().requires_grad_(), out=torch.zeros(3, 4))
    with pytest.raises(ValueError, match="requires a gradient"):
        embedding(t, w, out=torch.zeros(3, 4, requires_grad=True))
    with pytest.raises(ValueError, match="grad has shape"):
        embedding_grad(torch.zeros(4, 4), t, 8)
    with pytest.raises(ValueError, match="accumulate needs an out"):
        embedding_grad(torch.zeros(3, 4), t, 8, accumulate=True)
    with pytest.raises(ValueError, match="rows"):
        embedding_grad(torch.zeros(3, 4), t, -1)
    with pytest.raises(ValueError, match="shape"):
        embedding_grad(torch.zeros(3, 4), t, 8, out=torch.zeros(7, 4))


def test_entry_points_refuse_what_they_cannot_take():
    lib = nat.lib()
    look = lambda **k: lib.etha_embedding(*{**dict(t=0x1000, td=nat.I32, n=4, w=0x1000, wd=nat.F32, r=8, h=4, ws=4, f=0, s=1.0,
                                                   o=0x1000, od=nat.F32, os=4, st=None), **k}.values())
    assert look(td=nat.I16) == nat.ERR_INVALID
    assert look(t=None) == nat.ERR_INVALID
    assert look(w=None) == nat.ERR_INVALID
    assert look(o=None) == nat.ERR_INVALID
    assert look(wd=nat.F64) == nat.ERR_UNSUPPORTED
    assert look(od=nat.I8) == nat.ERR_UNSUPPORTED
    assert look(n=1 << 31) == nat.ERR_UNSUPPORTED
    assert look(r=1 << 31) == nat.ERR_UNSUPPORTED
    assert look(h=1 << 25) == nat.ERR_UNSUPPORTED
    assert look(n=0) == 0 and look(h=0) == 0  # nothing to do: nothing is launched
    grad = lambda **k: lib.etha_embedding_grad(*{**dict(g=0x1000, gd=nat.F32, gs=4, t=0x1000, td=nat.I32, n=4000, r=8, h=4, f=0, s=1.0,
                                                        o=0x1000, od=nat.F32, os=4, a=0, ws=0x1000, wb=1 << 20, st=None), **k}.values())
    assert grad(gd=nat.F64) == nat.ERR_UNSUPPORTED
    assert grad(wb=0) == nat.ERR_INVALID and b"workspace" in lib.etha_last_error()
    assert grad(ws=None) == nat.ERR_INVALID
    assert grad(ws=0x1004) == nat.ERR_INVALID
    assert grad(g=None) == nat.ERR_INVALID
    assert grad(r=0) == 0 and grad(n=0, a=1) == 0
    assert grad(n=(1 << 26) + 1) == nat.ERR_UNSUPPORTED and grad(n=(1 << 21) + 1, r=1 << 25) == nat.ERR_UNSUPPORTED
    need = nat.embedding_grad_workspace
    assert need(0, 8, 4, nat.F32) == 0 and need(4000, 8, 4, nat.F32) > 0
    with pytest.raises(nat.EthaNativeError):
        need(1, 8, 4, nat.I32)
    assert need(1 << 26, 8, 4, nat.F32) > 0
    with pytest.raises(nat.EthaNativeError):
        need((1 << 26) + 1, 8, 4, nat.F32)


# ---- lookup ---------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("out", DTYPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,rows,width", [(1, 1, 1), (1, 700, 4096), (5, 100, 7), (257, 33, 64), (64, 50, 1001), (1000, 9, 2056)])
def test_lookup(gpu_device, tokens, rows, width, dtype, out):
    gen = torch.Generator(device=gpu_device).manual_seed(tokens + width)
    weight = torch.randn(rows, width, generator=gen, device=gpu_device).to(dtype)
    ids = torch.randint(-3, 2 * rows + 3, (tokens,), generator=gen, device=gpu_device)  # half of them are other shards'
    for id_type in (torch.int64, torch.int32):
        got = embedding(ids.to(id_type), weight, scale=3.7, first_row=2, dtype=out)
        want = plain_lookup(ids, weight, 3.7, 2, out)
        assert got.dtype == out and torch.equal(got, want)


@pytest.mark.gpu
def test_lookup_of_views_and_extreme_ids(gpu_device):
    base = torch.randn(40, 131, device=gpu_device).bfloat16()
    weight = base[3:, 1:100]  # odd start, odd width, rows 131 apart
    ids = torch.tensor([[0, 36, 37], [-2 ** 62, 2 ** 62, 2 ** 32]], device=gpu_device)
    out = torch.full((2, 3, 110), 7.0, device=gpu_device)
    got = embedding(ids, weight, out=out[..., 4:103])
    assert torch.equal(got, plain_lookup(ids, weight, 1.0, 0, torch.float32))
    assert bool((out[..., :4] == 7).all()) and bool((out[..., 103:] == 7).all())
    assert torch.equal(embedding(ids.t(), weight), plain_lookup(ids.t(), weight, 1.0, 0, torch.bfloat16))
    far = embedding(ids, weight, first_row=-2 ** 62)
    assert torch.equal(far[1, 0], weight[0]) and int((far != 0).any(-1).sum()) == 1
    assert embedding(ids[:0], weight).shape == (0, 3, 99)
    assert embedding(ids, weight[:, :0]).shape == (2, 3, 0)
    assert bool((embedding(ids, weight[:0]) == 0).all())
    assert torch.equal(embedding(ids[0, 0], weight), weight[0])


@pytest.mark.gpu
def test_lookup_keeps_special_values(gpu_device):
    weight = torch.tensor([[float("inf"), float("-inf"), float("nan"), -0.0, 1e-42, 3e38]], device=gpu_device)
    got = embedding(torch.zeros(1, dtype=torch.int64, device=gpu_device), weight)
    assert torch.equal(got.view(torch.int32)[0, [0, 1, 3, 4, 5]], weight.view(torch.int32)[0, [0, 1, 3, 4, 5]]) and bool(got[0, 2].isnan())


@pytest.mark.gpu
def test_lookup_in_a_table_past_32_bits(gpu_device):
    """Row offsets beyond 2^32 elements: 2^21 rows of 2056 bytes' width (4.3 G elements of fp16)."""
    rows, width = (1 << 21) + 5, 2056
    weight = torch.empty(rows, width, dtype=torch.float16, device=gpu_device)
    ids = torch.tensor([0, 1, 1 << 20, rows - 1, rows], device=gpu_device)
    weight[ids[:4]] = torch.randn(4, width, device=gpu_device).half()
    got = embedding(ids, weight)
    assert torch.equal(got[:4], weight[ids[:4]]) and bool((got[4] == 0).all())


# ---- gradient -------------------------------------------------------------------------------------------------------

GRADIENT_CASES = [
    # tokens, rows, width, vocabulary (tokens outside rows are other shards')
    (1, 1, 1, 1), (1, 500, 64, 500), (7, 3, 5, 9), (63, 64, 130, 64), (64, 65, 512, 65), (65, 1, 1001, 1), (509, 4000, 1001, 32000), (512, 30, 2060, 40), (513, 30, 1032, 40), (700, 5000, 20, 9000),
    (1025, 2, 96, 2), (3000, 511, 72, 700), (8192, 100000, 40, 100000), (8193, 513, 64, 600), (20000, 1, 136, 3), (12289, 70000, 33, 140000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                       (torch.float16, torch.float16), (torch.float32, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("tokens,rows,width,vocab", GRADIENT_CASES)
def test_gradient(gpu_device, tokens, rows, width, vocab, dtype, out):
    gen = torch.Generator(device=gpu_device).manual_seed(tokens * 7 + rows)
    grad = torch.randn(tokens, width, generator=gen, device=gpu_device).to(dtype)
    first = (vocab - rows) // 2
    # squares: low ids are frequent, so that some rows take many tokens and some none
    ids = (torch.rand(tokens, generator=gen, device=gpu_device).square() * vocab).long().clamp(max=vocab - 1)
    got = embedding_grad(grad, ids, rows, scale=0.75, first_row=first, dtype=out)
    assert got.dtype == out and got.shape == (rows, width)
    check_gradient(got, grad, ids, rows, 0.75, first)
    again = embedding_grad(grad, ids.int(), rows, scale=0.75, first_row=first, dtype=out)
    assert torch.equal(got, again), "the same call gives the same bits"


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [300, 9000, 70000])
@pytest.mark.parametrize("id_of", ["one", "none", "ends"])
def test_gradient_of_repeated_tokens(gpu_device, tokens, id_of):
    grad = torch.randn(tokens, 24, device=gpu_device)
    ids = torch.full((tokens,), 5, device=gpu_device, dtype=torch.int32)
    if id_of == "none":
        ids = torch.where(torch.arange(tokens, device=gpu_device) % 2 == 0, -1, 11).int()
    elif id_of == "ends":
        ids[tokens // 2:] = 10
        ids[: tokens // 3] = 0
    check_gradient(embedding_grad(grad, ids, 11), grad, ids, 11, 1.0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,rows", [(5000, 600000), (5000, 262144), (5000, 262145), (40000, 256), (40000, 257), (40000, 1024)])
def test_gradient_by_number_of_rows(gpu_device, tokens, rows):
    """From more rows than the workgroups that group the tokens have room for, to one row a workgroup."""
    gen = torch.Generator(device=gpu_device).manual_seed(rows)
    grad = torch.randn(tokens, 3, generator=gen, device=gpu_device)
    ids = torch.randint(-5, rows + 5, (tokens,), generator=gen, device=gpu_device)
    check_gradient(embedding_grad(grad, ids, rows), grad, ids, rows, 1.0, 0)


@pytest.mark.gpu
def test_gradient_of_a_padded_batch(gpu_device):
    """One token half of the time in a part of the batch: some waves meet more of a workgroup's tokens than they can note."""
    gen = torch.Generator(device=gpu_device).manual_seed(8)
    grad = torch.randn(60000, 40, generator=gen, device=gpu_device).bfloat16()
    ids = torch.randint(0, 3000, (60000,), generator=gen, device=gpu_device)
    ids[20000:][torch.rand(40000, generator=gen, device=gpu_device) < 0.5] = 7
    ids[50000:] = 7
    check_gradient(embedding_grad(grad, ids, 3000, dtype=torch.float32), grad, ids, 3000, 1.0, 0)


@pytest.mark.gpu
def test_gradient_accumulates_and_leaves_the_rest(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(1)
    for tokens in (40, 10000):
        wide = torch.randn(90, 80, generator=gen, device=gpu_device)
        before = wide.clone()
        out = wide[2:82, 3:70]  # a view: odd start, odd width
        grad = torch.randn(tokens, 2, 67, generator=gen, device=gpu_device).bfloat16().transpose(0, 1)  # rows at two distances
        ids = torch.randint(0, 40, (2, tokens), generator=gen, device=gpu_device)
        got = embedding_grad(grad, ids, 80, scale=2.0, out=out, accumulate=True)
        assert got.data_ptr() == out.data_ptr()
        check_gradient(got, grad, ids, 80, 2.0, 0, before=before[2:82, 3:70])
        assert torch.equal(out[40:], before[42:82, 3:70]), "rows without a token are not touched"
        wide[2:82, 3:70] = before[2:82, 3:70]
        assert torch.equal(wide, before), "nothing around the view is touched"


@pytest.mark.gpu
def test_gradient_of_nothing(gpu_device):
    none = torch.empty(0, dtype=torch.int64, device=gpu_device)
    assert bool((embedding_grad(torch.empty(0, 70, device=gpu_device), none, 130) == 0).all())
    assert embedding_grad(torch.empty(5, 0, device=gpu_device), torch.zeros(5, dtype=torch.int64, device=gpu_device), 3).shape == (3, 0)
    assert embedding_grad(torch.ones(5, 4, device=gpu_device), torch.zeros(5, dtype=torch.int64, device=gpu_device), 0).shape == (0, 4)
    out = torch.ones(3, 4, device=gpu_device)
    embedding_grad(torch.empty(0, 4, device=gpu_device), none, 3, out=out, accumulate=True)
    assert bool((out == 1).all())


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_rows(gpu_device):
    grad = torch.randn(100, 70, device=gpu_device)
    grad[3, 5], grad[4, 6], grad[9] = float("nan"), float("inf"), float("nan")
    ids = torch.arange(100, device=gpu_device) % 7
    ids[9] = 50  # another shard's
    got = embedding_grad(grad, ids, 7)
    bad = ~got.isfinite()
    assert int(bad.sum()) == 2 and bool(bad[3, 5]) and bool(bad[4, 6])


@pytest.mark.gpu
def test_autograd_gives_the_formula(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(2)
    weight = torch.randn(50, 33, generator=gen, device=gpu_device, requires_grad=True)
    ids = torch.randint(0, 60, (4, 9), generator=gen, device=gpu_device)
    up = torch.randn(4, 9, 33, generator=gen, device=gpu_device)
    embedding(ids, weight, scale=1.5, first_row=4).backward(up)
    check_gradient(weight.grad, up, ids, 50, 1.5, 4)
    # against differences: the lookup is linear in the weight, so one difference along a direction has no error of its own
    # beyond the roundings of the two sums of 1188 fp32 products (2^-24 each, of at most their absolute sum)
    step = torch.randn(50, 33, generator=gen, device=gpu_device)
    moved = (embedding(ids, step, scale=1.5, first_row=4).double() * up.double())
    slope = (weight.grad.double() * step.double())
    assert abs(float(moved.sum() - slope.sum())) <= 1188 * 2.0 ** -23 * float(moved.abs().sum() + slope.abs().sum())
    weight.grad = None
    embedding(ids, weight).sum().backward()  # an expanded gradient: all its rows are one
    check_gradient(weight.grad, torch.ones(4, 9, 33), ids, 50, 1.0, 0)


@pytest.mark.gpu
def test_capture_and_streams(gpu_device):
    """Captured calls give the eager results on every replay, with other work between them; a backward pass is refused."""
    weight = torch.randn(300, 200, device=gpu_device).bfloat16()
    ids = torch.randint(0, 300, (9000,), device=gpu_device)
    grad = torch.randn(9000, 200, device=gpu_device).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = embedding_grad(embedding(ids, weight), ids, 300)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, embedding_grad(weight[ids], ids, 300))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = embedding(ids, weight, scale=2.0)
        total = embedding_grad(grad, ids, 300)
    for k in range(4):
        ids.copy_(torch.randint(0, 300 - 60 * k, (9000,), device=gpu_device))
        grad.mul_(-0.5)
        graph.replay()
        eager_rows, eager_total = embedding(ids, weight, scale=2.0), embedding_grad(grad, ids, 300)
        torch.cuda.synchronize()
        assert torch.equal(rows, eager_rows) and torch.equal(total, eager_total)


@pytest.mark.gpu
def test_two_graphs_replayed_in_turn(gpu_device):
    """Each graph has a workspace of its own, also where they share a pool."""
    ids = [torch.randint(0, 40, (n,), device=gpu_device) for n in (9000, 12000)]
    grad = [torch.randn(i.numel(), 72, device=gpu_device) for i in ids]
    graphs, totals, pool = [], [], None
    for i, g in zip(ids, grad):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            totals.append(embedding_grad(g, i, 40))
        pool = pool or graph.pool()
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for k in order:
            ids[k].copy_(torch.randint(0, 40, ids[k].shape, device=gpu_device))
            graphs[k].replay()
            eager = embedding_grad(grad[k], ids[k], 40)
            torch.cuda.synchronize()
            assert torch.equal(totals[k], eager)


@pytest.mark.gpu
def test_two_streams_at_once(gpu_device):
    ids = torch.randint(0, 500, (2, 30000), device=gpu_device)
    grad = torch.randn(2, 30000, 136, device=gpu_device)
    want = [embedding_grad(g, i, 500) for g, i in zip(grad, ids)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(embedding_grad(grad[k], ids[k], 500))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[k]) for k in (0, 1) for g in got[k])


@pytest.mark.gpu
def test_captured_backward_is_refused(gpu_device):
    from etha_amd._operands import refuse_captured_backward

    x = torch.zeros(4, device=gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            refuse_captured_backward("embedding")
        x.add_(1)
    graph.replay()
    refuse_captured_backward("embedding")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,rows,width,dtype", [(700, (1 << 26) + 5, 1, torch.float32), (40, (1 << 28) + 21, 2, torch.bfloat16)])
def test_gradient_of_more_rows_than_a_grid_takes(gpu_device, tokens, rows, width, dtype):
    gen = torch.Generator(device=gpu_device).manual_seed(rows)
    ids = torch.randint(0, rows, (tokens,), generator=gen, device=gpu_device)
    ids[:4] = torch.tensor([0, rows - 1, rows - 1, rows // 2], device=gpu_device)
    grad = (torch.rand(tokens, width, generator=gen, device=gpu_device) + 1).to(dtype)
    out = torch.full((rows, width), 3.0, dtype=dtype, device=gpu_device)
    embedding_grad(grad, ids, rows, out=out)
    there = ids.unique()
    assert int((out != 0).any(1).sum()) == there.numel()  # all others are zeros
    small = torch.searchsorted(there, ids)
    check_gradient(out[there], grad, small, there.numel(), 1.0, 0)
    before = out[there].clone()
    embedding_grad(grad, ids, rows, out=out, accumulate=True)
    assert int((out != 0).any(1).sum()) == there.numel()
    check_gradient(out[there], grad, small, there.numel(), 1.0, 0, before=before)


@pytest.mark.parametrize("graph", [False, True])
def test_scale_and_first_row_of_any_number_type(monkeypatch, graph):
    """The same numbers are taken with and without a graph, and none is wrapped around."""
    from etha_amd import embedding as module

    seen = []
    monkeypatch.setattr(module, "check_device", lambda what, first, *others: 0)
    monkeypatch.setattr(module, "call", lambda index, name, *args: seen.append(args))
    weight, tokens = torch.zeros(8, 4).requires_grad_(graph), torch.zeros(3, dtype=torch.int64)
    for scale in (2.0, 2, np.float32(2), np.float64(2), torch.tensor(2.0)):
        for first in (3, np.int64(3), torch.tensor(3)):
            embedding(tokens, weight, scale=scale, first_row=first)
            embedding_grad(torch.zeros(3, 4), tokens, 8, scale=scale, first_row=first)
    for args in seen:
        first, scale = (args[8], args[9])
        assert type(first) is int and type(scale) is float and (first, scale) == (3, 2.0)
    for call in (lambda **k: embedding(tokens, weight, **k), lambda **k: embedding_grad(torch.zeros(3, 4), tokens, 8, **k)):
        call(first_row=-2 ** 63)
        call(first_row=2 ** 63 - 1)
        for first in (2 ** 63, -2 ** 63 - 1, 2 ** 64):
            with pytest.raises(ValueError, match="first_row"):
                call(first_row=first)
        with pytest.raises(TypeError):
            call(first_row=1.5)

"""What autograd learns of the operators on local shards: buffers that a call writes, derivatives that it does not have.

On the CPU a stand-in takes the place of the launch: everything asked for here happens on the host.
"""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from etha_amd import embedding as embedding_module, experts as experts_module, int8 as int8_module
from etha_amd.embedding import embedding, embedding_grad
from etha_amd.experts import grouped_linear, grouped_linear_grad, grouped_linear_grad_rows, grouped_linear_grad_weight
from etha_amd.int8 import Int8Weight, int8_linear, int8_matmul, quantize_rows


@pytest.fixture(params=["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "gpu":
        return request.getfixturevalue("gpu_device")
    for module in (embedding_module, experts_module, int8_module):
        monkeypatch.setattr(module, "check_device", lambda what, first, *others: 0)
        monkeypatch.setattr(module, "call", lambda index, name, *args: None)
    return torch.device("cpu")


class Operands:
    def __init__(self, device):
        zeros = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device=device)
        self.tokens = zeros(6, dtype=torch.int64)
        self.table, self.rows = zeros(5, 8), zeros(6, 8)
        self.x, self.up, self.weight = zeros(6, 8).bfloat16(), zeros(6, 16).bfloat16(), zeros(2, 16, 8).bfloat16()
        self.offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device=device)
        self.q, self.w = zeros(6, 8, dtype=torch.int8), zeros(16, 8, dtype=torch.int8)
        self.row_scales, self.col_scales, self.bias = zeros(6), zeros(16), zeros(16)
        self.zeros = zeros


# name -> (shape of what it writes, a call that writes it)
WRITERS = {
    "embedding": ((6, 8), lambda o, out: embedding(o.tokens, o.table, out=out)),
    "embedding_grad": ((5, 8), lambda o, out: embedding_grad(o.rows, o.tokens, 5, out=out)),
    "embedding_grad, accumulate": ((5, 8), lambda o, out: embedding_grad(o.rows, o.tokens, 5, out=out, accumulate=True)),
    "grouped_linear": ((6, 16), lambda o, out: grouped_linear(o.x, o.weight, o.offsets, out=out)),
    "grouped_linear_grad_rows": ((6, 8), lambda o, out: grouped_linear_grad_rows(o.up, o.weight, o.offsets, out=out)),
    "grouped_linear_grad_weight": ((2, 16, 8), lambda o, out: grouped_linear_grad_weight(o.up, o.x, o.offsets, out=out)),
    "quantize_rows, scales": ((6,), lambda o, out: quantize_rows(o.rows, scales=out)),
    "int8_matmul": ((6, 16), lambda o, out: int8_matmul(o.q, o.row_scales, o.w, o.col_scales, out=out)),
    "int8_linear": ((6, 16), lambda o, out: int8_linear(o.rows, o.w, o.col_scales, out=out)),
}


@pytest.mark.parametrize("name", WRITERS)
def test_a_saved_buffer_that_is_written_again_is_noticed(device, name):
    """A graph holds the buffer that a call writes: a later backward pass through it must not use the new values."""
    shape, write = WRITERS[name]
    o = Operands(device)
    buffer, p = o.zeros(*shape), o.zeros(*shape).requires_grad_()
    with torch.no_grad():
        write(o, buffer)
    z = (buffer * p).sum()
    z.backward(retain_graph=True)  # what was written before is no trouble
    with torch.no_grad():
        write(o, buffer)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_views_and_integers_that_are_written_are_noticed(device):
    o = Operands(device)
    wide = o.zeros(6, 20)
    before = wide._version
    embedding(o.tokens, o.table, out=wide[:, 3:11])
    assert wide._version == before + 1
    values = o.zeros(6, 8, dtype=torch.int8)
    quantize_rows(o.rows, values=values)
    assert values._version == 1
    weight = Int8Weight(o.zeros(16, 8))
    before = weight.values._version, weight.scales._version, weight.landing._version
    weight.refresh()
    assert (weight.values._version, weight.scales._version, weight.landing._version) == (before[0] + 1, before[1] + 1, before[2])


def test_inference_tensors_are_written(device):
    o = Operands(device)
    with torch.inference_mode():
        buffer = o.zeros(6, 8)
        embedding(o.tokens, o.table, out=buffer)
    embedding(o.tokens, o.table, out=buffer)  # they count no versions


# name -> (floating-point operands, the call on them); every one of them may carry a tangent
DERIVATIVES = {
    "embedding": (("table",), lambda o, t: embedding(o.tokens, t["table"])),
    "embedding_grad": (("rows",), lambda o, t: embedding_grad(t["rows"], o.tokens, 5)),
    "grouped_linear": (("x", "weight"), lambda o, t: grouped_linear(t["x"], t["weight"], o.offsets)),
    "grouped_linear_grad_rows": (("up", "weight"), lambda o, t: grouped_linear_grad_rows(t["up"], t["weight"], o.offsets)),
    "grouped_linear_grad_weight": (("up", "x"), lambda o, t: grouped_linear_grad_weight(t["up"], t["x"], o.offsets)),
    "quantize_rows": (("rows",), lambda o, t: quantize_rows(t["rows"])),
    "int8_matmul": (("row_scales", "col_scales", "bias"),
                    lambda o, t: int8_matmul(o.q, t["row_scales"], o.w, t["col_scales"], bias=t["bias"])),
    "int8_linear": (("rows", "col_scales", "bias"), lambda o, t: int8_linear(t["rows"], o.w, t["col_scales"], bias=t["bias"])),
}
OPERANDS = [(name, operand) for name, (operands, _) in DERIVATIVES.items() for operand in operands]


def operands_of(o, name):
    return {operand: getattr(o, operand) for operand in DERIVATIVES[name][0]}


@pytest.mark.parametrize("name,operand", OPERANDS)
def test_a_tangent_is_refused(device, name, operand):
    """No call has a forward-mode derivative: one that dropped the tangent would stand for a derivative of zero."""
    o = Operands(device)
    call, given = DERIVATIVES[name][1], operands_of(Operands(device), name)
    with fwd.dual_level():
        call(o, given)  # a level alone is no trouble
        quantize_rows(o.rows, values=o.q, scales=o.row_scales)
        given[operand] = fwd.make_dual(given[operand], torch.ones_like(given[operand]))
        with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
            call(o, given)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):  # which does not switch tangents off
            call(o, given)
        if name in ("embedding", "grouped_linear"):  # nor does another operand's gradient
            given[operand].requires_grad_()
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(o, given)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: call(o, {**operands_of(o, name), operand: t}), (getattr(o, operand),), (getattr(o, operand),))


@pytest.mark.parametrize("name", WRITERS)
def test_a_tangent_of_the_output_is_refused(device, name):
    shape, write = WRITERS[name]
    o = Operands(device)
    with fwd.dual_level():
        out = fwd.make_dual(o.zeros(*shape), o.zeros(*shape))
        with pytest.raises(RuntimeError, match="forward-mode"):
            write(o, out)


@pytest.mark.parametrize("name,operand", [(n, t) for n, t in OPERANDS if n not in ("embedding", "grouped_linear")])
def test_a_call_without_a_gradient_refuses_to_cut_a_graph(device, name, operand):
    """One rule for all that have none, the gradient functions among them: operands come detached, or under no_grad."""
    o = Operands(device)
    call, given = DERIVATIVES[name][1], operands_of(o, name)
    given[operand] = given[operand].clone().requires_grad_()
    with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
        call(o, given)
    with torch.no_grad():
        call(o, given)
    given[operand] = given[operand].detach()
    call(o, given)


def test_both_gradients_refuse_before_either_runs(device):
    o = Operands(device)
    for k in range(3):
        operands = [o.up, o.x, o.weight]
        operands[k] = operands[k].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="grouped_linear_grad has no gradient"):
            grouped_linear_grad(*operands, o.offsets)

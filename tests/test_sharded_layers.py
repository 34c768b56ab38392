"""The operators together, on shards that a transfer has just delivered.

A small mixture-of-experts model goes from a trainer's layout to an inference layout; tokens then run through the delivered
shards as the inference ranks would run them, and Partial results through the framework's own reduction.  Every step is
compared with a plain form in 64 bits of the step's own inputs, within the bounds that tests/test_embedding.py,
tests/test_int8.py and tests/test_experts.py derive.
"""

import numpy as np
import pytest
import torch
from torch.distributed.tensor.placement_types import Partial, Replicate, Shard

from etha_amd.comm import LoopbackWire
from etha_amd.embedding import embedding, embedding_grad
from etha_amd.experts import grouped_linear, grouped_linear_grad
from etha_amd.int8 import Int8Weight, int8_linear
from etha_amd.layout import local_shard
from etha_amd.tensor_bus.client import BatchHandler, TensorBusClient
from etha_amd.tensor_bus.command_queue import Completion
from etha_amd.world import ReshardJob, TensorSpec

from test_embedding import check_gradient, plain_lookup
from test_experts import check_rows, check_weight
from test_int8 import check_product, check_rows as check_int8_rows, plain_rows
from test_tensor_bus import _client, agent_factory, run_ranks  # noqa: F401

TRAINER, EXPERTS, HIDDEN, INNER, VOCAB, OUT = list(range(8)), 8, 128, 192, 1003, 88


def specs():
    return [
        TensorSpec("embed", (VOCAB, HIDDEN), TRAINER[:6], (Shard(0),), [8, 9, 10, 11], (Shard(1),), torch.float32, torch.bfloat16, seed=1, std=1.0),
        TensorSpec("w1", (EXPERTS, INNER, HIDDEN), TRAINER, (Shard(0),), [8, 9, 10, 11], (Shard(1),), torch.bfloat16, seed=2, std=0.1),
        TensorSpec("w2", (EXPERTS, HIDDEN, INNER), TRAINER, (Shard(0),), [8, 9, 10, 11], (Shard(2),), torch.bfloat16, seed=3, std=0.1),
        TensorSpec("head", (OUT, HIDDEN), TRAINER, (Shard(0),), [8, 9], (Shard(0),), torch.float32, torch.bfloat16, seed=4, std=0.1, target_int8=True),
    ]


def collapse(parts, device):
    """The members of a Partial("sum") through the framework's reduction, to one rank."""
    n = len(parts)
    job = ReshardJob([TensorSpec("y", tuple(parts[0].shape), list(range(n)), (Partial("sum"),), [n], (Replicate(),), parts[0].dtype)], device=device)
    for r, part in enumerate(parts):
        job.source_locals[0][r].copy_(part)
    job.run()
    return job.target_locals[0][n]


def check_sum(got, parts):
    """fp32 sums in rank order (a rounding for each, of at most the sum of magnitudes), half a step of the type."""
    exact = sum(p.double() for p in parts)
    size = sum(p.double().abs() for p in parts)
    bound = (len(parts) - 1) * 2.0 ** -24 * size
    bound = bound + (exact.abs() + bound) * torch.finfo(got.dtype).eps / 2
    assert bool(((got.double() - exact).abs() <= bound).all())


@pytest.mark.gpu
def test_tokens_through_delivered_shards(gpu_device):
    job = ReshardJob(specs(), device=gpu_device, keep_globals=True)
    job.run()
    gen = torch.Generator(device=gpu_device).manual_seed(5)
    tokens = torch.randint(0, VOCAB, (157,), generator=gen, device=gpu_device)
    # vocabulary shards, the last one shorter: each gives its rows and zeros, the sum is the lookup
    shards = job.source_locals[0]
    rows = -(-VOCAB // 6)
    assert [shards[r].shape[0] for r in range(6)] == [rows] * 5 + [VOCAB - 5 * rows]
    parts = [embedding(tokens, shards[r], first_row=r * rows, dtype=torch.bfloat16) for r in range(6)]
    for r, part in enumerate(parts):
        assert torch.equal(part, plain_lookup(tokens, shards[r], 1.0, r * rows, torch.bfloat16))
    x = collapse(parts, gpu_device)
    # column shards, as they were delivered: parts of the row
    wide = torch.cat([embedding(tokens, job.target_locals[0][r]) for r in (8, 9, 10, 11)], 1)
    assert torch.equal(x, wide) and torch.equal(x, job.globals_[0].bfloat16()[tokens])  # one term is not zero: the sum is exact
    # rows sorted by expert, column-parallel, then row-parallel: the second product's results are members of a Partial
    expert = torch.randint(0, EXPERTS - 1, (157,), generator=gen, device=gpu_device)  # one expert gets nothing
    order = expert.argsort(stable=True)
    offsets = torch.zeros(EXPERTS + 1, dtype=torch.int32, device=gpu_device)
    offsets[1:] = torch.bincount(expert, minlength=EXPERTS).cumsum(0)
    xs = x[order]
    w1, w2 = job.target_locals[1], job.target_locals[2]
    partials = []
    for r in (8, 9, 10, 11):
        inner = grouped_linear(xs, w1[r], offsets)
        check_rows(inner, xs, w1[r], offsets)
        inner = torch.relu(inner)
        partials.append(grouped_linear(inner, w2[r], offsets))
        check_rows(partials[-1], inner, w2[r], offsets)
    y = collapse(partials, gpu_device)
    check_sum(y, partials)
    # an expert range, as a rank of an expert-parallel layout holds it: the other experts' rows stay zero
    mine = job.source_locals[1]
    for r in (0, 6):
        part = grouped_linear(xs, mine[r], offsets[r:r + 2])
        check_rows(part, xs, mine[r], offsets[r:r + 2])
    # the head in 8 bits, a shard of its channels on either rank
    for r in (8, 9):
        weight = job.target_int8[3][r]
        assert weight.landing is job.target_locals[3][r]
        check_int8_rows(weight.landing, weight.values, weight.scales)
        for batch in (y, y[:1]):
            logits = weight.linear(batch, dtype=torch.float32)
            q, s = plain_rows(batch)
            check_product(logits, q, s, weight.values, weight.scales, None)
            assert torch.equal(logits, int8_linear(batch, weight.values, weight.scales, dtype=torch.float32))
    # new weights through the same job: the converted ones follow, at their addresses
    before = {r: job.target_int8[3][r].values.data_ptr() for r in (8, 9)}
    for t in job.source_locals[3].values():
        t.mul_(-2.0)
    job.run()
    for r in (8, 9):
        weight = job.target_int8[3][r]
        assert weight.values.data_ptr() == before[r]
        check_int8_rows(weight.landing, weight.values, weight.scales)
        assert torch.equal(weight.landing, local_shard(-2.0 * job.globals_[3], (2,), (Shard(0),), (r - 8,)).bfloat16())


@pytest.mark.gpu
def test_gradients_on_the_trainers_shards(gpu_device):
    """The way back on the trainer's layout: gradients of its expert and vocabulary shards are the parts of the whole ones."""
    job = ReshardJob(specs(), device=gpu_device, keep_globals=True)
    gen = torch.Generator(device=gpu_device).manual_seed(6)
    tokens = torch.randint(0, VOCAB, (300,), generator=gen, device=gpu_device)
    expert = torch.randint(0, EXPERTS, (300,), generator=gen, device=gpu_device)
    order = expert.argsort(stable=True)
    offsets = torch.zeros(EXPERTS + 1, dtype=torch.int32, device=gpu_device)
    offsets[1:] = torch.bincount(expert, minlength=EXPERTS).cumsum(0)
    w1 = job.globals_[1]
    table = job.globals_[0].bfloat16()
    xs = embedding(tokens, table)[order]
    up = torch.randn(300, INNER, generator=gen, device=gpu_device).bfloat16()
    rows, matrices = grouped_linear_grad(up, xs, w1, offsets, weight_dtype=torch.float32)
    check_rows(rows, up, w1, offsets, transposed=True)
    check_weight(matrices, up, xs, offsets)
    parts = []
    for r in TRAINER:  # Shard(0)@8: an expert each
        part, matrix = grouped_linear_grad(up, xs, job.source_locals[1][r], offsets[r:r + 2], weight_dtype=torch.float32)
        assert torch.equal(matrix[0], matrices[r])
        parts.append(part)
    assert torch.equal(sum(p.float() for p in parts), rows.float())  # one of them is not zero in a row
    back = torch.empty_like(rows)
    back[order] = rows
    whole = embedding_grad(back, tokens, VOCAB, dtype=torch.float32)
    check_gradient(whole, back, tokens, VOCAB, 1.0, 0)
    n = -(-VOCAB // 6)
    for r in TRAINER[:6]:
        shard = job.source_locals[0][r]
        part = embedding_grad(back, tokens, shard.shape[0], first_row=r * n, dtype=torch.float32)
        assert torch.equal(part, whole[r * n:r * n + shard.shape[0]])
    # autograd through the same steps
    table.requires_grad_()
    w1 = w1.clone().requires_grad_()
    grouped_linear(embedding(tokens, table)[order], w1, offsets).backward(up)
    assert torch.equal(w1.grad, grouped_linear_grad(up, xs, w1.detach(), offsets)[1])
    check_gradient(table.grad, back, tokens, VOCAB, 1.0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("pool", ["ring", "resident"])
def test_a_captured_transfer_converts_its_weights(gpu_device, pool):
    spec = TensorSpec("w", (96, 640), [0, 1], (Shard(0),), [2], (Replicate(),), torch.float32, torch.bfloat16, seed=1, target_int8=True)
    job = ReshardJob([spec], device=gpu_device, pool=pool)
    job.run()
    weight = job.target_int8[0][2]
    check_int8_rows(weight.landing, weight.values, weight.scales)
    if pool == "ring":
        return
    graph = job.capture()
    for k in range(3):
        for t in job.source_locals[0].values():
            t.add_(0.01 * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(weight.landing, torch.cat([job.source_locals[0][r] for r in (0, 1)]).bfloat16())
        check_int8_rows(weight.landing, weight.values, weight.scales)


@pytest.mark.gpu
def test_an_8_bit_weight_through_the_bus(gpu_device, agent_factory):  # noqa: F811
    agent, naming = agent_factory(3, device=gpu_device)
    src = {r: torch.randn(40, 96, device=gpu_device) for r in range(2)}
    weight = Int8Weight(torch.zeros(80, 96, dtype=torch.bfloat16, device=gpu_device))
    clients = {r: _client(naming, r, connection_timeout=5) for r in range(3)}

    def body(r):
        c = clients[r]
        if r < 2:
            c.init_pair("w", "trainer", "inference", 2, device_mesh=torch.arange(2), placements=(Shard(0),))
            return c.register_tensors("b", [(src[r], "w")])
        c.init_pair("w", "inference", "trainer", 1, device_mesh=torch.arange(1), placements=(Replicate(),))
        return c.register_tensors("b", [(weight, "w")])

    handlers = run_ranks(body, range(3))
    for k in range(2):
        for t in src.values():
            t.mul_(-1.5)
        torch.cuda.synchronize()
        run_ranks(lambda r: handlers[r].transfer("send" if r < 2 else "recv", blocking=True), range(3))
        assert torch.equal(weight.landing, torch.cat([src[0], src[1]]).bfloat16())
        check_int8_rows(weight.landing, weight.values, weight.scales)
    for h in handlers.values():
        h.close()
    for c in clients.values():
        c.close()


def test_an_8_bit_target_is_staged_beside_its_landing():
    job = ReshardJob(specs(), device="cpu")
    assert [sorted(w) for w in job.target_int8] == [[], [], [], [8, 9]]
    weight = job.target_int8[3][9]
    assert weight.landing is job.target_locals[3][9]
    assert weight.values.shape == (OUT // 2, HIDDEN) and weight.values.dtype == torch.int8
    assert weight.scales.shape == (OUT // 2,) and weight.scales.dtype == torch.float32
    with pytest.raises(RuntimeError, match="no CPU path"):
        weight.refresh()
    with pytest.raises(ValueError, match="no channels"):
        Int8Weight(torch.zeros(4))
    with pytest.raises(ValueError, match="element type"):
        Int8Weight(torch.zeros(4, 4, dtype=torch.float64))
    three = Int8Weight(torch.zeros(2, 5, 7).bfloat16())
    assert three.values.shape == (2, 5, 7) and three.scales.shape == (2, 5)


def test_the_bus_takes_the_landing_of_an_8_bit_weight(agent_factory):  # noqa: F811
    agent, naming = agent_factory(2)
    weight = Int8Weight(torch.zeros(8, 4))
    clients = {r: _client(naming, r, connection_timeout=5) for r in range(2)}

    def body(r):
        names = ("trainer", "inference") if r == 0 else ("inference", "trainer")
        clients[r].init_pair("w", *names, 1, device_mesh=np.arange(1), placements=(Replicate(),), timeout=10)
        return clients[r].register_tensors("b", [(torch.ones(8, 4) if r == 0 else weight, "w")], timeout=10)

    handlers = run_ranks(body, range(2))
    assert handlers[0].int8_weights == () and handlers[1].int8_weights == (weight,)
    assert agent.batches["b"].recv_buckets[1][0].chunks[0].tensor.data_ptr() == weight.landing.data_ptr()
    for h in handlers.values():
        h.close()
    for c in clients.values():
        c.close()


def count_refreshes(monkeypatch):
    """Stands in for the conversion, which needs a GPU: notes what the landing held when it was called."""
    seen = []
    monkeypatch.setattr(Int8Weight, "refresh", lambda self: seen.append(self.landing.clone()) or self)
    return seen


@pytest.mark.parametrize("how", ["handler", "client", "handler, not blocking", "client, not blocking"])
def test_every_receive_through_the_bus_converts(agent_factory, monkeypatch, how):  # noqa: F811
    """Whichever call brings the new weights: what it leaves in the landing is converted once, when it is known to be there."""
    seen = count_refreshes(monkeypatch)
    agent, naming = agent_factory(2)
    weight = Int8Weight(torch.zeros(8, 4))
    clients = {r: _client(naming, r, connection_timeout=5) for r in range(2)}

    def body(r):
        names = ("trainer", "inference") if r == 0 else ("inference", "trainer")
        clients[r].init_pair("w", *names, 1, device_mesh=np.arange(1), placements=(Replicate(),), timeout=10)
        return clients[r].register_tensors("b", [(torch.ones(8, 4) if r == 0 else weight, "w")], timeout=10)

    handlers = run_ranks(body, range(2))

    class Done:
        """A command that the agent has finished."""

        def poll(self, timeout):
            return True

        def recv(self):
            return "ok", None

        def close(self):
            pass

    for c in clients.values():
        c.command_queue.enqueue = lambda command: Completion(Done(), "done")
    blocking = "not" not in how
    for k in range(1, 3):
        weight.landing.fill_(k)
        who = handlers[1].transfer if how.startswith("handler") else lambda *a, **kw: clients[1].transfer("b", *a, **kw)
        done = who("recv", blocking=blocking)
        if not blocking:
            assert len(seen) == k - 1
            done.acquire(timeout=5)
            done.acquire(timeout=5)  # once
        assert len(seen) == k and bool((seen[-1] == k).all())
    handlers[0].transfer("send", blocking=True)
    clients[1].transfer("b", "send", blocking=True)
    clients[1].transfer("another batch", "recv", blocking=True)
    assert len(seen) == 2
    for h in handlers.values():
        h.close()
    clients[1].transfer("b", "recv", blocking=True)
    assert len(seen) == 2, "a closed batch keeps no weights"


def test_a_failed_receive_does_not_convert():
    class Failed:
        def poll(self, timeout):
            return True

        def recv(self):
            return "error", ("ValueError", "no such batch")

    done = Completion(Failed(), "failed")
    called = []
    done.then = lambda: called.append(1)
    with pytest.raises(ValueError, match="no such batch"):
        done.acquire()
    done.acquire()
    assert not called


def test_the_halves_of_a_transfer_convert_too(monkeypatch):
    """run_send and run_recv, called apart: the call behind which nothing is waiting any more converts; run() once."""
    seen = count_refreshes(monkeypatch)
    spec = TensorSpec("w", (64, 16), [0, 1], (Shard(0),), [2, 3], (Shard(0),), torch.float32, target_int8=True)
    job = ReshardJob([spec], device="cpu", bucket_size=256, wire=LoopbackWire("cpu", host_inspection=True))
    job.wire.on_launch = lambda *a: None
    job.run_send()
    assert not seen and not job.wire.idle()
    job.run_recv()
    assert len(seen) == 2 and job.wire.idle()  # a target shard each
    del seen[:]
    job.run()
    assert len(seen) == 2
    # both halves queued, the wire stepped by hand: the caller says when
    del seen[:]
    job.run_send(drive=False)
    job.run_recv(drive=False)
    assert not seen and not job.wire.idle()
    job.wire.drive()
    job.refresh_int8()
    assert len(seen) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("pool", ["ring", "resident"])
def test_the_halves_of_a_transfer_bring_new_values(gpu_device, pool):
    spec = TensorSpec("w", (96, 640), [0, 1], (Shard(0),), [2], (Replicate(),), torch.float32, torch.bfloat16, seed=1, target_int8=True)
    job = ReshardJob([spec], device=gpu_device, pool=pool)
    weight = job.target_int8[0][2]
    for _ in range(3):
        for t in job.source_locals[0].values():
            t.mul_(-1.5)
        job.run_send()
        job.run_recv()
        check_int8_rows(weight.landing, weight.values, weight.scales)
        assert torch.equal(weight.landing, torch.cat([job.source_locals[0][r] for r in (0, 1)]).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("blocking", [True, False])
def test_an_8_bit_weight_through_the_clients_own_transfer(gpu_device, agent_factory, blocking):  # noqa: F811
    agent, naming = agent_factory(2, device=gpu_device)
    src = torch.randn(40, 96, device=gpu_device)
    weight = Int8Weight(torch.zeros(40, 96, dtype=torch.bfloat16, device=gpu_device))
    clients = {r: _client(naming, r, connection_timeout=5) for r in range(2)}

    def body(r):
        names = ("trainer", "inference") if r == 0 else ("inference", "trainer")
        clients[r].init_pair("w", *names, 1, device_mesh=np.arange(1), placements=(Replicate(),))
        return clients[r].register_tensors("b", [(src if r == 0 else weight, "w")])

    handlers = run_ranks(body, range(2))
    for _ in range(2):
        src.mul_(-1.5)
        torch.cuda.synchronize()
        done = run_ranks(lambda r: clients[r].transfer("b", "send" if r == 0 else "recv", blocking=blocking), range(2))
        if not blocking:
            for c in done.values():
                c.acquire(timeout=30)
        assert torch.equal(weight.landing, src.bfloat16())
        check_int8_rows(weight.landing, weight.values, weight.scales)
    for h in handlers.values():
        h.close()
    for c in clients.values():
        c.close()


def test_another_job_on_the_wire_does_not_hold_up_the_conversion(monkeypatch):
    seen = count_refreshes(monkeypatch)
    wire = LoopbackWire("cpu", host_inspection=True)
    wire.on_launch = lambda *a: None
    job, other = (ReshardJob([TensorSpec("w", (64, 16), [n, n + 1], (Shard(0),), [n + 2, n + 3], (Shard(0),), torch.float32, target_int8=n == 0)],
                             device="cpu", bucket_size=256, wire=wire) for n in (0, 4))
    other.run_send()
    job.run_send()
    assert not seen
    job.run_recv()
    assert len(seen) == 2 and not wire.idle()
    other.run_recv()
    assert len(seen) == 2 and wire.idle()


def test_a_handler_converts_the_weights_that_it_was_given(monkeypatch):
    """Also one that was made with them, and not by its client's registration."""
    seen = count_refreshes(monkeypatch)
    weight = Int8Weight(torch.zeros(8, 4))

    class Client:
        _int8_weights = {}
        agent_rank = 0
        _transfer = TensorBusClient._transfer
        _execute_command_with_semaphore = TensorBusClient._execute_command_with_semaphore

        class command_queue:
            @staticmethod
            def enqueue(command):
                class Done:
                    poll = staticmethod(lambda timeout: True)
                    recv = staticmethod(lambda: ("ok", None))
                    close = staticmethod(lambda: None)

                return Completion(Done(), "done")

    client = Client()
    handler = BatchHandler(client, "b", ["w"], (weight,))
    handler.transfer("send", blocking=True)
    assert not seen
    handler.transfer("recv", blocking=True)
    assert len(seen) == 1

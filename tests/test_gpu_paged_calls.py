"""Calls over paged caches that a program may make and the other tests do not: the way back as a recorded call, steps without a new token, every call on a stream of
the program's, a plan run op by op, gates and outputs in one tensor."""
import numpy as np
import pytest
import torch

from gpu_common import host, saetta
from paged_common import DIM, tables as plain_tables
from test_gpu_paged import BF16, F16, F32, Batch, compare_tables, ints, plain_state, poison, values_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_the_way_back_recorded(dtype, graph):
    """Slots and codes are read when the plan runs; rows without a slot stay."""
    gen = np.random.default_rng(1)
    cache = saetta.PagedCache(2, DIM, 6, 32)
    slots = ints([5 * 32 + i for i in range(32)] + [-1] + [32 + i for i in range(7)])
    keys, values, alone = (torch.full((50, 2, DIM), 7.25, dtype=dtype, device="cuda") for _ in range(3))
    plan = saetta.Plan()
    cache.record_dequantize(plan, slots, keys, values)
    cache.record_dequantize(plan, slots, None, alone)
    built = plan.build(graph=graph)
    for step in range(3):
        poison(cache, gen)
        k, v = values_of(gen, 40, 2, F16), values_of(gen, 40, 2, F16)
        if step == 2:
            slots.copy_(torch.cat([slots[20:], slots[:20]]))
        order = host(slots).tolist()
        cache.encode(k, v, ints(sorted(order, key=lambda s: (s < 0, s))))
        for t in (keys, values, alone):
            t.fill_(7.25)
        built.run()
        want = [torch.full((50, 2, DIM), 7.25, dtype=dtype, device="cuda") for _ in range(2)]
        cache.encode_dequantize(slots, *want)
        assert torch.equal(keys, want[0]) and torch.equal(values, want[1]) and torch.equal(alone, want[1])
        hole = order.index(-1)
        assert bool((keys[hole] == 7.25).all()) and bool((keys[40:] == 7.25).all()) and not bool((keys[:hole] == 7.25).all())


@pytest.mark.parametrize("rows", [1, 4, 100])
@pytest.mark.parametrize("requests, room", [(3, 7), (3, 3000), (300, 9), (1100, 2100)])
def test_a_step_without_a_token(rows, requests, room):
    """Nothing new of any request: tables and outputs stay, and the step after it is as if it had not been.  (The split took what its registers held for a tile.)"""
    t = saetta.PagedTables(requests, room, 6, 12, 16)
    cache, attention = saetta.PagedCache(2, DIM, 12, 16), saetta.PagedAttention(16, 2, DIM, t, rows=rows)
    q, out = torch.randn(room, 16, DIM, device="cuda").half(), torch.full((room, 16, DIM), 7.25, dtype=F16, device="cuda")
    k = torch.randn(room, 2, DIM, device="cuda")
    context = np.zeros(requests, int)
    for some in ((), (0, 1), (), (1, requests - 1), ()):
        new = np.isin(np.arange(requests), some).astype(int)
        state = plain_state(t)
        t.encode(ints(context), ints(new))
        compare_tables(t, state, plain_tables(state, context, new, 16, room), room)
        cache.encode(k, k, t.slots)
        out.fill_(7.25)
        attention.encode_split(t)
        attention.encode(q, cache, t, out)
        assert host(attention.split)[:8].view(np.int32).tolist() == [len(some), 0]
        assert bool((out[len(some):] == 7.25).all()) and not bool((out[:len(some)] == 7.25).any())
        context = context + new


def test_every_call_on_another_stream():
    results = []
    for stream in (None, torch.cuda.Stream()):
        torch.manual_seed(5)
        t = saetta.PagedTables(2, 40, 6, 9, 16)
        cache, attention = saetta.PagedCache(2, DIM, 9, 16), saetta.PagedAttention(16, 2, DIM, t, rows=30)
        context, new = ints([0, 0]), ints([30, 9])
        x, out = torch.randn(40, 20, DIM, device="cuda").half(), torch.zeros(40, 16, DIM, dtype=F16, device="cuda")
        back = [torch.zeros(40, 2, DIM, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        t.encode(context, new, stream=stream)
        cache.encode(x[:, 16:18], x[:, 18:], t.slots, stream=stream)
        attention.encode_split(t, stream=stream)
        attention.encode(x[:, :16], cache, t, out, stream=stream)
        cache.encode_dequantize(t.slots, *back, stream=stream)
        torch.cuda.synchronize()
        results.append([out, *back, *t.tensors(), *cache.tensors()])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and float(results[0][0].abs().max()) > 0


def test_a_plan_op_by_op():
    """run_serial and both kinds of built plans give the same bits."""
    b = Batch(71, [300, 20, 0], [2, 40, 1], 16, 16, 2, F16)
    plan = saetta.Plan()
    b.attention.record_split(plan, b.tables)
    b.attention.record(plan, b.q, b.cache, b.tables, b.out, gate=b.gate)
    b.run()
    b.compare()
    first = b.out.clone()
    for run in (plan.run_serial, plan.build().run, plan.build(graph=True).run):
        b.out.fill_(1.0)
        run()
        torch.cuda.synchronize()
        assert torch.equal(b.out, first)


@pytest.mark.parametrize("new", [[1, 2], [60, 3]])
def test_the_output_in_the_place_of_the_gates(new):
    b = Batch(72, [400, 70], new, 32, 16, 2, BF16)
    b.run()
    first = b.out.clone()
    b.out = b.gate
    b.run()
    assert torch.equal(b.out, first)

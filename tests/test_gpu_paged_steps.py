"""Steps over paged caches as a program goes on with them: short of blocks, and what the calls refuse."""
import numpy as np
import pytest
import torch

from gpu_common import host, saetta
from paged_common import DIM, Cache, attend, tables
from test_gpu_paged import F16, compare_tables, ints, numbers, plain_state, poison

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("room", [50, 600, 3001])
def test_a_step_short_of_blocks(room):
    """A recorded step that counts on by itself, with fewer blocks than its tokens want: those without one come again, and nobody sees what another request has left in
    the block that they get."""
    heads, kv_heads, block, blocks, requests = 16, 2, 16, 5, 3
    gen = np.random.default_rng(room)
    t = saetta.PagedTables(requests, room, 4, blocks, block)
    cache, plain = saetta.PagedCache(kv_heads, DIM, blocks, block), Cache(kv_heads, blocks, block)
    poison(cache, gen)
    attention = saetta.PagedAttention(heads, kv_heads, DIM, t, rows=40)
    new = ints([0] * requests)
    x = torch.zeros(room, heads + 2 * kv_heads, DIM, dtype=F16, device="cuda")
    out = torch.zeros(room, heads, DIM, dtype=F16, device="cuda")
    plan = saetta.Plan()
    t.record(plan, t.kv_lens, new)
    cache.record(plan, x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], t.slots)
    attention.record_split(plan, t)
    attention.record(plan, x[:, :heads], cache, t, out)
    built = plan.build(graph=True)
    short = []
    # as many as there are blocks for; more than there are blocks for; one request ends; the others' tokens again, twice; a row of the table is full
    for fresh, ended in [((20, 27, 3), []), ((14, 3, 14), []), ((5, 0, 2), [1]), ((5, 0, 2), []), ((30, 0, 12), []), ((9, 0, 0), [2]), ((9, 0, 0), []), ((20, 0, 0), []),
                         ((5, 0, 0), []), ((1, 4, 0), [0])]:
        for r in ended:
            t.kv_lens[r] = 0
        state = plain_state(t)
        context = np.minimum(host(t.kv_lens), np.array(state["held"]) * block)
        new.copy_(ints(fresh)), out.fill_(7.25)
        n = sum(fresh)
        x[:n] = torch.tensor(gen.standard_normal((n, heads + 2 * kv_heads, DIM)), dtype=F16, device="cuda")
        built.run()
        step = tables(state, context, fresh, block, room)
        compare_tables(t, state, step, room)
        plain.store(numbers(x[:n, heads:heads + kv_heads]), numbers(x[:n, heads + kv_heads:]), step["slots"][:n])
        want, bound = attend(numbers(x[:n, :heads]), plain, state["block_table"], step["query_starts"], step["kv_lens"], None, np.zeros((n, heads, DIM)))
        assert (np.abs(numbers(out)[:n] - want) <= bound * 1.001 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
        short.append(step["unplaced"][0])
    assert [s > 0 for s in short] == [False, True, True, False, True, True, False, True, True, False]


@pytest.mark.parametrize("block", [16, 32, 128])
def test_the_most_tokens_of_a_call(block):
    """Nearly 2^28 of them, all but a few without a slot; their rows are one and the same."""
    tokens, cache = (1 << 28) - 32, saetta.PagedCache(1, DIM, 4, block)
    k = torch.randn(1, 1, DIM, device="cuda")
    slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    there = {5: block, (1 << 27) + 3: 2 * block, tokens - 1: 0}
    for at, slot in there.items():
        slots[at] = slot
    cache.encode(k.expand(tokens, 1, DIM), k.expand(tokens, 1, DIM), slots)
    plain = Cache(1, 4, block)
    plain.store(numbers(k), numbers(k), [0])
    for want, got in zip(plain.gather([0, 0, 0]), Cache.of(cache).gather(list(there.values()))):
        assert np.array_equal(want, got)


def test_more_slots_than_32_bits_count():
    """Refused, by the calls that are made at once and by those that are recorded: 2^32 + 1 slots were taken for one."""
    n, cache = (1 << 32) + 1, saetta.PagedCache(1, DIM, 1, 16)
    slots, k = torch.empty(n, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, DIM, device="cuda").expand(n, 1, DIM)
    for call in (lambda: cache.encode(k, k, slots), lambda: cache.record(saetta.Plan(), k, k, slots)):
        with pytest.raises(ValueError, match="2\\^32"):
            call()

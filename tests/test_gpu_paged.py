"""A cache in blocks that several requests share, on the GPU against the plain statement in 64 bits: tables, store, gather and
attention, at the sizes where each can go wrong, and a step of all of them as a program takes it."""
import math

import numpy as np
import pytest
import torch

from gpu_common import host, saetta
from paged_common import DIM, Cache, attend, tables

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def ints(x):
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")


def numbers(t):
    torch.cuda.synchronize()
    return t.detach().double().cpu().numpy()


# ---- tables ----------------------------------------------------------------------------------------------------------

def compare_tables(t, state, step, room):
    assert host(t.held).tolist() == [int(h) for h in state["held"]]
    assert int(t.free_count) == len(state["free"])
    assert host(t.free_list)[:len(state["free"])].tolist() == state["free"]
    assert np.array_equal(host(t.block_table), state["block_table"])
    for name in ("query_starts", "kv_lens", "slots", "positions", "unplaced"):
        assert host(getattr(t, name)).tolist() == step[name], name


def plain_state(t):
    n = int(t.free_count)
    return {"block_table": host(t.block_table).copy(), "held": host(t.held).tolist(), "free": host(t.free_list)[:n].tolist()}


@pytest.mark.parametrize("requests, block, blocks, width, room, most", [
    (1, 16, 4, 3, 1, 1), (1, 16, 64, 70, 1100, 900), (3, 32, 40, 9, 64, 50), (64, 64, 300, 6, 700, 30), (65, 128, 90, 3, 2049, 60),
    (1023, 16, 4000, 40, 2048, 3), (1024, 16, 3000, 40, 5000, 9), (1025, 32, 1200, 8, 9000, 40), (2300, 16, 5000, 5, 30000, 25),
    (7, 16, 9, 50, 600, 100)])
def test_tables_over_steps(requests, block, blocks, width, room, most):
    """Steps that place tokens, take some back, finish requests and ask for more blocks, tokens and entries than there are."""
    gen = np.random.default_rng(requests)
    t = saetta.PagedTables(requests, room, width, blocks, block)
    t.free_list.copy_(ints(gen.permutation(blocks)))
    state, context = plain_state(t), np.zeros(requests, int)
    for step in range(6):
        new = gen.integers(0, most + 1, requests)
        if step % 2:
            new[gen.random(requests) < 0.5] = 0
        finished = gen.random(requests) < 0.2
        context[finished], new[finished & (step % 3 == 0)] = 0, 0
        context = np.maximum(context - (gen.integers(0, 3, requests) if step == 4 else 0), 0)  # rejected drafts
        t.encode(ints(context), ints(new))
        compare_tables(t, state, tables(state, context, new, block, room), room)
        context = np.minimum(context + new, width * block)


def test_tables_replayed_in_place():
    """A recorded step whose context lengths are what it makes: each replay goes on by the new tokens."""
    t = saetta.PagedTables(5, 12, 9, 30, 16)
    new = ints([1, 2, 0, 4, 3])
    plan = saetta.Plan()
    t.record(plan, t.kv_lens, new)
    built, state, context = plan.build(graph=True), plain_state(t), np.zeros(5, int)
    for _ in range(30):
        built.run()
        compare_tables(t, state, tables(state, context, host(new), 16, 12), 12)
        context = context + host(new)


def test_tables_of_wrong_numbers():
    """Counts and blocks that cannot be lead nowhere outside."""
    t = saetta.PagedTables(4, 40, 3, 6, 16)
    t.free_count.fill_(1000), t.free_list.fill_(77777), t.held.fill_(-5)
    t.encode(ints([10, -3, 2000000000, 5]), ints([5, 9, 2000000000, 5]))
    torch.cuda.synchronize()
    assert (host(t.slots) == -1).all() and 0 <= int(t.free_count) <= 6


def test_tables_without_new_tokens():
    """Requests that only finish: a step with no room for tokens gives their blocks back."""
    import ctypes
    ffi = saetta.ffi
    requests, blocks = 1100, 2500
    t = saetta.PagedTables(requests, 2200, 3, blocks, 16)
    t.encode(ints([0] * requests), ints([20] * requests))
    state = plain_state(t)
    zeros = ints([0] * requests)
    at = [x.data_ptr() for x in t.tensors()]
    p = ffi.PagedTablesParamsC(requests, 3, 16, blocks, 0)
    ffi.check(ffi.lib().saetta_paged_tables(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), zeros.data_ptr(), zeros.data_ptr(),
                                            ffi.PagedStateC(*at[:4]), ffi.PagedStepC(*at[4:]), p), "paged_tables")
    want = tables(state, [0] * requests, [0] * requests, 16, 0)
    assert host(t.free_list).tolist() == state["free"] and host(t.held).tolist() == [0] * requests and (host(t.block_table) == -1).all()
    assert host(t.query_starts).tolist() == want["query_starts"] and int(t.unplaced) == 0


# ---- store and gather --------------------------------------------------------------------------------------------------

def values_of(gen, tokens, kv_heads, dtype):
    x = gen.standard_normal((tokens, kv_heads, DIM)) * np.exp2(gen.uniform(-3, 3, (tokens, kv_heads, 1)))
    x[..., [7, 101, 230]] *= 8.0
    return torch.tensor(x, dtype=dtype, device="cuda")


def poison(cache, gen):
    """What memory may hold that nobody has cleared, NaN codes among it."""
    for name in ("keys", "values", "key_scales", "value_scales"):
        t = getattr(cache, name)
        t.copy_(torch.from_numpy(gen.integers(0, 256, tuple(t.shape), dtype=np.uint8)))
    cache.keys[:, :, ::3] = 0x7f
    cache.values[:, :, ::5] = 0xff


def runs_of(gen, blocks, block, pieces):
    """Slots of runs in blocks of their own, each (offset, tokens); -1 between some."""
    order, slots = gen.permutation(blocks), []
    for b, (at, n) in zip(order, pieces):
        slots += [int(b) * block + at + i for i in range(n)]
        if gen.random() < 0.3:
            slots.append(-1)
    return slots


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("block, kv_heads", [(16, 1), (32, 4), (64, 2), (128, 2)])
def test_store_and_gather(dtype, block, kv_heads):
    gen = np.random.default_rng(block)
    cache = saetta.PagedCache(kv_heads, DIM, 9, block)
    first = [(0, block), (0, 1), (0, 5), (0, block - 1), (0, 3)]
    slots = runs_of(gen, 9, block, first)
    k, v = values_of(gen, len(slots), kv_heads, dtype), values_of(gen, len(slots), kv_heads, dtype)
    cache.encode(k, v, ints(slots))
    want = Cache(kv_heads, 9, block)
    want.store(numbers(k), numbers(v), slots)
    # more tokens behind them, louder and softer, the last of a block alone, and a run over tokens that were taken back
    starts = [s for s in slots if s >= 0 and s % block == 0]
    more = [starts[1] + 1 + i for i in range(block - 1)] + [starts[2] + 5, -1] + [starts[3] + block - 1] + [starts[4] + 1 + i for i in range(7)]
    for loud in (0.1, 30.0, 1e-6):
        k, v = values_of(gen, len(more), kv_heads, F32) * loud, values_of(gen, len(more), kv_heads, F32) * loud
        k, v = k.to(dtype), v.to(dtype)
        cache.encode(k, v, ints(more))
        want.store(numbers(k), numbers(v), more)
    got = Cache.of(cache)
    for w in ("keys", "values"):
        assert np.array_equal(got.e[w], want.e[w])
        assert np.array_equal(got.rows[w], want.rows[w])
    back = [s for s in slots + more if s >= 0] + [starts[0] + 3, starts[0] + 2]
    gen.shuffle(back)
    for out_type in (F32, F16, BF16):
        outs = [torch.empty(len(back), kv_heads, DIM, dtype=out_type, device="cuda") for _ in range(2)]
        cache.encode_dequantize(ints(back), *outs)
        for o, x in zip(outs, want.gather(back)):
            assert torch.equal(o, torch.tensor(x, dtype=out_type, device="cuda"))


def test_store_of_many_short_runs():
    """More tokens than workgroups of their own: runs of one to a few tokens, blocks begun anew and continued, in one call."""
    gen = np.random.default_rng(41)
    cache, want = saetta.PagedCache(2, DIM, 900, 16), Cache(2, 900, 16)
    for call in range(2):
        pieces = []
        for _ in range(700):
            at = 0 if call == 0 else int(gen.integers(0, 16))
            pieces.append((at, int(gen.integers(1, 17 - at))))
        slots = runs_of(gen, 900, 16, pieces)
        assert len(slots) > 1500
        k, v = values_of(gen, len(slots), 2, F16), values_of(gen, len(slots), 2, F16)
        cache.encode(k, v, ints(slots))
        want.store(numbers(k), numbers(v), slots)
    got = Cache.of(cache)
    for w in ("keys", "values"):
        assert np.array_equal(got.e[w], want.e[w]) and np.array_equal(got.rows[w], want.rows[w])


@pytest.mark.parametrize("block, kv_heads, room", [(16, 2, 2100), (32, 1, 700), (64, 2, 1300), (128, 3, 5000)])
def test_store_of_steps_in_a_large_room(block, kv_heads, room):
    """Steps of single tokens, drafts and a few long runs among many places without a slot; scales that rise at every step."""
    gen = np.random.default_rng(block)
    blocks = 40
    cache, plain = saetta.PagedCache(kv_heads, DIM, blocks, block), Cache(kv_heads, blocks, block)
    poison(cache, gen)
    filled = np.zeros(blocks, int)
    for step in range(5):
        slots = []
        for b in gen.permutation(blocks):
            n = int(min(gen.choice([0, 1, 1, 2, 3, 4, 5, 6, block // 2]), block - filled[b]))
            slots += [int(b) * block + int(filled[b]) + i for i in range(n)]
            filled[b] += n
            slots += [-1] * int(gen.integers(0, 3))
        slots = (slots + [-1] * room)[:max(room, len(slots))]
        k, v = (values_of(gen, len(slots), kv_heads, F16) * 2.0 ** step for _ in range(2))
        cache.encode(k, v, ints(slots))
        plain.store(numbers(k), numbers(v), slots)
    there = [b * block + t for b in range(blocks) for t in range(int(filled[b]))]
    for got, want in zip(Cache.of(cache).gather(there), plain.gather(there)):
        assert np.array_equal(got, want)


def test_store_of_no_numbers_and_the_range():
    """Not finite: NaN, and the others' scale is theirs.  Zero, the smallest, the largest, past the range."""
    cache = saetta.PagedCache(1, DIM, 2, 16)
    k = torch.zeros(8, 1, DIM, device="cuda")
    k[0, 0, 3], k[1, 0, 200], k[2, 0, 0] = float("nan"), float("inf"), float("-inf")
    k[3] = torch.linspace(-448, 448, DIM, device="cuda")
    k[4, 0, :3] = torch.tensor([2.0 ** -10, 2.0 ** -10 * 1.001, -2.0 ** -9], device="cuda")  # a tie to zero, and what is past it
    slots = list(range(8))
    cache.encode(k, -k, ints(slots))
    want = Cache(1, 2, 16)
    want.store(numbers(k), -numbers(k), slots)
    got = Cache.of(cache)
    assert np.array_equal(got.rows["keys"], want.rows["keys"], equal_nan=True) and got.e["keys"][0, 0] == 0
    assert np.array_equal(got.rows["values"], want.rows["values"], equal_nan=True)
    for top, e in ((0.0, -40), (1e-30, -40), (448 * 2.0 ** 60, 60), (449 * 2.0 ** 60, 60), (3e38, 60)):
        k = torch.full((1, 1, DIM), top, device="cuda")
        cache.encode(k, k, ints([16]))
        want.store(numbers(k), numbers(k), [16])
        got = Cache.of(cache)
        assert got.e["keys"][1, 0] == e == want.e["keys"][1, 0]
        assert np.array_equal(got.rows["keys"][1, 0, 0], want.rows["keys"][1, 0, 0], equal_nan=True)


def test_store_from_strided_rows_into_what_was_never_cleared():
    gen = np.random.default_rng(3)
    cache = saetta.PagedCache(2, DIM, 5, 64)
    poison(cache, gen)
    both = values_of(gen, 40, 2 * 3, F16)  # q, k and v of a projection side by side
    k, v = both[:, 2:4], both.transpose(0, 1)[4:6].transpose(0, 1)
    slots = [3 * 64 + i for i in range(30)] + [64 + i for i in range(10)]
    cache.encode(k, v, ints(slots))
    want = Cache(2, 5, 64)
    want.store(numbers(k), numbers(v), slots)
    got = Cache.of(cache)
    for w in ("keys", "values"):
        assert np.array_equal(got.rows[w][3, :, :30], want.rows[w][3, :, :30])
        assert np.array_equal(got.rows[w][1, :, :10], want.rows[w][1, :, :10])


def test_slots_that_do_not_exist():
    gen = np.random.default_rng(4)
    cache = saetta.PagedCache(2, DIM, 3, 32)
    k = values_of(gen, 5, 2, F32)
    before = [t.clone() for t in cache.tensors()]
    slots = ints([-1, 3 * 32, 2 ** 31 - 1, -2 ** 31, 3 * 32 + 1])
    cache.encode(k, k, slots)
    assert all(torch.equal(a, b) for a, b in zip(before, cache.tensors()))
    outs = [torch.full((5, 2, DIM), 7.5, device="cuda") for _ in range(2)]
    cache.encode_dequantize(slots, *outs)
    assert all(bool((o == 7.5).all()) for o in outs)
    cache.encode_dequantize(ints([0] * 5), outs[0], None)  # keys alone, one slot again and again
    assert bool((outs[0] == 0).all()) and bool((outs[1] == 7.5).all())


def test_a_call_without_tokens():
    cache, none = saetta.PagedCache(2, DIM, 3, 32), torch.zeros(0, 2, DIM, device="cuda")
    cache.encode(none, none, ints([]))
    cache.encode_dequantize(ints([]), none, none)


# ---- attention -----------------------------------------------------------------------------------------------------------

class Batch:
    """Requests with `context` tokens in their blocks and `new` ones, whose keys and values are there too."""

    def __init__(self, seed, context, new, block, heads, kv_heads, dtype, gate=True, room=0, garbage=True):
        self.gen = gen = np.random.default_rng(seed)
        lengths = [c + n for c, n in zip(context, new)]
        counts = [-(-n // block) for n in lengths]
        blocks, width = sum(counts) + 2, max(counts + [1]) + 1
        self.cache = saetta.PagedCache(kv_heads, DIM, blocks, block)
        if garbage:
            poison(self.cache, gen)
        tokens = sum(new)
        self.tables = t = saetta.PagedTables(len(new), max(tokens + room, 1), width, blocks, block)
        order, at, slots = gen.permutation(blocks), 0, []
        for r, n in enumerate(counts):
            t.block_table[r, :n] = ints(order[at:at + n])
            slots += [int(order[at + p // block]) * block + p % block for p in range(lengths[r])]
            at += n
        t.kv_lens.copy_(ints(lengths)), t.query_starts.copy_(ints(np.concatenate([[0], np.cumsum(new)])))
        if slots:
            # (a request's keys a few tokens at a time, as a conversation brings them, would raise scales; here at once)
            k, v = values_of(gen, len(slots), kv_heads, F16), values_of(gen, len(slots), kv_heads, F16)
            self.cache.encode(k, v, ints(slots))
        self.slots = slots
        self.both = torch.tensor(gen.standard_normal((max(tokens + room, 1), heads, 2 * DIM)), dtype=dtype, device="cuda")
        self.q, self.gate = self.both[..., :DIM], self.both[..., DIM:] if gate else None
        self.out = torch.full((max(tokens + room, 1), heads, DIM), 7.25, dtype=dtype, device="cuda")
        self.attention = saetta.PagedAttention(heads, kv_heads, DIM, t, rows=max(list(new) + [1]))

    def run(self):
        self.attention.encode_split(self.tables)
        self.attention.encode(self.q, self.cache, self.tables, self.out, gate=self.gate)

    def want(self):
        out = np.full(tuple(self.out.shape), 7.25)
        t = self.tables
        return attend(numbers(self.q), Cache.of(self.cache), host(t.block_table), host(t.query_starts), host(t.kv_lens),
                      None if self.gate is None else numbers(self.gate), out)

    def compare(self):
        got, (want, bound) = numbers(self.out), self.want()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        half = HALF_STEP[self.out.dtype]
        off = np.abs(got - want) - (bound * (1 + half) + half * np.abs(want) + 2.0 ** -25)
        assert np.nanmax(off, initial=-1.0) <= 0, (np.nanmax(off), np.unravel_index(np.nanargmax(off), off.shape))


FEW = [
    # context, new, block, heads, kv heads
    ([0], [1], 16, 16, 2), ([1], [1], 16, 16, 2), ([15], [1], 16, 8, 1), ([16], [1], 16, 32, 4), ([31, 32, 33], [1, 1, 1], 32, 16, 2),
    ([127, 128, 129, 500], [1, 1, 1, 1], 64, 16, 2), ([700, 3, 90], [2, 1, 2], 128, 16, 2), ([200, 40], [16, 9], 16, 2, 2),
    ([333, 20], [8, 3], 32, 4, 2), ([100, 301], [1, 1], 64, 32, 2), ([50, 77], [3, 4], 16, 4, 1), ([900, 0, 4], [0, 2, 0], 64, 16, 2)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("context, new, block, heads, kv_heads", FEW)
def test_few_rows(context, new, block, heads, kv_heads, dtype):
    b = Batch(len(context) + block, context, new, block, heads, kv_heads, dtype, gate=block != 64, room=2)
    b.run()
    b.compare()


CHUNKS = [
    ([0], [3], 16, 16, 2), ([0], [33], 16, 16, 2), ([5], [40], 32, 16, 2), ([0, 90, 1], [31, 70, 3], 64, 16, 2), ([300], [17], 128, 8, 1),
    ([17], [260], 16, 1, 1), ([40, 2], [20, 5], 64, 32, 2), ([64], [130], 32, 4, 2), ([513, 0, 60, 7], [9, 0, 1, 33], 64, 16, 2),
    ([31], [64], 16, 8, 4)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("context, new, block, heads, kv_heads", CHUNKS)
def test_chunks(context, new, block, heads, kv_heads, dtype):
    b = Batch(len(context) + block, context, new, block, heads, kv_heads, dtype, gate=block != 64, room=5)
    b.run()
    b.compare()


@pytest.mark.parametrize("new, block", [(1, 16), (2, 128), (7, 32)])
def test_keys_in_parts(new, block):
    """Keys enough for many parts, a last part of few, and more units than a workgroup looks up at a time; random scales."""
    b = Batch(new, [20011, 130], [new, new], block, 16, 2, F16)
    b.run()
    b.compare()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads, kv_heads", [(16, 2), (4, 4), (16, 1)])
def test_a_few_rows_beside_a_chunk(heads, kv_heads, dtype):
    """Requests of every width of a tile of few rows, short and long, whole and in parts, in the step of a chunk."""
    new = [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 65, 90]
    b = Batch(18, [2600, 0, 1, 900, 31, 1700, 2, 0, 450, 7, 100, 33, 70], new, 32, heads, kv_heads, dtype, room=3)
    b.run()
    b.compare()


def test_no_numbers_beside_a_chunk():
    """NaN among the values and keys of drafts and of a prompt's last tokens: rows that see it are NaN, the others are not touched."""
    b = Batch(19, [700, 40, 64, 500], [3, 2, 70, 1], 16, 16, 2, F16)
    block = host(b.tables.block_table)
    for request, at in ((0, 701), (1, 41), (2, 130), (3, 3)):  # token t of its block, dim 5
        t = at % 16
        b.cache.values[int(block[request, at // 16]), 1, (t // 4 * 16 + 5) * 16 + t % 4] = 0x7f
    b.run()
    b.compare()
    got = numbers(b.out)
    assert np.isnan(got[:, 8:, 5]).sum() == 8 * (2 + 1 + 4 + 1) and not np.isnan(got[:, :8]).any()


@pytest.mark.parametrize("new", [[20], [9, 40]])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_chunk_in_many_parts(new, dtype):
    """One tile, and a few, whose keys are as many parts as the device has workgroups for."""
    b = Batch(24, [5001, 1003][:len(new)], new, 64, 8, 1, dtype, room=1)
    b.run()
    b.compare()


def test_scales_that_differ_widely():
    """Neighbouring blocks 2^20 apart, keys and values; a block of zeros."""
    for new in (1, 5):
        b = Batch(9, [400, 70], [new, new], 16, 16, 2, BF16)
        gen = np.random.default_rng(5)
        loud = np.repeat(np.exp2(gen.integers(-14, 7, len(b.slots) // 16 + 1)), 16)[:len(b.slots), None, None]
        loud[32:48] = 0.0
        k, v = gen.standard_normal((2, len(b.slots), 2, DIM)) * loud
        b.cache.encode(torch.tensor(np.clip(k, -4, 4), dtype=F32, device="cuda"), torch.tensor(v, dtype=F32, device="cuda"), ints(b.slots))
        b.run()
        b.compare()


def test_many_small_weights_beside_a_large_one():
    """20000 keys whose weights are subnormal in f16 beside one of weight 1: together they are half of the output."""
    for new in (1, 9):
        b = Batch(31, [20000], [new], 64, 16, 2, F16, gate=False)
        b.q.zero_(), b.q[..., 0].fill_(16.0)
        n = len(b.slots)
        k, v = torch.zeros(n, 2, DIM, device="cuda"), torch.ones(n, 2, DIM, device="cuda")
        k[777, :, 0], v[777] = 10.0, -1.0  # a score of 10 above the others': 4.5e-5 of weight each, 0.9 of the largest together
        b.cache.encode(k, v, ints(b.slots))
        b.run()
        b.compare()


@pytest.mark.parametrize("new", [2, 40])
def test_no_numbers_in_places_that_some_rows_do_not_see(new):
    """NaN keys and values of new tokens reach the rows that see them, in the dims that have them, and no others."""
    b = Batch(11, [100, 3], [new, new], 32, 16, 2, F16)
    k, v = numbers_in = [torch.randn(new, 2, DIM, device="cuda") for _ in range(2)]
    del numbers_in
    v[new // 2, 1, 17], v[new - 1, 0, 200] = float("nan"), float("inf")
    last = b.slots[100 + new - new:100 + new]
    b.cache.encode(k, v, ints(last))
    b.run()
    b.compare()
    got = numbers(b.out)
    assert np.isnan(got[new - 1, 8:, 17]).all() and not np.isnan(got[:new // 2]).any()
    k[new - 1, 0, 5] = float("nan")
    b.cache.encode(k, v, ints(last))
    b.run()
    b.compare()
    assert np.isnan(numbers(b.out)[new - 1, :8]).all()


@pytest.mark.parametrize("new", [1, 30])
def test_blocks_that_are_not_there(new):
    """Missing blocks and numbers of blocks that do not exist are not seen; a row that sees nothing is zeros; padding rows stay."""
    b = Batch(12, [200, 40, 16], [new, new, new], 16, 16, 2, F16, room=3)
    t = b.tables
    t.block_table[0, 3], t.block_table[0, 5], t.block_table[0, 6] = -1, b.cache.blocks, 2 ** 31 - 1
    t.block_table[2] = -1
    b.run()
    b.compare()
    got = numbers(b.out)
    assert (got[2 * new:3 * new] == 0).all() and (got[3 * new:] == 7.25).all()
    t.kv_lens[1] = 0  # a request that is not there any more, its rows still counted
    t.kv_lens[0] = 2 ** 31 - 1  # past a row of the table
    b.run()
    torch.cuda.synchronize()
    assert (numbers(b.out)[new:2 * new] == 0).all()


def test_order_of_heads_and_tokens():
    """q, gate and out as views of other orders: heads outermost, every other token, into the place of q."""
    b = Batch(13, [90, 33], [1, 1], 32, 16, 2, F16)
    heads_first = torch.empty(16, 2, 2 * DIM, dtype=F16, device="cuda")
    heads_first.copy_(b.both.transpose(0, 1))
    b.q, b.gate = heads_first.transpose(0, 1)[..., :DIM], heads_first.transpose(0, 1)[..., DIM:]
    wide = torch.full((4, 16, DIM), 7.25, dtype=F16, device="cuda")
    b.out = wide[::2]
    b.run()
    b.compare()
    assert bool((wide[1::2] == 7.25).all())
    first = b.out.clone()
    b.out = b.q
    b.run()
    assert torch.equal(b.out, first)


def test_same_bits_every_time_and_on_another_stream():
    b = Batch(14, [5000, 200, 31], [2, 1, 2], 64, 16, 2, BF16)
    b.run()
    torch.cuda.synchronize()
    first = b.out.clone()
    side = torch.cuda.Stream()
    for _ in range(3):
        b.out.fill_(1.0)
        side.wait_stream(torch.cuda.current_stream())
        b.attention.encode_split(b.tables, stream=side)
        b.attention.encode(b.q, b.cache, b.tables, b.out, gate=b.gate, stream=side)
        side.synchronize()
        assert torch.equal(b.out, first)


def test_two_calls_at_once():
    """Two objects on two streams share nothing but the cache."""
    one, two = Batch(15, [3000, 8], [1, 1], 64, 16, 2, F16), Batch(16, [700, 20], [40, 3], 32, 16, 2, F16)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for b, s in zip((one, two), streams):
            b.attention.encode_split(b.tables, stream=s)
            b.attention.encode(b.q, b.cache, b.tables, b.out, gate=b.gate, stream=s)
    torch.cuda.synchronize()
    one.compare(), two.compare()


def test_chunks_same_bits_every_time_and_in_the_place_of_q():
    """Prompts in parts beside drafts: which workgroup takes what differs from call to call, the bits do not."""
    b = Batch(20, [6000, 10, 900, 0, 2500], [100, 3, 7, 200, 1], 32, 16, 2, F16)
    b.run()
    b.compare()
    first = b.out.clone()
    for _ in range(4):
        b.out.fill_(1.0)
        b.run()
        assert torch.equal(b.out, first)
    b.out = b.q
    b.run()
    assert torch.equal(b.out, first)


@pytest.mark.parametrize("chunk", [0, 70])
def test_more_requests_than_a_workgroup_has_threads(chunk):
    """Tables, split and attention of 1500 requests (and one with a chunk): their rounds."""
    gen = np.random.default_rng(22)
    context, new = gen.integers(0, 40, 1500).tolist(), gen.integers(0, 3, 1500).tolist()
    if chunk:
        new[1100] = chunk
    b = Batch(22, context, new, 16, 2, 1, F16, room=2)
    b.run()
    b.compare()
    starts, lens = b.tables.query_starts.clone(), b.tables.kv_lens.clone()
    t = saetta.PagedTables(1500, sum(new) + 2, b.tables.max_blocks, 6000, 16)
    state = plain_state(t)
    t.encode(ints(context), ints(new))
    compare_tables(t, state, tables(state, context, new, 16, sum(new) + 2), sum(new) + 2)
    assert torch.equal(t.query_starts, starts) and torch.equal(t.kv_lens, lens)


@pytest.mark.parametrize("new", [1, 40])
def test_blocks_that_requests_share(new):
    """Three requests behind one prefix: their tables name the same blocks."""
    b = Batch(23, [96, 96, 96, 5], [new, new, new, 1], 32, 16, 2, BF16)
    t = b.tables
    t.block_table[1, :3], t.block_table[2, :3] = t.block_table[0, :3], t.block_table[0, :3]
    b.run()
    b.compare()


def test_python_objects_refuse_on_the_gpu():
    b = Batch(17, [9], [1], 16, 16, 2, F16)
    other = saetta.PagedTables(2, 1, 2, 4, 16)
    with pytest.raises(ValueError):
        b.attention.encode_split(other)
    for q, out, gate, error in ((b.q.float(), b.out, None, TypeError), (b.q, b.out.bfloat16(), None, ValueError), (b.q[:, :8], b.out, None, ValueError),
                                (b.q, b.out, b.gate[:0], ValueError), (b.q, b.out[:, :1].expand(1, 16, DIM), None, ValueError),
                                (b.both[..., 1:DIM + 1], b.out, None, saetta.ffi.SaettaError)):
        with pytest.raises(error):
            b.attention.encode(q, b.cache, b.tables, out, gate=gate)
    with pytest.raises(ValueError):
        b.attention.encode(b.q, saetta.PagedCache(2, DIM, 4, 32), b.tables, b.out)
    k = torch.zeros(2, 2, DIM, device="cuda")
    for args, error in (((k, k.half(), ints([0, 1])), ValueError), ((k, k, ints([0])), ValueError), ((k.double(), k.double(), ints([0, 1])), TypeError),
                        ((k, k, torch.zeros(2, dtype=torch.int64, device="cuda")), TypeError), ((k[:, :1], k[:, :1], ints([0, 1])), ValueError)):
        with pytest.raises(error):
            b.cache.encode(*args)
    with pytest.raises(ValueError):
        b.cache.encode_dequantize(ints([0, 1]), torch.zeros(1, 2, DIM, device="cuda"), None)


# ---- together ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("graph", [False, True])
def test_steps_of_a_program(graph):
    """Tables, two layers' stores and attention, recorded once: a step with prompts, then tokens and drafts, some rejected."""
    heads, kv_heads, block, requests, room = 16, 2, 16, 4, 48
    gen = np.random.default_rng(21)
    t = saetta.PagedTables(requests, room, 20, 60, block)
    caches = [saetta.PagedCache(kv_heads, DIM, 60, block) for _ in range(2)]
    for c in caches:
        poison(c, gen)
    context, new = ints([0] * requests), ints([0] * requests)
    qkv = torch.zeros(2, room, heads + 2 * kv_heads, DIM, dtype=F16, device="cuda")
    out = torch.zeros(2, room, heads, DIM, dtype=F16, device="cuda")
    attention = saetta.PagedAttention(heads, kv_heads, DIM, t, rows=40)
    plan = saetta.Plan()
    t.record(plan, context, new)
    attention.record_split(plan, t)
    for x, c, o in zip(qkv, caches, out):
        c.record(plan, x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], t.slots)
        attention.record(plan, x[:, :heads], c, t, o)
    built = plan.build(graph=graph)
    wants = [Cache(kv_heads, 60, block) for _ in range(2)]
    lengths = np.zeros(requests, int)
    for step, fresh in enumerate([(17, 0, 31, 0), (1, 5, 1, 3), (4, 4, 4, 4), (1, 1, 1, 1), (0, 40, 1, 1), (1, 1, 0, 0), (3, 0, 2, 16)]):
        if step == 3:
            lengths -= np.array([3, 1, 0, 4])  # rejected
        if step == 5:
            lengths[2] = 0  # finished
        x = torch.tensor(gen.standard_normal(tuple(qkv.shape)), dtype=F16, device="cuda")
        qkv.copy_(x), context.copy_(ints(lengths)), new.copy_(ints(fresh)), out.fill_(7.25)
        built.run()
        slots = host(t.slots).tolist()
        for i in range(2):
            wants[i].store(numbers(x[i, :, heads:heads + kv_heads]), numbers(x[i, :, heads + kv_heads:]), slots)
            seen = Cache.of(caches[i])
            want, bound = attend(numbers(x[i, :, :heads]), wants[i], host(t.block_table), host(t.query_starts), host(t.kv_lens), None,
                                 np.full((room, heads, DIM), 7.25))
            got = numbers(out[i])
            assert np.array_equal(got[sum(fresh):], want[sum(fresh):])
            assert (np.abs(got - want) <= bound * 1.001 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
            used = [s for s in slots if s >= 0]
            for a, b in zip(seen.gather(used), wants[i].gather(used)):
                assert np.array_equal(a, b)
        lengths += np.array(fresh)
    assert math.isclose(float(t.unplaced[0]), 0.0)


@pytest.mark.parametrize("room, fresh", [(20, (12, 12, 3)), (4, (1, 2, 9)), (3, (1, 1, 1, 1, 1))])
def test_a_step_past_its_room(room, fresh):
    """More new tokens than the step has room for: those that have room are at their own positions, and the next step goes on behind them."""
    heads, kv_heads, block, requests = 16, 2, 16, len(fresh)
    gen = np.random.default_rng(33)
    t = saetta.PagedTables(requests, room, 4, 20, block)
    cache, plain = saetta.PagedCache(kv_heads, DIM, 20, block), Cache(kv_heads, 20, block)
    poison(cache, gen)
    attention = saetta.PagedAttention(heads, kv_heads, DIM, t, rows=max(fresh))
    left = list(fresh)
    for _ in range(2):
        state, context = plain_state(t), host(t.kv_lens).tolist()
        step = tables(state, context, left, block, room)
        t.encode(t.kv_lens, ints(left))
        compare_tables(t, state, step, room)
        x = torch.tensor(gen.standard_normal((room, heads + 2 * kv_heads, DIM)), dtype=F16, device="cuda")
        out = torch.full((room, heads, DIM), 7.25, dtype=F16, device="cuda")
        cache.encode(x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], t.slots)
        attention.encode_split(t)
        attention.encode(x[:, :heads], cache, t, out)
        plain.store(numbers(x[:, heads:heads + kv_heads]), numbers(x[:, heads + kv_heads:]), step["slots"])
        want, bound = attend(numbers(x[:, :heads]), plain, state["block_table"], step["query_starts"], step["kv_lens"], None,
                             np.full((room, heads, DIM), 7.25))
        assert (np.abs(numbers(out) - want) <= bound * 1.001 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
        left = [n - (after - before) for n, after, before in zip(left, step["kv_lens"], context)]
    assert sum(fresh) - sum(left) == min(sum(fresh), 2 * room)


def test_starts_that_go_back():
    """First tokens that do not rise name more tiles than a step can have: as many as it can are dealt out, no row is outside."""
    requests, room = 2000, 600
    t = saetta.PagedTables(requests, room, 2, 4, 16)
    cache, attention = saetta.PagedCache(2, DIM, 4, 16), saetta.PagedAttention(16, 2, DIM, t, rows=40)
    t.query_starts.copy_(ints([0, 0xfffff] * (requests // 2) + [0])), t.kv_lens.fill_(700)
    q = torch.zeros(room, 16, DIM, dtype=F16, device="cuda")
    whole = torch.full((room + 8, 16, DIM), 7.25, dtype=F16, device="cuda")
    attention.encode_split(t)
    attention.encode(q, cache, t, whole[:room])
    torch.cuda.synchronize()
    assert int(attention.split[:4].view(torch.int32)) <= attention.split.numel() // 32 and bool((whole[room:] == 7.25).all())


def test_a_cache_of_more_than_four_gigabytes():
    """Blocks whose codes lie past 2^32 bytes: stored, read back and attended over."""
    blocks, block = 70000, 128  # 4.6 GB of keys, as many of values
    cache = saetta.PagedCache(2, DIM, blocks, block)
    gen = np.random.default_rng(51)
    order = [blocks - 1, 3, blocks - 2, 65536, 65535, 0]
    for new in (1, 20):
        t = saetta.PagedTables(1, new, 8, blocks, block)
        length = 5 * block + 40 + new
        t.block_table[0, :6] = ints(order)
        t.kv_lens.fill_(length), t.query_starts.copy_(ints([0, new]))
        slots = [order[p // block] * block + p % block for p in range(length)]
        k, v = values_of(gen, length, 2, F16), values_of(gen, length, 2, F16)
        cache.encode(k, v, ints(slots))
        small = saetta.PagedCache(2, DIM, 6, block)  # the same in a cache of six blocks
        near = [(p // block) * block + p % block for p in range(length)]
        small.encode(k, v, ints(near))
        outs = [torch.empty(2, length, 2, DIM, device="cuda") for _ in range(2)]
        cache.encode_dequantize(ints(slots), *outs[0]), small.encode_dequantize(ints(near), *outs[1])
        assert torch.equal(outs[0], outs[1])
        q = torch.randn(new, 16, DIM, dtype=F16, device="cuda")
        got, want = torch.zeros_like(q), torch.zeros_like(q)
        attention = saetta.PagedAttention(16, 2, DIM, t, rows=new)
        attention.encode_split(t)
        attention.encode(q, cache, t, got)
        t.block_table[0, :6] = ints(range(6))
        attention.encode(q, small, t, want)
        assert torch.equal(got, want) and float(want.abs().max()) > 0


def test_calls_captured_by_torch():
    """The calls as they are, under torch's own capture, replayed over other lengths with eager work between."""
    b = Batch(61, [150, 40, 3], [2, 1, 2], 16, 16, 2, F16)
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    for lengths in ([152, 41, 5], [100, 41, 4], [17, 2, 2], [152, 41, 5]):
        b.tables.kv_lens.copy_(ints(lengths))
        b.out.fill_(7.25)
        graph.replay()
        b.compare()
        first = b.out.clone()
        b.run()
        assert torch.equal(b.out, first)


def test_a_split_of_another_call_leads_nowhere_outside():
    """Attention by a split that was made for other rows: what it says is followed only as far as the buffers go."""
    b = Batch(62, [70, 40], [1, 1], 16, 16, 2, F16)
    other = saetta.PagedAttention(16, 2, DIM, b.tables, rows=30)
    other.encode_split(b.tables)
    n = min(other.split.numel(), b.attention.split.numel())
    b.attention.split[:n].copy_(other.split[:n])
    b.attention.encode(b.q, b.cache, b.tables, b.out, gate=b.gate)
    b.attention.split.fill_(0x5a)
    b.attention.encode(b.q, b.cache, b.tables, b.out, gate=b.gate)
    torch.cuda.synchronize()
    b.run()
    b.compare()

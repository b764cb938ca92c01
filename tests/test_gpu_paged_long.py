"""Items of many keys: the attention kernels past what a wave, or a workgroup, looks up of a table at a time.  Requests whose tables name the same blocks fill the
device, so that their keys stay whole or in a few parts; the split is looked at, so that a test whose items have become short fails."""
import numpy as np
import pytest
import torch

from gpu_common import host, saetta
from paged_common import DIM, Cache
from test_gpu_paged import BF16, F16, HALF_STEP, ints, numbers, poison, values_of

pytestmark = pytest.mark.gpu
GROUP = 8


class Long:
    """`requests` of `new` tokens behind about n keys of one kv head each, blocks in any order, some of them missing late in the walk."""

    def __init__(self, seed, requests, new, n, block, dtype=F16, rows=None):
        self.gen = gen = np.random.default_rng(seed)
        blocks = -(-n // block)
        self.new, self.cache = new, saetta.PagedCache(1, DIM, blocks + 1, block)
        poison(self.cache, gen)
        order = gen.permutation(blocks + 1)[:blocks]
        slots = [int(order[p // block]) * block + p % block for p in range(n)]
        k, v = values_of(gen, n, 1, F16), values_of(gen, n, 1, F16)
        self.cache.encode(k, v, ints(slots))
        self.tables = t = saetta.PagedTables(requests, requests * new, blocks, blocks + 1, block)
        table = np.tile(order, (requests, 1))
        for r in range(0, requests, 3):  # a hole: of every third request
            table[r, int(gen.integers(blocks // 2, blocks))] = -1
        t.block_table.copy_(torch.from_numpy(table.astype(np.int32)))
        self.lengths = np.array([max(n - r % 37, new) for r in range(requests)])
        t.kv_lens.copy_(ints(self.lengths)), t.query_starts.copy_(ints(range(0, requests * new + 1, new)))
        self.q = torch.randn(requests * new, GROUP, DIM, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)
        self.out = torch.zeros_like(self.q)
        self.attention = saetta.PagedAttention(GROUP, 1, DIM, t, rows=rows or new)

    def run(self):
        """The items as (keys from, to, tokens, parts)."""
        self.attention.encode_split(self.tables)
        self.attention.encode(self.q, self.cache, self.tables, self.out)
        words = host(self.attention.split).view(np.int32)
        items = words[4:4 + 8 * words[0]].reshape(-1, 8)
        return items[:, [4, 5, 2, 7]]

    def compare(self, requests):
        """Rows of some requests, with the bound of test_gpu_paged_weights (values of ordinary sizes: a weight is off by 2^-11 of it or 2^-32 of the largest)."""
        c, q, got, table = Cache.of(self.cache), numbers(self.q), numbers(self.out), host(self.tables.block_table)
        half = HALF_STEP[self.out.dtype]
        for r in requests:
            at = np.arange(self.lengths[r])
            block = table[r][at // c.block_tokens]
            k, v = c.rows["keys"][block, 0, at % c.block_tokens], c.rows["values"][block, 0, at % c.block_tokens]
            for i in sorted({0, self.new // 2, self.new - 1}):
                row = r * self.new + i
                seen = (at <= self.lengths[r] - self.new + i) & (block >= 0)
                s = np.where(seen, q[row] @ k.T / 16.0, -np.inf)
                p = np.exp(s - s.max(axis=1, keepdims=True))
                p /= p.sum(axis=1, keepdims=True)
                seen_k, seen_v = np.where(seen[:, None], np.abs(k), 0.0), np.where(seen[:, None], np.abs(v), 0.0)
                spread = (np.abs(q[row]) @ seen_k.T).max(axis=1) / 16.0
                rel = 2.0 ** -11 + 2.0 ** -23 * (264 * spread + 4 * np.abs(s[:, seen]).max(axis=1) + seen.sum() / 16 + 32)
                want, bound = p @ np.where(seen[:, None], v, 0.0), rel[:, None] * (p @ seen_v) + 2.0 ** -32 * p.max(axis=1)[:, None] * seen_v.sum(axis=0)
                off = np.abs(got[row] - want) - (bound * (1 + half) + half * np.abs(want) + 2.0 ** -25)
                assert off.max() <= 0, (r, i, off.max(), np.unravel_index(off.argmax(), off.shape))


def steps_of(items):
    """Steps of 32 keys (two units of 16, from the item's first)."""
    return -(-(-(-items[:, 1] // 16) - items[:, 0] // 16) // 2)


@pytest.mark.parametrize("steps", [27, 28, 31, 32, 33, 64, 127, 128, 129, 160, 256, 257, 300, 520])
@pytest.mark.parametrize("block, dtype", [(16, F16), (64, BF16)])
def test_chunk_items_of_many_steps(steps, block, dtype):
    """Whole items, around every count at which a wave takes the places of its next 32 steps, fills a window of 512 units, and fills half of it again."""
    new, n = 40, 32 * steps - 5
    b = Long(steps, 300, new, n, block, dtype)
    items = b.run()
    chunks = items[items[:, 2] * GROUP > 64]
    assert (chunks[:, 3] == 1).all() and (chunks[:, 0] == 0).all()  # of the first request one tile ends at n - 8, of others up to 36 earlier
    assert steps - 2 <= steps_of(chunks).max() <= steps
    b.compare([0, 1, 36, 299])


@pytest.mark.parametrize("block", [16, 128])
def test_chunk_items_in_parts_of_many_steps(block):
    """The same in two parts, of which the second begins at a key that is not the window's first."""
    b = Long(7, 90, 40, 20000, block)
    items = b.run()
    late = items[(items[:, 2] * GROUP > 64) & (items[:, 0] > 0)]
    assert steps_of(late).max() > 256 and (late[:, 3] > 1).all() and (late[:, 0] % 1024 != 0).any()
    b.compare([0, 1, 50, 89])


@pytest.mark.parametrize("block, dtype", [(16, F16), (64, BF16), (128, F16)])
@pytest.mark.parametrize("new, requests", [(1, 600), (1, 300), (2, 600), (3, 300), (3, 150), (5, 300), (8, 150)])
def test_few_rows_of_many_keys(new, requests, block, dtype):
    """Waves that look their places up more than once (4096 keys at a time of four waves), in whole items and in parts."""
    b = Long(new + requests, requests, new, 20000, block, dtype)
    items = b.run()
    whole = requests > (512 if new * GROUP <= 16 else 256)
    assert (items[:, 1] - items[:, 0]).max() > (16384 if whole else 8192)
    assert (items[:, 3] == 1).all() if whole else items[:, 0].max() > 0
    b.compare([0, 1, 35, requests - 1])


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("new, requests", [(1, 400), (2, 200), (4, 400), (4, 150), (7, 400), (7, 150)])
def test_few_rows_beside_chunks_of_many_keys(new, requests, block):
    """The same by the kernel for chunks, whose eight waves look up 8192 keys at a time."""
    b = Long(new * requests, requests, new, 30000, block, rows=100)
    items = b.run()
    assert (items[:, 1] - items[:, 0]).max() > 8192 + 1024
    if requests < 256:
        assert items[:, 0].max() > 0
    b.compare([0, 1, 35, requests - 1])

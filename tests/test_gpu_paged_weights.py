"""The weights of the attention over paged caches where f16 holds them least well: a great many small ones beside a large one, values of every
exponent that a block can have, and blocks whose exponents lie far apart.  Against the formula in 64 bits over what the cache holds."""
import numpy as np
import pytest
import torch

from gpu_common import host, saetta
from paged_common import DIM, Cache
from test_gpu_paged import BF16, F16, F32, HALF_STEP, ints, numbers

pytestmark = pytest.mark.gpu


class One:
    """One request of one kv head, its blocks in order: keys and values [tokens, 256], queries [new, heads, 256]."""

    def __init__(self, keys, values, queries, dtype, block=16, kv_heads=1):
        tokens, new, heads = len(keys), len(queries), queries.shape[1]
        blocks = -(-tokens // block)
        self.cache = saetta.PagedCache(kv_heads, DIM, blocks, block)
        self.tables = t = saetta.PagedTables(1, new, blocks, blocks, block)
        t.block_table[0] = ints(range(blocks))
        t.kv_lens.fill_(tokens), t.query_starts.copy_(ints([0, new]))
        k, v = (torch.tensor(x, dtype=F32, device="cuda")[:, None].expand(tokens, kv_heads, DIM) for x in (keys, values))
        self.cache.encode(k, v, ints(range(tokens)))
        self.q = torch.tensor(queries, dtype=dtype, device="cuda")
        self.out = torch.zeros(new, heads, DIM, dtype=dtype, device="cuda")
        self.attention = saetta.PagedAttention(heads, kv_heads, DIM, t, rows=new)

    def run(self):
        self.attention.encode_split(self.tables)
        self.attention.encode(self.q, self.cache, self.tables, self.out)

    def compare(self, rows=(0, -1)):
        """The first head of every kv head, of the rows given.  A weight w = p 2^rest, in units of its largest W in the row, is rounded to f16 by 2^-11 of it or
        2^-32 of W; a score is off as `attend` has it, by (256 + 4) 2^-24 sum |q k| / 16 and 4 2^-24 of itself, in numerator and denominator; sums
        of n keys by (n / 16 + 32) 2^-24, 2^-23 for both; then the output's own half step (and half of its least step)."""
        c, q, got = Cache.of(self.cache), numbers(self.q), numbers(self.out)
        group, half = q.shape[1] // c.kv_heads, HALF_STEP[self.out.dtype]
        least = 2.0 ** -25 if self.out.dtype is F16 else 2.0 ** -134
        for i in rows:
            seen = int(self.tables.kv_lens[0]) - len(q) + 1 + i % len(q)
            at = np.arange(seen)
            block, t = host(self.tables.block_table)[0][at // c.block_tokens], at % c.block_tokens
            for h in range(c.kv_heads):
                k, v = c.rows["keys"][block, h, t], c.rows["values"][block, h, t]
                s = k @ q[i, h * group] / 16.0
                p = np.exp(s - s.max())
                p /= p.sum()
                e = c.e["values"][block, h].astype(float)
                rest = e - np.clip(e, -15, 7)
                w = p * np.exp2(rest - rest.max())  # (times 2^rest.max())
                small = (2.0 ** -32 * w.max() * np.exp2(rest.max() - rest)) @ np.abs(v)
                spread = np.abs(k) @ np.abs(q[i, h * group]) / 16.0
                rel = 2.0 ** -11 + 2.0 ** -23 * (264 * spread.max() + 4 * np.abs(s).max() + seen / 16 + 32)
                want = p @ v
                bound = rel * (p @ np.abs(v)) + small
                off = np.abs(got[i, h * group] - want) - (bound * (1 + half) + half * np.abs(want) + least)
                assert off.max() <= 0, (i, h, off.max(), int(off.argmax()), got[i, h * group][off.argmax()], want[off.argmax()], bound[off.argmax()])


# rows of a tile: a token; two, three and five tokens of 8 q heads; a chunk, whose last row is compared (and its first)
ROWS = [1, 2, 3, 5, 40]


@pytest.mark.parametrize("new", [1, 3, 5, 9])
def test_many_small_weights_behind_a_large_one(new):
    """400 thousand keys whose weights are 2^-25.06 of the first one's, 1.1 % of a row together, by one workgroup from end to end: 600 requests whose tables name the
    same blocks, so that no request's keys are taken in parts.  With two kinds of keys the row follows from two numbers.  Bound: weights by 2^-11 of them, or 2^-32 of
    the largest; sums in f32 of n / 16 products' results at most, and n / 32 sums of weights, 2^-24 each (of a wave: of few rows a quarter of the keys, 32 at once);
    the output's half step."""
    n, requests = 400000, 600
    blocks = n // 128
    cache = saetta.PagedCache(1, DIM, blocks, 128)
    t = saetta.PagedTables(requests, requests * new, blocks, blocks, 128)
    t.block_table.copy_(ints(range(blocks)).expand(requests, blocks))
    t.kv_lens.fill_(n), t.query_starts.copy_(ints(range(0, requests * new + 1, new)))
    k, v = torch.zeros(n, 1, DIM, dtype=F16, device="cuda"), torch.full((n, 1, DIM), -1.0, dtype=F16, device="cuda")
    k[0, 0, 0], v[0] = 18.0, 1.0
    cache.encode(k, v, ints(range(n)))
    q = torch.zeros(requests * new, 8, DIM, dtype=F16, device="cuda")
    q[..., 0] = 15.4375
    out = torch.zeros_like(q)
    attention = saetta.PagedAttention(8, 1, DIM, t, rows=new)
    attention.encode_split(t)
    attention.encode(q, cache, t, out)
    assert int(attention.split[:4].view(torch.int32)) == requests
    got = numbers(out).reshape(requests, new, -1)
    for i in range(new):
        others = n - new + i
        small = np.exp(-18.0 * 15.4375 / 16.0)
        want = (1.0 - others * small) / (1.0 + others * small)
        sums = n / 16 + n / 32 if new * 8 > 64 else n / 128 + n / 128
        bound = 2.0 ** -11 + others * 2.0 ** -32 + 2.0 ** -24 * (sums + 64) + 2.0 ** -23 * 16 * 18
        assert np.abs(got[:, i] - want).max() <= bound + 2.0 ** -11, (i, np.abs(got[:, i] - want).max(), bound)


@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("loud", [-45, -38, -26, -23, -22, -15, -8, 0, 7, 8, 20, 50])
def test_values_of_every_exponent(new, loud):
    """Values of sizes over all that e4m3 holds, subnormals too, at loudnesses on both sides of what the conversion to f16 takes of an exponent."""
    gen = np.random.default_rng(new + 100)
    keys, queries = gen.standard_normal((300, DIM)), gen.standard_normal((new, 8, DIM))
    values = gen.standard_normal((300, DIM)) * np.exp2(gen.uniform(-16, 0, (300, DIM))) * 2.0 ** loud
    b = One(keys, values, queries, BF16)
    b.run()
    b.compare()


@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("gap", [16, 24, 28, 34, 39])
@pytest.mark.parametrize("first", [False, True])
def test_a_loud_dim_in_one_block(new, gap, first):
    """One value of 1 in a block, all others 2^-gap, and 8.7 powers of two of score in favour of the quiet blocks: they are the output of every other dim."""
    gen = np.random.default_rng(gap)
    keys, values = np.zeros((128, DIM)), gen.uniform(0.5, 1.0, (128, DIM)) * 2.0 ** -gap
    at = 3 if first else 100
    quiet = np.arange(128) // 16 != at // 16
    keys[quiet, 0], values[at, 9] = 6.0, 1.0  # exp(6) is 2^8.66
    queries = np.zeros((new, 8, DIM))
    queries[..., 0] = 16.0
    b = One(keys, values, queries, BF16)
    b.run()
    b.compare()


@pytest.mark.parametrize("new, rows_of", [(1, 8), (2, 8), (1, 16), (16, 1)])
@pytest.mark.parametrize("beside", [False, True])
def test_weights_of_up_to_16_rows_keep_22_bits(new, rows_of, beside):
    """Three keys whose values nearly cancel in some dims: a weight off by 2^-12 of it would be seen there, 2^-22 is not.  By themselves and beside a chunk.  Scores are
    single products; the exponential is off by 2^-23 of it, and so are the few sums."""
    gen = np.random.default_rng(new * rows_of)
    keys = np.zeros((2 + new, DIM))
    keys[:3, 0] = [1.0, 0.875, 0.75]
    values = gen.uniform(0.25, 1.0, (2 + new, DIM)) * gen.choice([-1.0, 1.0], (2 + new, DIM))
    queries = np.zeros((new, rows_of, DIM))
    queries[..., 0] = gen.uniform(2, 30, (new, rows_of))
    b = One(keys, values, queries, F16)
    if beside:  # another request, of no keys that count, whose tokens are a chunk's
        t = saetta.PagedTables(2, new + 130, b.tables.max_blocks, b.cache.blocks, 16)
        t.block_table[0] = b.tables.block_table[0]
        t.kv_lens.copy_(ints([2 + new, 130])), t.query_starts.copy_(ints([0, new, new + 130]))
        b.tables, q = t, b.q
        b.q = torch.cat([q, torch.ones(130, rows_of, DIM, dtype=F16, device="cuda")])
        b.out = torch.zeros_like(b.q)
        b.attention = saetta.PagedAttention(rows_of, 1, DIM, t, rows=130)
    b.run()
    c, q, got = Cache.of(b.cache), numbers(b.q), numbers(b.out)
    for i in range(new):
        k, v = (c.rows[w][:, 0].reshape(-1, DIM)[:3 + i] for w in ("keys", "values"))
        for h in range(rows_of):
            s = k @ q[i, h] / 16.0
            p = np.exp(s - s.max())
            p /= p.sum()
            want, size = p @ v, p @ np.abs(v)
            rel = 2.0 ** -22 + 2.0 ** -23 * (4 + 8 * np.abs(s).max() + len(s))
            off = np.abs(got[i, h] - want) - (rel * size * (1 + 2.0 ** -11) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25)
            assert off.max() <= 0, (i, h, off.max(), int(off.argmax()))

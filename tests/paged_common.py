"""A cache in blocks, stated plainly: codes, scales, tables and attention in 64 bits, on the CPU."""
import math

import numpy as np

DIM, LOW, HIGH = 256, -40, 60
E4M3 = np.array([math.nan if c & 127 == 127 else (-1.0) ** (c >> 7) * (math.ldexp(8 + (c & 7), (c >> 3 & 15) - 10) if c >> 3 & 15
                                                                      else math.ldexp(c & 7, -9)) for c in range(256)])


def key_byte(t, d):
    return d // 64 * 1024 + (d // 16 % 4 * 16 + t) * 16 + d % 16


def value_byte(t, d):
    return d // 64 * 1024 + (t // 4 * 16 + d % 16) * 16 + d // 16 % 4 * 4 + t % 4


def places(block_tokens, byte):
    """[block_tokens, 256]: where the code of a token's dim lies in a block."""
    t, d = np.arange(block_tokens)[:, None], np.arange(DIM)[None, :]
    return t // 16 * 4096 + byte(t % 16, d)


def nearest(x):
    """x rounded to what e4m3 holds; past 448 and no numbers: NaN."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        _, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
        step = np.ldexp(1.0, np.maximum(e - 4, -9))
        r = np.rint(x / step) * step
        return np.where(np.abs(x) <= 448.0, r, np.nan)


def exponent(amax):
    """The least e of LOW..HIGH with amax <= 448 * 2^e."""
    e = LOW
    while e < HIGH and amax > math.ldexp(448.0, e):
        e += 1
    return e


class Cache:
    """Values [blocks][kv_heads][block_tokens][256] as the codes stand for them, with the exponents."""

    def __init__(self, kv_heads, blocks, block_tokens):
        self.kv_heads, self.blocks, self.block_tokens = kv_heads, blocks, block_tokens
        self.rows = {w: np.zeros((blocks, kv_heads, block_tokens, DIM)) for w in ("keys", "values")}
        self.e = {w: np.full((blocks, kv_heads), LOW) for w in ("keys", "values")}

    @classmethod
    def of(cls, cache):
        """What a PagedCache holds."""
        self = cls(cache.kv_heads, cache.blocks, cache.block_tokens)
        for w, byte in (("keys", key_byte), ("values", value_byte)):
            codes = getattr(cache, w).cpu().numpy()
            self.e[w] = getattr(cache, w[:-1] + "_scales").cpu().numpy().astype(int) - 127
            self.rows[w] = E4M3[codes[:, :, places(self.block_tokens, byte)]] * np.ldexp(1.0, self.e[w])[..., None, None]
        return self

    def store(self, k, v, slots):
        """Runs of slots of one block, one after the other."""
        runs, i, bt = [], 0, self.block_tokens
        while i < len(slots):
            n = 1
            while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] // bt == slots[i] // bt:
                n += 1
            if 0 <= slots[i] < self.blocks * bt:
                runs.append((i, n))
            i += n
        for i, n in runs:
            block, at = divmod(int(slots[i]), bt)
            for w, x in (("keys", k), ("values", v)):
                for h in range(self.kv_heads):
                    new = np.asarray(x[i:i + n, h], np.float64)
                    size = np.abs(new[np.isfinite(new)])
                    e = exponent(size.max() if size.size else 0.0)
                    if at > 0:
                        e = max(e, int(np.clip(self.e[w][block, h], LOW, HIGH)))
                    rows = self.rows[w][block, h]
                    rows[:at] = nearest(np.ldexp(rows[:at], -e)) * math.ldexp(1.0, e)
                    rows[at:at + n] = nearest(np.ldexp(new, -e)) * math.ldexp(1.0, e)
                    # (the codes behind stay, so what they stand for moves with the scale)
                    rows[at + n:] = np.ldexp(rows[at + n:], e - self.e[w][block, h])
                    self.e[w][block, h] = e

    def gather(self, slots):
        block, at = np.asarray(slots) // self.block_tokens, np.asarray(slots) % self.block_tokens
        return self.rows["keys"][block, :, at], self.rows["values"][block, :, at]


def attend(q, cache, table, query_starts, kv_lens, gate, out, scale=1.0 / 16.0):
    """q [tokens][heads][256] in 64 bits; rows of `out` that belong to a request are replaced.  Blocks that do not exist are
    not seen.  What comes back bounds how far sums in f32 over weights in f16 may be from it, before the last rounding:
      a weight is rounded by 2^-11 of itself, or by 2^-25 of the largest where it is subnormal,
      a score is off by (256 + 4) 2^-24 sum |q k| scale and 4 2^-24 of itself, which is a relative error of its weight in numerator and
      denominator, and the sums over n keys by n 2^-24 (tiles of 16 and 32 add up apart: n / 16 + 32 is enough)."""
    heads, group = q.shape[1], q.shape[1] // cache.kv_heads
    bt, bound = cache.block_tokens, np.zeros(out.shape)
    for r in range(len(kv_lens)):
        first, n, length = int(query_starts[r]), int(query_starts[r + 1] - query_starts[r]), int(kv_lens[r])
        for i in range(n):
            at = length - n + i
            t = np.arange(max(min(at + 1, table.shape[1] * bt), 0))
            block = table[r][t // bt]
            t, block = t[(block >= 0) & (block < cache.blocks)], block[(block >= 0) & (block < cache.blocks)]
            if len(t) == 0:
                out[first + i] = 0.0
                continue
            k, v = cache.rows["keys"][block, :, t % bt], cache.rows["values"][block, :, t % bt]
            for h in range(heads):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k[:, h // group] @ q[first + i, h] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    o, size = p @ v[:, h // group], p @ np.abs(v[:, h // group])
                    spread = np.abs(k[:, h // group]) @ np.abs(q[first + i, h]) * scale
                    g = 1.0 if gate is None else 1.0 / (1.0 + np.exp(-gate[first + i, h]))
                    rel = 2.0 ** -11 + 2.0 ** -23 * (264 * spread.max() + 4 * np.abs(s).max() + len(t) / 16 + 32)
                    out[first + i, h] = o * g
                    bound[first + i, h] = g * (rel * size + len(t) * 2.0 ** -25 * np.abs(v[:, h // group]).max() * p.max()) + 2.0 ** -20 * np.abs(o * g)
    return out, bound


def tables(state, context, new, block_tokens, tokens):
    """A step: state is a dict of block_table, held, free (the list's used part).  What the step is given.  New tokens past the room
    (`tokens`) are no part of it."""
    asked, before = sum(int(n) for n in new), 0
    cut = []
    for n in new:
        cut.append(min(int(n), max(tokens - before, 0)))
        before += int(n)
    new = cut
    width = state["block_table"].shape[1]
    free, slots, positions, starts, kv_lens = state["free"], [], [], [0], []
    want = [min(-(-(int(c) + int(n)) // block_tokens), width) for c, n in zip(context, new)]
    takes = [max(0, w - h) for w, h in zip(want, state["held"])]
    taken = min(sum(takes), len(free))
    segment, at = free[len(free) - taken:], 0
    free = free[:len(free) - taken]
    for r, n in enumerate(takes):
        got = segment[at:at + n]
        state["block_table"][r, state["held"][r]:state["held"][r] + len(got)] = got
        state["held"][r] += len(got)
        at += len(got)
    for r, w in enumerate(want):
        if state["held"][r] > w:
            free = free + [int(b) for b in state["block_table"][r, w:state["held"][r]]]
            state["block_table"][r, w:state["held"][r]] = -1
            state["held"][r] = w
    state["free"] = free
    unplaced = asked - sum(new)
    for r, (c, n) in enumerate(zip(context, new)):
        for p in range(int(c), int(c) + int(n)):
            has = p // block_tokens < state["held"][r]
            slot = int(state["block_table"][r, p // block_tokens]) * block_tokens + p % block_tokens if has else -1
            slots.append(slot), positions.append(p)
            unplaced += slot < 0
        starts.append(starts[-1] + int(n)), kv_lens.append(int(c) + int(n))
    behind = [-1] * (tokens - len(slots))
    return {"slots": slots + behind, "positions": positions + behind, "query_starts": starts, "kv_lens": kv_lens, "unplaced": [unplaced]}

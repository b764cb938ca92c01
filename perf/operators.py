"""The operators of a cache in blocks that several requests share, as cases that can be timed and compared.

A program that serves several conversations at once keeps their keys and values in blocks of 16 to 128 tokens.  A
block holds 8-bit floating point codes (e4m3) with one power of two per block and kv head, for keys and for values.
The sizes are those of the model the kernels are written for (16 q heads, 2 kv heads, head dim 256) and other head
layouts of the same kind.  A case names one kind of work:

  tables     block tables, slots and positions of a step, from the requests' lengths: the last draft's rejected
             tokens are given back, the next tokens are placed
  store      new keys and values into their blocks, and the blocks read back as the values they stand for
  gather     keys and values of many slots read back, as for a prefix that another program gets
  attention  a step's attention: of single tokens, of a few drafted ones, of chunks of prompts, or mixed

Layout of a block of one kv head, 256 bytes a token, in units of 16 tokens (4096 bytes each).  Keys: the byte of token
t, dim d of a unit is at d / 64 * 1024 + (d / 16 % 4 * 16 + t) * 16 + d % 16.  Values: at
d / 64 * 1024 + (t / 4 * 16 + d % 16) * 16 + d / 16 % 4 * 4 + t % 4.
"""
import importlib
import math
import random
import types

import torch

own = False

DIM, LOWEST, HIGHEST = 256, -40, 60      # the scales' exponents
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OUTLIERS = [7, 101, 230]                 # 1 % of the channels are larger, as in real layers
MOST_PAIRS = 4096 * (28672 + 4097 / 2) * 16     # (query, key) pairs times heads of the largest listed case
MOST_KEYS = 8 * 131072 * 2               # tokens times kv heads of the longest caches


def listed():
    return [
        # a draft of 4 tokens for each of 32 conversations
        {"name": "tables-draft4-32", "kind": "tables", "requests": 32, "new_low": 4, "new_high": 4, "context_low": 500,
         "context_high": 32000, "lens_seed": 1, "block": 64},
        # 512 requests admitted at once, prompts of all lengths, small blocks
        {"name": "tables-admit-512", "kind": "tables", "requests": 512, "new_low": 1, "new_high": 1900, "context_low": 0,
         "context_high": 0, "lens_seed": 2, "block": 16},
        # the new token's keys and values of 64 conversations
        {"name": "store-token-64", "kind": "store", "requests": 64, "new_low": 1, "new_high": 1, "context_low": 100,
         "context_high": 9000, "lens_seed": 3, "block": 64, "kv_heads": 2, "type": "f16"},
        # five prompts' chunks, as f32 from the norms and rotations before
        {"name": "store-chunks-f32", "kind": "store", "requests": 5, "new_low": 700, "new_high": 3500, "context_low": 0,
         "context_high": 9000, "lens_seed": 4, "block": 16, "kv_heads": 2, "type": "f32"},
        # a long shared prefix handed out as halves
        {"name": "gather-32k-f16", "kind": "gather", "requests": 1, "new_low": 0, "new_high": 0, "context_low": 32768,
         "context_high": 32768, "lens_seed": 5, "block": 64, "kv_heads": 2, "type": "f16"},
        # what 37 short conversations hold, another head layout
        {"name": "gather-ragged-bf16", "kind": "gather", "requests": 37, "new_low": 0, "new_high": 0, "context_low": 1,
         "context_high": 900, "lens_seed": 6, "block": 32, "kv_heads": 4, "type": "bf16"},
        # one conversation that has just begun: nothing but latency and launches
        {"name": "token-1-at-517", "kind": "attention", "requests": 1, "new_low": 1, "new_high": 1, "context_low": 517,
         "context_high": 517, "lens_seed": 7, "block": 64, "heads": 16, "kv_heads": 2, "type": "f16", "layers": 4,
         "gate": True, "chunk": 0, "chunk_at": 0},
        # a batch of conversations of all lengths
        {"name": "token-48-ragged", "kind": "attention", "requests": 48, "new_low": 1, "new_high": 1, "context_low": 300,
         "context_high": 30000, "lens_seed": 8, "block": 32, "heads": 16, "kv_heads": 2, "type": "bf16", "layers": 4,
         "gate": True, "chunk": 0, "chunk_at": 0},
        # few long contexts
        {"name": "token-8-at-131k", "kind": "attention", "requests": 8, "new_low": 1, "new_high": 1, "context_low": 131071,
         "context_high": 131071, "lens_seed": 9, "block": 128, "heads": 16, "kv_heads": 2, "type": "f16", "layers": 1,
         "gate": True, "chunk": 0, "chunk_at": 0},
        # first prompts of odd lengths, taken together
        {"name": "prompts-7-ragged", "kind": "attention", "requests": 7, "new_low": 90, "new_high": 1900, "context_low": 0,
         "context_high": 0, "lens_seed": 10, "block": 16, "heads": 16, "kv_heads": 2, "type": "f16", "layers": 1,
         "gate": True, "chunk": 0, "chunk_at": 0},
        # a chunk of a long prompt
        {"name": "chunk-4096-at-28k", "kind": "attention", "requests": 0, "new_low": 0, "new_high": 0, "context_low": 0,
         "context_high": 0, "lens_seed": 11, "block": 64, "heads": 16, "kv_heads": 2, "type": "bf16", "layers": 1,
         "gate": False, "chunk": 4096, "chunk_at": 28672},
        # a chunk of one prompt beside the verify steps and single tokens of 30 conversations
        {"name": "mixed-1500-and-30", "kind": "attention", "requests": 30, "new_low": 1, "new_high": 5, "context_low": 200,
         "context_high": 20000, "lens_seed": 12, "block": 64, "heads": 16, "kv_heads": 2, "type": "f16", "layers": 2,
         "gate": True, "chunk": 1500, "chunk_at": 8200},
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over its logarithm where that spans more than a factor of ten."""
    if high <= 10 * max(low, 1):
        return rng.randint(low, high)
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["tables", "store", "gather", "token", "token", "verify", "prompts", "chunk", "mixed"])
    case = {"kind": kind, "lens_seed": rng.randrange(1 << 20), "block": rng.choice([16, 32, 64, 128])}
    if kind == "tables":
        fresh = rng.random() < 0.5
        requests = _between(rng, 1, 512)
        high = _between(rng, 1, 250000 // requests) if fresh else rng.randint(1, 8)
        context = 0 if fresh else _between(rng, 100, 32000)
        return {**case, "requests": requests, "new_low": 1, "new_high": high, "context_low": context // 8, "context_high": context}
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (8, 1), (32, 4), (16, 4), (8, 8), (32, 2)])
    type_ = rng.choice(["f16", "bf16"])
    if kind in ("store", "gather"):
        case.update(kv_heads=kv_heads, type=rng.choice(["f32", "f16", "bf16"]))
        if kind == "gather":
            requests = _between(rng, 1, 64)
            longest = _between(rng, 1, 32768 * 2 // (requests * kv_heads))
            return {**case, "requests": requests, "new_low": 0, "new_high": 0, "context_low": 1, "context_high": longest}
        requests = _between(rng, 1, 128)
        longest = _between(rng, 1, max(1, 8192 * 2 // (requests * kv_heads)))
        return {**case, "requests": requests, "new_low": 1, "new_high": longest, "context_low": 0,
                "context_high": _between(rng, 10, 9000)}
    case.update(kind="attention", heads=heads, kv_heads=kv_heads, type=type_, gate=rng.random() < 0.7, chunk=0, chunk_at=0,
                layers=1, context_low=0, context_high=0, requests=0, new_low=0, new_high=0)
    if kind in ("token", "verify"):
        requests = _between(rng, 1, 128)
        longest = _between(rng, 10, min(131072, MOST_KEYS // (2 * kv_heads * requests)))
        new = 1 if kind == "token" else rng.randint(2, 8)
        return {**case, "requests": requests, "new_low": 1, "new_high": new, "context_low": longest // 20,
                "context_high": longest, "layers": rng.randint(1, 4) if requests * longest * kv_heads < MOST_KEYS // 8 else 1}
    if kind == "prompts":
        requests = _between(rng, 1, 16)
        longest = _between(rng, 10, min(4000, int(math.sqrt(MOST_PAIRS / 8 / (heads * requests)))))
        return {**case, "requests": requests, "new_low": max(1, longest // 20), "new_high": longest}
    chunk = _between(rng, 9, 4096)
    at = _between(rng, 1, min(60000, int(MOST_PAIRS / 2 / (heads * chunk))))
    case.update(chunk=chunk, chunk_at=at)
    if kind == "mixed":
        case.update(requests=_between(rng, 1, 40), new_low=1, new_high=rng.randint(1, 8), context_low=10,
                    context_high=_between(rng, 100, 20000))
    return case


def _lengths(case):
    """Tokens that each request has in its cache, and its new ones."""
    rng = random.Random(case["lens_seed"])
    context = [_between(rng, case["context_low"], case["context_high"]) for _ in range(case["requests"])]
    new = [_between(rng, case["new_low"], case["new_high"]) for _ in range(case["requests"])]
    if case.get("chunk"):
        context.append(case["chunk_at"]), new.append(case["chunk"])
    return context, new


class _Maker:
    """Tensors of a seed, made on the GPU."""

    def __init__(self, seed):
        self.generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.generator, device="cuda")

    def kv(self, *shape):
        x = self.normal(*shape, DIM)
        x[..., OUTLIERS] *= 8.0
        return x

    def shuffled(self, n):
        return torch.randperm(n, generator=self.generator, device="cuda").to(torch.int32)


# ---- the cache's form ----------------------------------------------------------------------------------------------

def _power(e):
    """2^e as f32, for e in -126..127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The least e in LOWEST..HIGHEST with amax <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(amax)
    return torch.clamp(torch.where(amax > 0, exponent - 9 + (mantissa > 0.875), LOWEST), LOWEST, HIGHEST)


def _to_codes(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _of_codes(c):
    return c.view(torch.float8_e4m3fn).to(torch.float32)


def _keys_as_rows(c, block):
    """Codes [..., block * 256] of keys, as [..., block, 256]."""
    s = c.shape[:-1]
    n = len(s)
    return c.view(*s, block // 16, 4, 4, 16, 16).permute(*range(n), n, n + 3, n + 1, n + 2, n + 4).reshape(*s, block, DIM)


def _keys_as_codes(r, block):
    s = r.shape[:-2]
    n = len(s)
    return r.reshape(*s, block // 16, 16, 4, 4, 16).permute(*range(n), n, n + 2, n + 3, n + 1, n + 4).reshape(*s, block * DIM)


def _values_as_rows(c, block):
    s = c.shape[:-1]
    n = len(s)
    return c.view(*s, block // 16, 4, 4, 16, 4, 4).permute(*range(n), n, n + 2, n + 5, n + 1, n + 4, n + 3).reshape(*s, block, DIM)


def _values_as_codes(r, block):
    s = r.shape[:-2]
    n = len(s)
    return r.reshape(*s, block // 16, 4, 4, 4, 4, 16).permute(*range(n), n, n + 3, n + 1, n + 5, n + 4, n + 2).reshape(*s, block * DIM)


_ORDER = {"keys": (_keys_as_rows, _keys_as_codes), "values": (_values_as_rows, _values_as_codes)}


def _cache(make, blocks, kv_heads, block):
    """A cache whose blocks are full: what conversations have left there."""
    cache = types.SimpleNamespace(blocks=blocks, kv_heads=kv_heads, block=block)
    for which in ("keys", "values"):
        codes = torch.empty(blocks, kv_heads, block * DIM, dtype=torch.uint8, device="cuda")
        scales = torch.empty(blocks, kv_heads, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 19) // (block * kv_heads))
        for first in range(0, blocks, step):
            x = make.kv(min(step, blocks - first), kv_heads, block)
            e = _exponent(x.abs().amax(dim=(-1, -2)))
            codes[first:first + step] = _ORDER[which][1](_to_codes(x * _power(-e)[..., None, None]), block)
            scales[first:first + step] = (e + 127).to(torch.uint8)
        setattr(cache, which, codes), setattr(cache, which[:-1] + "_scales", scales)
    return cache


def _package():
    return importlib.import_module("saetta-macqwen_amd")


def _own_cache(cache):
    c = _package().PagedCache(cache.kv_heads, DIM, cache.blocks, cache.block)
    for name in ("keys", "values", "key_scales", "value_scales"):
        getattr(c, name).view(-1).copy_(getattr(cache, name).view(-1))
    return c


# ---- preparation ---------------------------------------------------------------------------------------------------

def _tables(make, context, new, block, spare=3):
    """Tables of requests that hold their whole length, in blocks that lie anywhere; slots and positions of the new tokens."""
    counts = [-(-(c + n) // block) for c, n in zip(context, new)]
    blocks = sum(counts) + spare
    order = make.shuffled(blocks)
    width = max(counts + [1]) + 1
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at, slots = 0, []
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n]
        positions = torch.arange(context[r], context[r] + new[r], device="cuda")
        slots.append(table[r][positions // block] * block + (positions % block).to(torch.int32))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    t = types.SimpleNamespace(requests=len(counts), tokens=starts[-1], max_blocks=width, blocks=blocks, block=block,
                              block_table=table, slots=torch.cat(slots))
    t.query_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    t.kv_lens = torch.tensor([c + n for c, n in zip(context, new)], dtype=torch.int32, device="cuda")
    return t


def _own_tables(t):
    o = _package().PagedTables(t.requests, max(t.tokens, 1), t.max_blocks, t.blocks, t.block)
    o.block_table.copy_(t.block_table), o.query_starts.copy_(t.query_starts), o.kv_lens.copy_(t.kv_lens)
    o.slots[:t.tokens].copy_(t.slots)
    return o


def _prepare_tables(case, make):
    context, new = _lengths(case)
    block, requests = case["block"], len(context)
    held = [-(-c // block) for c in context]
    want = [-(-(c + n) // block) for c, n in zip(context, new)]
    blocks, width = sum(want) + 7, max(want) + 2
    order = make.shuffled(blocks)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    at = blocks
    for r, n in enumerate(held):
        table[r, :n] = order[at - n:at]
        at -= n
    free = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
    free[:at] = order[:at]
    state = types.SimpleNamespace(block_table=table, held=torch.tensor(held, dtype=torch.int32, device="cuda"), free_list=free,
                                  free_count=torch.tensor([at], dtype=torch.int32, device="cuda"))
    tokens = sum(new) + 5  # the room for new tokens is a step's most, not what this one has
    ints = {"dtype": torch.int32, "device": "cuda"}
    out = {"context": torch.tensor(context, **ints), "new": torch.tensor(new, **ints), "none": torch.zeros(requests, **ints),
           "block": block, "tokens": tokens, "tables": state}
    if own:
        o = _package().PagedTables(requests, tokens, width, blocks, block)
        for name, value in vars(state).items():
            getattr(o, name).copy_(value)
        out["tables"] = o
    return out


def _prepare_store(case, make):
    context, new = _lengths(case)
    block, kv_heads, type_ = case["block"], case["kv_heads"], TYPES[case["type"]]
    t = _tables(make, context, new, block)
    cache = _cache(make, t.blocks, kv_heads, block)
    # every block that the new tokens touch, from its first token to the last one stored
    back = []
    for r, (c, n) in enumerate(zip(context, new)):
        positions = torch.arange(c // block * block, c + n, device="cuda") if n else torch.arange(0, device="cuda")
        back.append(t.block_table[r][positions // block] * block + (positions % block).to(torch.int32))
    # larger values than those that the blocks hold come now and then
    louder = 1.0 + 3.0 * (make.normal(t.tokens, 1, 1) > 1.5)
    state = {"cache": _own_cache(cache) if own else cache, "slots": t.slots, "back": torch.cat(back),
             "k": (make.kv(t.tokens, kv_heads) * louder).to(type_), "v": (make.kv(t.tokens, kv_heads) * louder).to(type_)}
    shape = (state["back"].numel(), kv_heads, DIM)
    state["out"] = {n: torch.zeros(shape, device="cuda") for n in ("keys", "values")}
    return state


def _prepare_gather(case, make):
    context, _ = _lengths(case)
    block, kv_heads = case["block"], case["kv_heads"]
    t = _tables(make, [0] * len(context), context, block)
    cache = _cache(make, t.blocks, kv_heads, block)
    shape = (t.tokens, kv_heads, DIM)
    return {"cache": _own_cache(cache) if own else cache, "slots": t.slots,
            "out": {n: torch.zeros(shape, dtype=TYPES[case["type"]], device="cuda") for n in ("keys", "values")}}


def _prepare_attention(case, make):
    context, new = _lengths(case)
    heads, kv_heads, type_, layers = case["heads"], case["kv_heads"], TYPES[case["type"]], case["layers"]
    t = _tables(make, context, new, case["block"])
    caches = [_cache(make, t.blocks, kv_heads, case["block"]) for _ in range(layers)]
    # a projection that gives queries and gates side by side: both are views of it
    both = make.normal(layers, t.tokens, heads, 2 * DIM)
    state = {"context": context, "new": new, "heads": heads, "kv_heads": kv_heads, "both": both.to(type_), "gate": case["gate"],
             "out": torch.zeros(layers, t.tokens, heads, DIM, dtype=type_, device="cuda"), "tables": t, "caches": caches}
    if own:
        state["tables"], state["caches"] = _own_tables(t), [_own_cache(c) for c in caches]
        state["attention"] = _package().PagedAttention(heads, kv_heads, DIM, state["tables"], rows=max(new))
    return state


def prepare(case, seed):
    make = _Maker(seed)
    state = {"tables": _prepare_tables, "store": _prepare_store, "gather": _prepare_gather,
             "attention": _prepare_attention}[case["kind"]](case, make)
    state["kind"] = case["kind"]
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _plain_tables(t, context, new, block, tokens):
    requests, width = t.block_table.shape
    kv_lens = context + new
    want = torch.clamp((kv_lens + block - 1) // block, max=width)
    take, give = torch.clamp(want - t.held, min=0), torch.clamp(t.held - want, min=0)
    before = torch.cumsum(take, 0) - take
    got = torch.minimum(torch.clamp(t.free_count - before, min=0), take)
    rows = torch.arange(requests, device="cuda")

    def entries(counts, first):
        """(request, entry) of counts[r] entries from first[r] on, in order."""
        r = torch.repeat_interleave(rows, counts)
        at = torch.arange(r.numel(), device="cuda") - torch.repeat_interleave(torch.cumsum(counts, 0) - counts, counts)
        return r, first[r] + at

    start = t.free_count - got.sum()
    r, e = entries(got, t.held)
    t.block_table[r, e] = t.free_list[start + torch.arange(r.numel(), device="cuda")]
    r, e = entries(give, want)
    t.free_list[start + torch.arange(r.numel(), device="cuda")] = t.block_table[r, e]
    t.block_table[r, e] = -1
    t.held.copy_(t.held + got - give)
    t.free_count.copy_(start + give.sum())
    ends = torch.cumsum(new, 0)
    query_starts = torch.clamp(torch.cat([ends.new_zeros(1), ends]), max=tokens).to(torch.int32)
    r, p = entries(new, context)
    entry = p // block
    has = entry < t.held[r]
    slot = torch.where(has, t.block_table[r, torch.clamp(entry, max=width - 1)] * block + p % block, -1)
    slots, positions = (torch.full((tokens,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    n = min(tokens, r.numel())
    slots[:n], positions[:n] = slot[:n].to(torch.int32), p[:n].to(torch.int32)
    unplaced = (r.numel() - (slots[:n] >= 0).sum()).to(torch.int32).view(1)
    return {"block_table": t.block_table, "held": t.held, "free_count": t.free_count, "query_starts": query_starts,
            "kv_lens": kv_lens.to(torch.int32), "slots": slots, "positions": positions, "unplaced": unplaced}


def _plain_gather(cache, slots):
    """Keys and values of slots (of 0 and more), as f32 [slots, kv_heads, 256]."""
    units = cache.block // 16
    block, unit, t = slots // cache.block, slots % cache.block // 16, slots % 16
    k = cache.keys.view(cache.blocks, cache.kv_heads, units, 4, 4, 16, 16)[block, :, unit, :, :, t, :]
    k = _of_codes(k.reshape(-1, cache.kv_heads, DIM)) * _power(cache.key_scales[block].int() - 127)[..., None]
    v = cache.values.view(cache.blocks, cache.kv_heads, units, 4, 4, 16, 4, 4)[block, :, unit, :, t // 4, :, :, t % 4]
    v = v.permute(0, 1, 2, 4, 3).reshape(-1, cache.kv_heads, DIM)
    return k, _of_codes(v) * _power(cache.value_scales[block].int() - 127)[..., None]


def _plain_store(cache, which, x, slots):
    as_rows, as_codes = _ORDER[which]
    codes, scales = getattr(cache, which), getattr(cache, which[:-1] + "_scales")
    x, x_slots = x[slots >= 0].float(), slots[slots >= 0].long()
    touched, of = torch.unique(x_slots // cache.block, return_inverse=True)
    offset = x_slots % cache.block
    first = torch.full_like(touched, cache.block).scatter_reduce(0, of, offset, "amin")
    size = x.abs()
    size = torch.where(size < math.inf, size, 0.0).amax(dim=-1)
    amax = torch.zeros(touched.numel(), cache.kv_heads, device="cuda")
    amax = amax.scatter_reduce(0, of[:, None].expand(-1, cache.kv_heads), size, "amax")
    old = scales[touched].int() - 127
    e = _exponent(amax).int()
    e = torch.where((first > 0)[:, None], torch.maximum(old, e), e)
    rows = as_rows(codes[touched], cache.block)
    kept = (torch.arange(cache.block, device="cuda") < first[:, None])[:, None, :, None]
    rows = torch.where(kept, _to_codes(_of_codes(rows) * _power(old - e)[..., None, None]), rows)
    rows[of, :, offset] = _to_codes(x * _power(-e)[of][..., None])
    codes[touched] = as_codes(rows, cache.block)
    scales[touched] = (e + 127).to(torch.uint8)


def _plain_attention(q, gate, cache, t, context, new, out):
    heads, group = q.shape[1], q.shape[1] // cache.kv_heads
    first = 0
    for r, (c, n) in enumerate(zip(context, new)):
        positions = torch.arange(c + n, device="cuda")
        k, v = _plain_gather(cache, t.block_table[r][positions // cache.block] * cache.block + positions % cache.block)
        for kv in range(cache.kv_heads):
            of = slice(kv * group, kv * group + group)  # the q heads that share the kv head
            kh, vh = k[:, kv].contiguous(), v[:, kv].contiguous()
            for i in range(first, first + n, 512):
                rows = slice(i, min(i + 512, first + n))
                s = (q[rows, of].float().reshape(-1, DIM) @ kh.T) / math.sqrt(DIM)
                at = torch.arange(c + i - first, c + rows.stop - first, device="cuda").repeat_interleave(group)
                s = torch.where(positions <= at[:, None], s, -math.inf)
                p = torch.exp(s - s.amax(dim=1, keepdim=True))
                o = ((p @ vh) / p.sum(dim=1, keepdim=True)).view(-1, group, DIM)
                if gate is not None:
                    o = o / (1.0 + torch.exp(-gate[rows, of].float()))
                out[rows, of] = o.to(out.dtype)
        first += n
    return out


def run(state):
    kind = state["kind"]
    if kind == "tables":
        t = state["tables"]
        if not own:
            _plain_tables(t, state["context"], state["none"], state["block"], state["tokens"])
            return _plain_tables(t, state["context"], state["new"], state["block"], state["tokens"])
        t.encode(state["context"], state["none"])
        t.encode(state["context"], state["new"])
        return {n: getattr(t, n) for n in ("block_table", "held", "free_count", "query_starts", "kv_lens", "slots", "positions",
                                           "unplaced")}
    if kind in ("store", "gather"):
        cache, out = state["cache"], state["out"]
        back = state["back"] if kind == "store" else state["slots"]
        if own:
            if kind == "store":
                cache.encode(state["k"], state["v"], state["slots"])
            cache.encode_dequantize(back, out["keys"], out["values"])
            return out
        if kind == "store":
            _plain_store(cache, "keys", state["k"], state["slots"])
            _plain_store(cache, "values", state["v"], state["slots"])
        k, v = _plain_gather(cache, back)
        return {"keys": k.to(out["keys"].dtype), "values": v.to(out["values"].dtype)}
    t, out = state["tables"], state["out"]
    if own:
        state["attention"].encode_split(t)
    for layer, cache in enumerate(state["caches"]):
        q = state["both"][layer, :, :, :DIM]
        gate = state["both"][layer, :, :, DIM:] if state["gate"] else None
        if own:
            state["attention"].encode(q, cache, t, out[layer], gate=gate)
        else:
            _plain_attention(q, gate, cache, t, state["context"], state["new"], out[layer])
    return out


def work(case):
    context, new = _lengths(case)
    requests, tokens = len(context), sum(new)
    if case["kind"] == "tables":
        taken = sum(-(-(c + n) // case["block"]) - -(-c // case["block"]) for c, n in zip(context, new))
        # lengths and held blocks in; held, lengths and starts out; every block's number from list to table and back; slot and
        # position a token
        return {"bytes": 4 * (requests * 7 + 4 * taken + 2 * tokens), "flops": 0}
    kv_heads = case["kv_heads"]
    row = kv_heads * DIM
    if case["kind"] == "gather":
        size = TYPES[case["type"]].itemsize
        return {"bytes": 2 * sum(context) * row * (1 + size), "flops": 0}
    if case["kind"] == "store":
        size, block = TYPES[case["type"]].itemsize, case["block"]
        touched = sum(c + n - c // block * block for c, n in zip(context, new))
        return {"bytes": 2 * row * (tokens * (size + 1) + touched * (1 + 4)), "flops": 0}
    heads, size = case["heads"], 2
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(context, new))
    nbytes = 2 * row * (sum(context) + tokens) + tokens * heads * DIM * size * (3 if case["gate"] else 2)
    return {"bytes": case["layers"] * nbytes, "flops": case["layers"] * 4.0 * heads * DIM * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def _e4m3_values():
    """What each of the 256 codes stands for."""
    out = []
    for c in range(256):
        field, mantissa = c >> 3 & 15, c & 7
        x = math.ldexp(8 + mantissa, field - 10) if field else math.ldexp(mantissa, -9)
        out.append(math.nan if c & 127 == 127 else -x if c & 128 else x)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _double_power(e):
    """2^e, as it is."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _nearest_e4m3(x):
    """x, of magnitudes up to 448, rounded to what e4m3 holds, ties to even."""
    _, exponent = torch.frexp(x)
    step = _double_power(torch.clamp(exponent - 4, min=-9))
    return torch.round(x / step) * step


def _exact_rows(cache, which, slot):
    """[kv_heads, 256] values of every slot of a list, byte by byte of the layout."""
    d = torch.arange(DIM, device="cuda")
    t = (slot % 16)[:, None]
    if which == "keys":
        byte = d // 64 * 1024 + (d // 16 % 4 * 16 + t) * 16 + d % 16
    else:
        byte = d // 64 * 1024 + (t // 4 * 16 + d % 16) * 16 + d // 16 % 4 * 4 + t % 4
    byte = byte + (slot % cache.block // 16 * 4096)[:, None]
    block = slot // cache.block
    scales = cache.key_scales if which == "keys" else cache.value_scales
    flat = (block[:, None] * cache.kv_heads + torch.arange(cache.kv_heads, device="cuda")) * cache.block * DIM
    codes = getattr(cache, which).reshape(-1)[flat[:, :, None] + byte[:, None, :]]
    return _e4m3_values()[codes.long()] * _double_power(scales[block].long() - 127)[..., None]


def _exact_tables(state, case):
    context, new = _lengths(case)
    t, block, tokens = state["tables"], state["block"], state["tokens"]
    table, held, free = t.block_table.tolist(), t.held.tolist(), t.free_list.tolist()[:int(t.free_count)]
    slots, positions, starts = [], [], [0]
    takes = [max(0, -(-(c + n) // block) - h) for c, n, h in zip(context, new, held)]
    first = len(free) - sum(takes)
    for r, n in enumerate(takes):
        table[r][held[r]:held[r] + n] = free[first:first + n]
        held[r] += n
        first += n
    for r, (c, n) in enumerate(zip(context, new)):
        for p in range(c, c + n):
            slots.append(table[r][p // block] * block + p % block), positions.append(p)
        starts.append(starts[-1] + n)
    behind = [-1] * (tokens - len(slots))
    ints = {"dtype": torch.int32, "device": "cuda"}
    return {"block_table": torch.tensor(table, **ints), "held": torch.tensor(held, **ints),
            "free_count": torch.tensor([len(free) - sum(takes)], **ints), "query_starts": torch.tensor(starts, **ints),
            "kv_lens": torch.tensor([c + n for c, n in zip(context, new)], **ints), "slots": torch.tensor(slots + behind, **ints),
            "positions": torch.tensor(positions + behind, **ints), "unplaced": torch.tensor([0], **ints)}


def _exact_store(state):
    cache, block, slots = state["cache"], state["cache"].block, state["slots"].long()
    out = {}
    for which, x in (("keys", state["k"]), ("values", state["v"])):
        x = x.double()
        back = state["back"].long()
        scales = cache.key_scales if which == "keys" else cache.value_scales
        value = _exact_rows(cache, which, back)
        place = torch.full((cache.blocks * block,), -1, device="cuda")
        place[back] = torch.arange(back.numel(), device="cuda")
        old = scales.long() - 127
        top = torch.zeros(cache.blocks, cache.kv_heads, dtype=torch.float64, device="cuda")
        top.index_reduce_(0, slots // block, x.abs().amax(dim=-1), "amax")
        m, e = torch.frexp(top / 448.0)  # the least power of two that is no less than top / 448
        e = torch.clamp(torch.where(m == 0.5, e - 1, e), LOWEST, HIGHEST).long()
        starts_over = torch.zeros(cache.blocks, dtype=torch.bool, device="cuda")
        starts_over[slots[slots % block == 0] // block] = True
        e = torch.where(starts_over[:, None], e, torch.maximum(e, old))
        scale = _double_power(e)
        value = _nearest_e4m3(value / scale[back // block][..., None]) * scale[back // block][..., None]
        s = scale[slots // block][..., None]
        value[place[slots]] = _nearest_e4m3(x / s) * s
        out[which] = value
    return out


def _exact_attention(state, case):
    heads, kv_heads = case["heads"], case["kv_heads"]
    t, out = state["tables"], []
    for layer, cache in enumerate(state["caches"]):
        both = state["both"][layer].double()
        result, first = torch.zeros(both.shape[0], heads, DIM, dtype=torch.float64, device="cuda"), 0
        for r, (c, n) in enumerate(zip(state["context"], state["new"])):
            p = torch.arange(c + n, device="cuda")
            slot = t.block_table[r].long()[p // cache.block] * cache.block + p % cache.block
            parts = [[_exact_rows(cache, w, s) for s in slot.split(8192)] for w in ("keys", "values")]
            keys, values = (torch.cat(x).transpose(0, 1).contiguous() for x in parts)
            for h in range(heads):
                kv = h // (heads // kv_heads)
                for i in range(0, n, 1024):
                    m = min(1024, n - i)
                    weights = both[first + i:first + i + m, h, :DIM] @ keys[kv].T / 16.0
                    unseen = p[None, :] > (c + i + torch.arange(m, device="cuda"))[:, None]
                    weights = torch.softmax(weights.masked_fill(unseen, -math.inf), dim=1)
                    o = weights @ values[kv]
                    if state["gate"]:
                        o = o * torch.sigmoid(both[first + i:first + i + m, h, DIM:])
                    result[first + i:first + i + m, h] = o
            first += n
        out.append(result)
    return torch.stack(out)


def exact(case, seed):
    global own
    was, own = own, False  # (the inputs alone)
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "tables":
        return _exact_tables(state, case)
    if case["kind"] == "store":
        return _exact_store(state)
    if case["kind"] == "gather":
        return {w: _exact_rows(state["cache"], w, state["slots"].long()) for w in ("keys", "values")}
    return _exact_attention(state, case)

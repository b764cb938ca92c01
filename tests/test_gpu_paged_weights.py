"""The weights of the attention over paged caches where f16 holds them least well: a great many small ones beside a large one."""
import numpy as np
import pytest
import torch

from gpu_common import saetta
from paged_common import DIM
from test_gpu_paged import F16, ints, numbers

pytestmark = pytest.mark.gpu


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

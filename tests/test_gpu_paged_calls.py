"""Calls over paged caches that a program may make and the other tests do not: steps without a new token."""
import numpy as np
import pytest
import torch

from gpu_common import host, saetta
from paged_common import DIM, tables as plain_tables
from test_gpu_paged import F16, compare_tables, ints, plain_state

pytestmark = pytest.mark.gpu


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

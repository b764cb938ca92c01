"""What the calls over a cache in blocks refuse, by arguments alone: on the CPU, through the C ABI, and the plain statement of
the cache that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from paged_common import DIM, E4M3, Cache, exponent, key_byte, nearest, places, tables, value_byte

saetta = entry.load_package()
ffi = saetta.ffi
A = 0x10000  # an address that no call gets as far as using


def cache(**over):
    fields = dict(keys=A, values=A, key_scales=A, value_scales=A, blocks=8, block_tokens=64, kv_heads=2)
    return ffi.PagedCacheC(**{**fields, **over})


def batch(**over):
    fields = dict(query_starts=A, kv_lens=A, block_table=A, requests=3, max_blocks=4, block_tokens=64)
    return ffi.PagedBatchC(**{**fields, **over})


def params(**over):
    return ffi.PagedAttnParamsC(**{**dict(heads=16, kv_heads=2, tokens=5, rows=1, scale=0.0625), **over})


def rows(data=A, token=4096, head=256):
    return ffi.StridedRowsC(data, token, head)


def refused(rc, code, text):
    assert rc == code, (rc, ffi.lib().saetta_last_error())
    assert text in ffi.lib().saetta_last_error().decode()


@pytest.mark.parametrize("over, code, text", [
    (dict(block_tokens=48), -2, "blocks of 48 tokens"), (dict(block_tokens=0), -2, "blocks of 0"), (dict(block_tokens=256), -2, "256"),
    (dict(blocks=0), -2, "0 blocks"), (dict(blocks=1 << 25), -2, "2^31"), (dict(kv_heads=0), -2, "kv heads"),
    (dict(keys=None), -3, "null"), (dict(value_scales=None), -3, "null"), (dict(values=A + 8), -4, "16-byte")])
def test_a_cache_that_is_none(over, code, text):
    l = ffi.lib()
    refused(l.saetta_paged_store(None, 1, rows(), rows(), A, cache(**over), 1), code, text)
    refused(l.saetta_paged_gather(None, 1, cache(**over), A, A, A, 1), code, text)
    if "block_tokens" not in over and "kv_heads" not in over:
        refused(l.saetta_paged_attn(None, 1, rows(), cache(**over), batch(), A, rows(None), rows(), params(), A, 1 << 40), code, text)


def test_store_and_gather_refuse():
    l = ffi.lib()
    refused(l.saetta_paged_store(None, 3, rows(), rows(), A, cache(), 1), -1, "type 3")
    refused(l.saetta_paged_store(None, 1, rows(None), rows(), A, cache(), 1), -3, "null")
    refused(l.saetta_paged_store(None, 1, rows(), rows(), None, cache(), 1), -3, "null")
    refused(l.saetta_paged_store(None, 1, rows(A + 2), rows(), A, cache(), 1), -4, "16-byte")
    refused(l.saetta_paged_store(None, 1, rows(), rows(head=260), A, cache(), 1), -4, "16-byte")
    refused(l.saetta_paged_store(None, 0, rows(), rows(token=513), A, cache(), 1), -4, "16-byte")
    refused(l.saetta_paged_store(None, 0, rows(), rows(), A, cache(), 1 << 28), -2, "2^28")
    refused(l.saetta_paged_gather(None, 0, cache(), A, A, A, 1 << 28), -2, "2^28")
    refused(l.saetta_paged_gather(None, -1, cache(), A, A, A, 1), -1, "type")
    refused(l.saetta_paged_gather(None, 0, cache(), None, A, A, 1), -3, "null")
    refused(l.saetta_paged_gather(None, 0, cache(), A, A + 4, A, 1), -4, "16-byte")


@pytest.mark.parametrize("over, code", [(dict(block_tokens=8), -2), (dict(blocks=0), -2), (dict(max_blocks=0), -2), (dict(max_blocks=1 << 26), -2),
                                        (dict(requests=1 << 24), -2), (dict(tokens=1 << 31), -2)])
def test_tables_refuse(over, code):
    fields = {**dict(requests=3, max_blocks=4, block_tokens=64, blocks=8, tokens=10), **over}
    p, state, step = ffi.PagedTablesParamsC(**fields), ffi.PagedStateC(A, A, A, A), ffi.PagedStepC(A, A, A, A, A)
    l = ffi.lib()
    assert l.saetta_paged_tables(None, A, A, state, step, p) == code
    good = ffi.PagedTablesParamsC(3, 4, 64, 8, 10)
    assert l.saetta_paged_tables(None, None, A, state, step, good) == -3
    assert l.saetta_paged_tables(None, A, A, ffi.PagedStateC(A, A, None, A), step, good) == -3
    assert l.saetta_paged_tables(None, A, A, state, ffi.PagedStepC(A, A, A, A + 2, A), good) == -4


@pytest.mark.parametrize("over, text", [(dict(heads=15), "15 q heads"), (dict(heads=6), "3 q heads per kv head"), (dict(heads=64), "32 q heads"),
                                        (dict(kv_heads=0), "0 kv heads"), (dict(heads=0), "0 q heads"), (dict(rows=0), "rows 0"),
                                        (dict(tokens=1 << 31), "tokens"), (dict(scale=0.0), "scale"), (dict(scale=-0.0625), "scale"),
                                        (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                                        (dict(tokens=(1 << 30), rows=100), "tokens")])
def test_attention_refuses_shapes(over, text):
    l = ffi.lib()
    refused(l.saetta_paged_split(None, batch(), params(**over), A), -2, text)
    refused(l.saetta_paged_attn(None, 1, rows(), cache(), batch(), A, rows(None), rows(), params(**over), A, 1 << 40), -2, text)
    assert l.saetta_paged_split_bytes(params(**over), 3) == 0 and l.saetta_paged_workspace_bytes(params(**over), 3) == 0


def test_sizes_that_no_memory_holds():
    p = ffi.PagedTablesParamsC(1 << 23, 1 << 9, 16, 8, 10)
    refused(ffi.lib().saetta_paged_tables(None, A, A, ffi.PagedStateC(A, A, A, A), ffi.PagedStepC(A, A, A, A, A), p), -2, "2^31 entries")
    refused(ffi.lib().saetta_paged_store(None, 0, rows(), rows(), A, cache(blocks=1 << 22, block_tokens=16, kv_heads=4096), 1), -2, "2^32")


def test_attention_refuses_buffers():
    l, p = ffi.lib(), params()
    need = l.saetta_paged_workspace_bytes(p, 3)

    def attn(type_=1, q=rows(), c=cache(), b=batch(), split=A, gate=rows(None), out=rows(), ws=A, size=need):
        return l.saetta_paged_attn(None, type_, q, c, b, split, gate, out, p, ws, size)

    refused(attn(type_=0), -1, "f16 or bf16")
    refused(attn(q=rows(None)), -3, "null")
    refused(attn(split=None), -3, "null")
    refused(attn(ws=None), -3, "null")
    refused(attn(ws=A + 8), -4, "16-byte")
    refused(attn(q=rows(head=252)), -4, "16-byte")
    refused(attn(gate=rows(A + 2)), -4, "16-byte")
    refused(attn(q=rows(token=1 << 32)), -2, "2^32")
    refused(attn(out=rows(head=1 << 33)), -2, "2^32")
    refused(attn(size=need - 1), -6, "needed")
    refused(attn(c=cache(kv_heads=4)), -2, "kv heads")
    refused(attn(c=cache(block_tokens=32)), -2, "blocks of 32")
    refused(attn(b=batch(kv_lens=None)), -3, "null")
    refused(attn(b=batch(max_blocks=0)), -2, "0 blocks")
    refused(l.saetta_paged_split(None, batch(), p, None), -3, "null")
    refused(l.saetta_paged_split(None, batch(), p, A + 4), -4, "16-byte")


def test_python_objects_refuse():
    for wrong in (dict(head_dim=128), dict(block_tokens=8), dict(blocks=0), dict(blocks=1 << 25)):
        with pytest.raises(ValueError):
            saetta.PagedCache(**{**dict(kv_heads=2, head_dim=256, blocks=4, block_tokens=64, device="cpu"), **wrong})
    for wrong in (dict(requests=0), dict(tokens=0), dict(max_blocks=0), dict(block_tokens=24)):
        with pytest.raises(ValueError):
            saetta.PagedTables(**{**dict(requests=2, tokens=4, max_blocks=4, blocks=8, block_tokens=64, device="cpu"), **wrong})
    c = saetta.PagedCache(2, 256, 4, 64, device="cpu")
    with pytest.raises(TypeError):  # nothing of it runs on the CPU
        c.encode(torch.zeros(1, 2, 256), torch.zeros(1, 2, 256), torch.zeros(1, dtype=torch.int32))
    t = saetta.PagedTables(2, 4, 4, 8, device="cpu")
    with pytest.raises(TypeError):
        t.encode(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_recorded_calls_refuse_tensors_of_two_devices():
    import sys
    one_device = sys.modules[saetta.PagedCache.__module__]._one_device
    a, b = torch.zeros(2), torch.zeros(2, device="meta")
    one_device("x", a, None, a), one_device("x", b, b)
    with pytest.raises(ValueError, match="one device"):
        one_device("x", a, None, b)


def test_parameter_blocks_have_the_header_sizes():
    import os
    import subprocess
    import tempfile
    names = {"saetta_paged_cache": ffi.PagedCacheC, "saetta_paged_state": ffi.PagedStateC, "saetta_paged_step": ffi.PagedStepC,
             "saetta_paged_tables_params": ffi.PagedTablesParamsC, "saetta_strided_rows": ffi.StridedRowsC,
             "saetta_paged_batch": ffi.PagedBatchC, "saetta_paged_attn_params": ffi.PagedAttnParamsC}
    header = os.path.join(entry.ROOT, "include", "saetta_hip.h")
    body = "".join(f'printf("%zu\\n", sizeof({n}));' for n in names)
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(src, "w").write(f'#include "{header}"\n#include <stdio.h>\nint main(void) {{ {body} return 0; }}\n')
        subprocess.run(["gcc", "-std=c99", src, "-o", exe], check=True)
        sizes = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(c) for c in names.values()]


# ---- the plain statement ----------------------------------------------------------------------------------------------

def test_codes_are_torchs():
    """The table of values and the rounding, against torch's own e4m3."""
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(E4M3, codes.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)
    gen = np.random.default_rng(1)
    x = np.concatenate([gen.standard_normal(5000) * np.exp2(gen.uniform(-12, 8, 5000)), (E4M3[:126] + E4M3[1:127]) / 2]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    assert np.array_equal(nearest(x), torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(nearest([449.0, np.inf, -np.inf, np.nan])).all()


def test_places_are_a_permutation():
    for byte in (key_byte, value_byte):
        for bt in (16, 64, 128):
            assert np.array_equal(np.sort(places(bt, byte).ravel()), np.arange(bt * DIM))


def test_exponents():
    assert [exponent(x) for x in (0.0, 448.0, 448.0001, 896.0, 1.75, 1.7500001, 1e-30, 1e30)] == [-40, 0, 1, 1, -8, -7, -40, 60]


def test_a_later_token_moves_the_scale():
    c = Cache(1, 1, 16)
    k = np.ones((3, 1, DIM))
    k[1] *= 0.3
    k[2] *= 1000.0
    c.store(k[:2], k[:2], [0, 1])
    assert c.e["keys"][0, 0] == -8 and c.rows["keys"][0, 0, 1, 0] == 0.3125
    c.store(k[2:], k[2:], [2])
    assert c.e["keys"][0, 0] == 2 and c.rows["keys"][0, 0, 2, 0] == 1024.0 and c.rows["keys"][0, 0, 1, 0] == 0.3125
    c.store(k[:1], k[:1], [0])  # begins the block anew
    assert c.e["keys"][0, 0] == -8


def test_tables_take_and_give_back():
    state = {"block_table": np.full((3, 4), -1), "held": [0, 0, 0], "free": list(range(6))}
    step = tables(state, [0, 0, 0], [17, 0, 32], 16, 60)
    assert state["held"] == [2, 0, 2] and state["free"] == [0, 1] and state["block_table"][0, :2].tolist() == [2, 3]
    assert step["slots"][16] == 48 and step["query_starts"] == [0, 17, 17, 49] and step["unplaced"] == [0]
    tables(state, [0, 0, 0], [0, 0, 0], 16, 60)
    assert state["free"] == list(range(6)) and (state["block_table"] == -1).all()
    step = tables(state, [0, 0, 0], [90, 10, 10], 16, 200)  # past a row of the table, and past the blocks there are
    assert state["held"] == [4, 1, 1] and step["unplaced"] == [90 - 64]

"""What the paged calls refuse of strides and sizes, by arguments alone: on the CPU."""
import pytest
import torch

from test_paged_refusals import A, batch, cache, ffi, params, refused, rows, saetta


def attn(out, **over):
    p = params(**over)
    return ffi.lib().saetta_paged_attn(None, 1, rows(), cache(kv_heads=p.kv_heads), batch(), A, rows(None), out, p, A, 1 << 40)


@pytest.mark.parametrize("token, head, over", [
    (0, 0, {}), (0, 256, {}), (4096, 0, {}), (4096, 128, {}), (128, 4096, {}), (4088, 256, {}), (512, 256, {}), (256, 256, {}), (3840, 256, {}), (256, 1024, {}),
    (768, 512, {}),  # three heads on is two tokens on
    (256, 8, dict(tokens=2, heads=2)), (0, 256, dict(tokens=2, heads=2)), (4294967288, 4294967288, dict(tokens=3, heads=16))])
def test_rows_of_the_output_that_overlap(token, head, over):
    refused(attn(rows(token=token, head=head), **over), -2, "overlap")


@pytest.mark.parametrize("token, head, over", [
    (4096, 256, {}), (256, 1280, {}), (8192, 512, {}), (0, 256, dict(tokens=1)), (256, 0, dict(heads=1, kv_heads=1)), (0, 0, dict(tokens=1, heads=1, kv_heads=1)),
    (768, 512, dict(tokens=2, heads=4, kv_heads=4)), (4096, 256, dict(tokens=(1 << 24) - 1)), (0, 0, dict(tokens=0, heads=1, kv_heads=1))])
def test_rows_of_the_output_that_lie_apart(token, head, over):
    """Refused for something else that is looked at later: a workspace that is not aligned."""
    p = params(**over)
    out = ffi.lib().saetta_paged_attn(None, 1, rows(), cache(kv_heads=p.kv_heads), batch(), A, rows(None), rows(token=token, head=head), p, A + 8, 1 << 40)
    refused(out, -4, "split and workspace")


def test_buffers_and_sizes_cannot_be_replaced():
    """A buffer put in another's place was read by recorded calls and not by others."""
    for made, names in ((saetta.PagedCache(2, 256, 4, 64, device="cpu"), ("keys", "value_scales", "blocks", "kv_heads")),
                        (saetta.PagedTables(2, 4, 4, 8, device="cpu"), ("block_table", "free_count", "kv_lens", "slots", "tokens", "max_blocks"))):
        for name in names:
            was = getattr(made, name)
            with pytest.raises(AttributeError, match=name):
                setattr(made, name, was.clone() if isinstance(was, torch.Tensor) else was + 1)
            assert getattr(made, name) is was


@pytest.mark.parametrize("tokens, ok", [((1 << 28) - 32, True), ((1 << 28) - 31, False), ((1 << 28) - 1, False)])
def test_the_most_tokens_of_a_call(tokens, ok):
    """A launch has fewer than 2^32 threads."""
    l = ffi.lib()
    for size in (16, 32, 64):
        for rc in (l.saetta_paged_store(None, 1, rows(), rows(), A + (2 if ok else 0), cache(block_tokens=size), tokens),
                   l.saetta_paged_gather(None, 1, cache(block_tokens=size), A + (2 if ok else 0), A, A, tokens)):
            refused(rc, -4, "") if ok else refused(rc, -2, "2^28 - 32")


def test_sizes_past_32_bits():
    """Cut to 32 bits they would be another call's: rows 2^32 + 1 were taken for 1."""
    tables = saetta.PagedTables(2, 4, 4, 8, device="cpu")
    for over in (dict(rows=(1 << 32) + 1), dict(heads=(1 << 32) + 16, kv_heads=(1 << 32) + 16)):
        with pytest.raises(ValueError, match="2\\^32"):
            saetta.PagedAttention(**{**dict(heads=16, kv_heads=2, head_dim=256, tables=tables, rows=1), **over})
    for over in (dict(requests=(1 << 32) + 1), dict(tokens=1 << 32)):
        with pytest.raises(ValueError, match="2\\^32"):
            saetta.PagedTables(**{**dict(requests=1, tokens=1, max_blocks=1, blocks=1, device="meta"), **over})
    with pytest.raises(ValueError, match="2\\^32"):
        saetta.PagedCache((1 << 32) + 2, 256, 4, 64, device="meta")

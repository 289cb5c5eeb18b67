"""The paged operators' limits of counts, without a GPU."""
import pytest

from frizzle_b200 import _native

from test_paged import P, cache, query, refused, rows


@pytest.mark.parametrize("sequences,kv_heads,page_slots,heads", [
    (1 << 29, 1, 1 << 30, 8), ((1 << 31) - 1, 1, 1 << 30, 8), (1 << 20, 1 << 11, 1 << 30, 1 << 14), (0xFFFFFFFF, 65535, 1 << 30, 8 * 65535)])
def test_workspace_of_more_than_64_bits_is_no_small_one(sequences, kv_heads, page_slots, heads):
    """4 bytes a query head and table entry: 2^64 bytes and more, for which no workspace is long enough."""
    lib = _native.load()
    c = cache(sequences=sequences, kv_heads=kv_heads, table_stride=1, page_slots=page_slots)
    assert sequences * page_slots * heads * 4 >= 1 << 64
    assert lib.fz_paged_attention_workspace(c, heads) >= 1 << 62
    if sequences * kv_heads < 1 << 31 and heads <= 8 * kv_heads:
        refused(lib.fz_paged_attention(c, query(heads=heads, q_stride=1 << 20, out_stride=1 << 20, workspace_bytes=(1 << 62) - 1), None),
                1, "workspace")


@pytest.mark.parametrize("sequences,kv_heads", [(1 << 31, 1), (0xFFFFFFFF, 1), (1 << 20, 1 << 12)])
def test_more_sequences_than_31_bits_are_refused(sequences, kv_heads):
    """Counters of 32 bits run over sequences times KV heads in steps."""
    lib = _native.load()
    c = cache(sequences=sequences, kv_heads=kv_heads)
    refused(lib.fz_paged_append(c, rows(), None), 1, "sequences")
    refused(lib.fz_paged_bounds(c, None, None), 1, "sequences")
    refused(lib.fz_paged_select(c, P, kv_heads * 256, kv_heads, 2, 0, 0, P, None, None), 1, "sequences")
    refused(lib.fz_paged_attention(c, query(heads=kv_heads, q_stride=kv_heads * 256, out_stride=kv_heads * 256), None), 1, "sequences")
    refused(lib.fz_paged_evict(c, c, 8, 0, 0, P, None), 1, "sequences")


@pytest.mark.parametrize("count", [(1 << 30) + 1, 0xFFFFFFFF])
def test_lists_longer_than_any_table_are_refused(count):
    """`top` and `budget` are lengths of lists that every call writes whole; no table has more than 2^30 entries."""
    lib = _native.load()
    refused(lib.fz_paged_select(cache(), P, 1024, 4, count, 0, 0, P, None, None), 1, "2^30")
    refused(lib.fz_paged_evict(cache(), cache(), count, 0, 0, P, None), 1, "2^30")

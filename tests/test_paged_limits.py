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

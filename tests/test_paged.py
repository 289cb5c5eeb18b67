"""The paged operators' refusals and descriptions, without a GPU: every check made on the host comes before a pointer
is looked at or a kernel launched."""
import ctypes as C

import pytest

from frizzle_b200 import _native

P = 0x10000        # an aligned stand-in address; nothing is dereferenced


def cache(**kw):
    c = _native.PagedKv()
    base = dict(keys=P, values=P, page_table=P, lengths=P, weights=P, bounds=P, error=None, page_stride=16 * 256,
                slot_stride=256, head_stride=256, sequences=2, table_stride=4, pages=8, page_slots=16, kv_heads=1,
                head_dim=256, type=0)
    for k, v in dict(base, **kw).items():
        setattr(c, k, v)
    return c


def rows(**kw):
    r = _native.PagedRows()
    base = dict(q=P, k=P, v=P, q_out=P, q_stride=1536, k_stride=1536, v_stride=1536, q_out_stride=1024, q_gain=P, k_gain=P,
                turns=P, sequence=P, index=P, position=None, rows=2, heads=4, eps=1e-6)
    for k, v in dict(base, **kw).items():
        setattr(r, k, v)
    return r


def query(**kw):
    q = _native.PagedQuery()
    base = dict(q=P, out=P, q_stride=1024, out_stride=1024, blocks=None, workspace=P, workspace_bytes=1 << 40, heads=4,
                top=0, window=0, scale=0.0625, decay=0.0)
    for k, v in dict(base, **kw).items():
        setattr(q, k, v)
    return q


def refused(status, want, part):
    assert status == want, (status, _native.load().fz_last_error())
    assert part in _native.load().fz_last_error().decode(), _native.load().fz_last_error()


def test_struct_sizes_match_header():
    assert C.sizeof(_native.PagedKv) == 112
    assert C.sizeof(_native.PagedRows) == 128
    assert C.sizeof(_native.PagedQuery) == 80


CACHES = [
    (dict(type=2), 1, "type"), (dict(head_dim=96), 11, "head dimension"), (dict(kv_heads=0), 1, "nonzero"),
    (dict(page_slots=0), 1, "nonzero"), (dict(pages=0), 1, "nonzero"), (dict(table_stride=0), 1, "nonzero"),
    (dict(table_stride=1 << 20, page_slots=1 << 12), 1, "2^30"), (dict(page_table=None), 1, "null page table"),
    (dict(lengths=None), 1, "null page table"), (dict(lengths=P + 2), 1, "4-byte"), (dict(error=P + 1), 1, "4-byte"),
]
KEYS = [
    (dict(keys=None), 1, "null keys"), (dict(values=P + 8), 1, "16-byte"), (dict(slot_stride=260), 1, "multiples of 8"),
    (dict(page_stride=128), 1, "shorter"), (dict(kv_heads=2, head_stride=128), 1, "shorter"),
]


@pytest.mark.parametrize("kw,status,part", CACHES + KEYS)
def test_cache_refusals(kw, status, part):
    lib = _native.load()
    c, ok = cache(**kw), cache()
    refused(lib.fz_paged_append(c, rows(), None), status, part)
    refused(lib.fz_paged_attention(c, query(heads=4 * max(1, c.kv_heads)), None), status, part)
    refused(lib.fz_paged_bounds(c, None, None), status, part)
    refused(lib.fz_paged_evict(c, ok, 8, 0, 0, P, None), status, part)
    refused(lib.fz_paged_evict(ok, c, 8, 0, 0, P, None), status, part)
    if (kw, status, part) in CACHES:
        refused(lib.fz_paged_select(c, P, 1024, 4, 2, 0, 0, P, None, None), status, part)


@pytest.mark.parametrize("kw,part", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(index=None), "null"),
    (dict(q_out=None), "null"), (dict(q=P + 4), "16-byte"), (dict(turns=P + 8), "16-byte"), (dict(index=P + 2), "4-byte"),
    (dict(k_stride=1538), "multiples of 4"), (dict(q_stride=512), "shorter"), (dict(v_stride=128), "shorter"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(heads=1 << 17), "heads"),
])
def test_append_refusals(kw, part):
    refused(_native.load().fz_paged_append(cache(), rows(**kw), None), 1, part)


@pytest.mark.parametrize("kw,part", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=P + 8), "16-byte"), (dict(out_stride=1022), "multiples of 4"),
    (dict(heads=0), "heads"), (dict(heads=9), "heads"), (dict(q_stride=512), "shorter"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(decay=-0.5), "decay"),
    (dict(decay=float("nan")), "decay"), (dict(blocks=P), "top"), (dict(blocks=P + 1, top=2), "4-byte"),
    (dict(workspace=None), "workspace"), (dict(workspace=P + 16), "workspace"), (dict(workspace_bytes=0), "workspace"),
])
def test_attention_refusals(kw, part):
    refused(_native.load().fz_paged_attention(cache(), query(**kw), None), 1, part)


def test_select_bounds_and_evict_refusals():
    lib = _native.load()
    for c, args, status, part in [
        (cache(bounds=None), {}, 1, "null bounds"), (cache(bounds=P + 8), {}, 1, "16-byte"),
        (cache(), dict(q=None), 1, "null q"), (cache(), dict(blocks=None), 1, "null q"),
        (cache(), dict(q=P + 4), 1, "16-byte"), (cache(), dict(stride=1026), 1, "multiple of 4"),
        (cache(), dict(stride=512), 1, "shorter"), (cache(), dict(heads=9), 1, "heads"), (cache(), dict(top=0), 1, "top"),
        (cache(), dict(sink=2, recent=1), 1, "sink + recent"),
        (cache(), dict(sink=0xFFFFFFFF, recent=0xFFFFFFFF), 1, "sink + recent"),
        (cache(table_stride=300000, page_slots=1), {}, 11, "more pages"),
    ]:
        a = dict(dict(q=P, stride=1024, heads=4, top=2, sink=0, recent=0, blocks=P), **args)
        refused(lib.fz_paged_select(c, a["q"], a["stride"], a["heads"], a["top"], a["sink"], a["recent"], a["blocks"], None,
                                    None), status, part)
    refused(lib.fz_paged_bounds(cache(), P + 2, None), 1, "first")
    for a, b, budget, sink, recent, kept, status, part in [
        (cache(weights=None), cache(), 8, 0, 0, P, 1, "null weights"), (cache(), cache(), 8, 0, 0, None, 1, "null kept"),
        (cache(), cache(), 0, 0, 0, P, 1, "budget"), (cache(), cache(), 8, 5, 4, P, 1, "budget"),
        (cache(), cache(type=1), 8, 0, 0, P, 1, "differ"), (cache(), cache(sequences=3), 8, 0, 0, P, 1, "differ"),
        (cache(), cache(table_stride=1), 20, 0, 0, P, 1, "destination"),
        (cache(table_stride=50000), cache(table_stride=50000), 8, 0, 0, P, 11, "more entries"),
    ]:
        refused(lib.fz_paged_evict(a, b, budget, sink, recent, kept, None), status, part)
    assert lib.fz_paged_append(None, rows(), None) == 1 and lib.fz_paged_append(cache(), None, None) == 1
    assert lib.fz_paged_attention(cache(), None, None) == 1


def test_nothing_to_do_is_ok_and_touches_nothing():
    lib = _native.load()
    assert lib.fz_paged_append(cache(), rows(rows=0), None) == 0
    c = cache(sequences=0)
    assert lib.fz_paged_attention(c, query(), None) == 0
    assert lib.fz_paged_bounds(c, None, None) == 0
    assert lib.fz_paged_select(c, P, 1024, 4, 2, 0, 0, P, None, None) == 0
    assert lib.fz_paged_evict(c, cache(sequences=0), 8, 0, 0, P, None) == 0


def test_without_a_device_the_calls_fail_loudly():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    lib = _native.load()
    assert lib.fz_paged_append(cache(), rows(), None) == 2
    assert lib.fz_paged_attention(cache(), query(), None) == 2
    assert lib.fz_last_error()

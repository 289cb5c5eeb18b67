"""The paged cache's operators on the GPU against their definitions in 64 bits (paged_cases.py, which derives the
bounds): appended rows, page bounds, selected pages, one-token attention and eviction, each where it can go wrong,
and a run of them together, captured and replayed."""
import math

import numpy as np
import pytest

from frizzle_b200 import _native

from paged_cases import (HALF_STEP, NONE, Cache, Rows, attend, attend_exact, best, bounds, chosen, evict, page_scores,
                         select, stream, torch_cuda)

pytestmark = pytest.mark.gpu


def u32(t):
    return t.cpu().numpy().view(np.uint32)


def randn(*shape, seed=0, scale=1.0):
    torch = torch_cuda()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def check_out(got, want, bound):
    torch = torch_cuda()
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), float((err / bound.clamp_min(1e-30)).max())
    rel = float(err.norm() / want.norm().clamp_min(1e-30))
    assert rel < 1e-5, rel       # (the f32 parity bar of the kernel tests)


# ------------------------------------------------------------------ append

def check_append(cache, rows, keys0, values0, lengths0):
    """Every output of an append against the definition, and everything else left as it was."""
    torch = torch_cuda()
    q, qe, k, ke, v = rows.exact(cache)
    want_k, want_v = keys0.clone().double().cpu().numpy(), values0.clone().double().cpu().numpy()
    tol_k, tol_v = np.zeros_like(want_k), np.zeros_like(want_v)
    lengths = np.array(lengths0, dtype=np.int64)
    step = HALF_STEP[cache.type]
    got_q = rows.q_out.reshape(q.shape).double().cpu().numpy() if rows.heads else None
    for r, (s, j) in enumerate(zip(rows.sequence, rows.index)):
        if s == NONE:
            assert not rows.heads or np.isnan(got_q[r]).all()        # a padding row's output is left as it was
            continue
        if rows.heads:
            assert (np.abs(got_q[r] - q[r]) <= qe[r]).all(), np.max(np.abs(got_q[r] - q[r]) / qe[r])
        p, o = cache.table_np[s, j // cache.page], j % cache.page
        most = 65504.0 if cache.type == "f16" else np.inf
        want_k[p, o], want_v[p, o] = np.clip(k[r], -most, most), np.clip(v[r], -most, most)
        tol_k[p, o] = ke[r] * (1 + step) + np.abs(want_k[p, o]) * step + 2.0 ** -25
        tol_v[p, o] = np.abs(want_v[p, o]) * step + 2.0 ** -25
        lengths[s] = max(lengths[s], int(j) + 1)
    for got, want, tol in ((cache.keys, want_k, tol_k), (cache.values, want_v, tol_v)):
        got = got.double().cpu().numpy()
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)
    assert np.array_equal(u32(cache.len).astype(np.int64), lengths)
    torch.cuda.synchronize()


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("d,heads,kv,order,page", [(256, 4, 1, "nhd", 16), (256, 8, 2, "hnd", 24), (128, 6, 2, "hnd", 1),
                                                    (64, 3, 3, "nhd", 40), (128, 8, 1, "nhd", 7), (256, 0, 2, "nhd", 16)])
def test_append(type, d, heads, kv, order, page):
    cache = Cache([5, 0, 37, 3], page=page, kv=kv, d=d, type=type, order=order, capacity=70, seed=d + heads, weights=True)
    keys0, values0, w0 = cache.keys.clone(), cache.values.clone(), cache.weights.clone()
    sequence = [0, 0, 0, 1, NONE, 2, 2, 3, NONE]
    index = [5, 6, 7, 0, 999999, 36, 37, 60, NONE]     # 36 is held already (a rewind), 60 past the length
    rows = Rows(cache, heads, sequence, index, seed=d)
    rows.append(cache)
    check_append(cache, rows, keys0, values0, cache.lengths)
    new = {(int(cache.table_np[s, j // page]), j % page) for s, j in zip(sequence, index) if s != NONE}
    w = cache.weights.cpu().numpy()
    for p in range(cache.pages):
        for o in range(page):
            assert (w[p, :, o] == (0 if (p, o) in new else w0[p, :, o].cpu().numpy())).all()
    assert int(cache.error) == 0


@pytest.mark.parametrize("rows_n,heads,kv,d", [(1, 4, 1, 256), (700, 4, 1, 256), (333, 16, 2, 64), (257, 5, 5, 128),
                                               (2500, 4, 1, 256), (2100, 7, 3, 128), (2001, 13, 4, 64)])
def test_append_many_rows(rows_n, heads, kv, d):
    cache = Cache([0], page=16, kv=kv, d=d, capacity=rows_n + 9)
    keys0, values0 = cache.keys.clone(), cache.values.clone()
    order = np.random.default_rng(1).permutation(rows_n)             # rows in any order, some of them padding
    sequence = [NONE if i % 50 == 49 else 0 for i in range(rows_n)]
    rows = Rows(cache, heads, sequence, order + 9, position=order * 3 + 100)
    rows.append(cache)
    check_append(cache, rows, keys0, values0, [0])


def test_append_far_positions():
    """Angles of positions past 2^24 and up to 2^32 - 1, where position x turns in f32 has no fraction left."""
    cache = Cache([0], page=16, kv=1, d=256, capacity=64)
    keys0, values0 = cache.keys.clone(), cache.values.clone()
    position = [0, 1, 32767, 131071, (1 << 24) + 1, (1 << 31) + 12345, (1 << 32) - 1]
    rows = Rows(cache, 4, [0] * 7, list(range(7)), position=position, base=1e6)
    rows.append(cache)
    check_append(cache, rows, keys0, values0, [0])


@pytest.mark.parametrize("gains,turns", [(False, True), (True, False), (False, False)])
def test_append_without_norm_or_rotation(gains, turns):
    cache = Cache([0, 0], page=16, kv=2, d=128, capacity=32, type="f16")
    keys0, values0 = cache.keys.clone(), cache.values.clone()
    rows = Rows(cache, 4, [0, 1, 1], [0, 3, 4], gains=gains, turns=turns)
    rows.append(cache)
    check_append(cache, rows, keys0, values0, [0, 0])


def test_append_saturates_f16_and_keeps_nan():
    torch = torch_cuda()
    cache = Cache([0], page=16, kv=1, d=64, capacity=16, type="f16")
    rows = Rows(cache, 1, [0], [2], gains=False, turns=False)
    v = rows.qkv[0, 128:]
    v[:6] = torch.tensor([1e6, -1e6, 65519.0, float("inf"), -float("inf"), float("nan")])
    rows.append(cache)
    p, o = cache.at(0, [2])
    got = cache.values[p, o, 0][0, :6].float().cpu().numpy()
    assert list(got[:5]) == [65504.0, -65504.0, 65504.0, 65504.0, -65504.0] and np.isnan(got[5])


def test_append_in_place_default_sequence_and_zero_row():
    """q_out = q (the fused matrix rotated where it lies), sequence NULL (row r is sequence r's), a row of zeros."""
    cache = Cache([4, 9, 0], page=8, kv=1, d=256, capacity=16)
    keys0, values0 = cache.keys.clone(), cache.values.clone()
    rows = Rows(cache, 4, [0, 1, 2], [4, 9, 0])
    rows.qkv[1] = 0.0
    want = rows.exact(cache)
    rows.desc.sequence = None
    rows.desc.q_out, rows.desc.q_out_stride = rows.qkv.data_ptr(), rows.qkv.shape[1]
    rows.append(cache)
    got = rows.qkv[:, :1024].reshape(3, 4, 256).double().cpu().numpy()
    assert (np.abs(got - want[0]) <= want[1]).all()
    rows.q_out = rows.qkv[:, :1024].clone()
    rows.exact = lambda c: want
    check_append(cache, rows, keys0, values0, cache.lengths)


def test_append_reports_bad_rows_and_pages_and_stores_the_rest():
    cache = Cache([0, 0], page=16, kv=1, d=64, capacity=32)
    for sequence, index, table, bit in [(2, 0, None, 4), (0, 32, None, 4), (1, 1 << 31, None, 4), (0, 3, (0, 0), 1)]:
        if table:
            bad = cache.table.clone()
            bad[table] = cache.pages
            cache.desc.page_table = bad.data_ptr()
        keys0, len0 = cache.keys.clone(), u32(cache.len).copy()
        rows = Rows(cache, 2, [sequence, 1], [index, 5])
        cache.error.zero_()
        rows.append(cache)
        assert int(cache.error) == bit
        p, o = cache.at(1, [5])
        keys0[p, o] = cache.keys[p, o]
        assert (keys0 == cache.keys).all()                           # the good row alone was stored
        assert list(u32(cache.len)) == [len0[0], 6]


# ------------------------------------------------------------------ bounds

@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("d,kv,order,page,lengths,first", [
    (256, 1, "nhd", 16, [0, 1, 15, 16, 17, 100], None), (128, 3, "hnd", 24, [50, 47, 48, 0], [49, 47, 0, 0]),
    (64, 2, "nhd", 1, [5, 3], [2, 3]), (256, 2, "hnd", 64, [300, 64], [128, 500]),
    (256, 1, "nhd", 150, [1000, 151], None), (64, 3, "hnd", 8, [3000] * 3 + [0] * 70 + [1, 700], None),
    (128, 2, "nhd", 16, [100] * 200, [99] * 200), (64, 1, "nhd", 600, [599, 601, 5000], None)])
def test_bounds(type, d, kv, order, page, lengths, first):
    torch = torch_cuda()
    cache = Cache(lengths, page=page, kv=kv, d=d, type=type, order=order, bounds=True).hide()
    before = torch.full_like(cache.bounds, 9.0)
    cache.bounds.copy_(before)
    bounds(cache, first)
    want = before.double()
    for s, n in enumerate(lengths):
        lo = 0 if first is None else first[s]
        for p in range((n + page - 1) // page):
            if lo < n and (p + 1) * page > lo:
                j = np.arange(p * page, min(n, (p + 1) * page))
                at, o = cache.at(s, j)
                k = cache.keys[at, o].double()
                want[at[0], :, 0], want[at[0], :, 1] = k.amin(0), k.amax(0)
    assert (cache.bounds.double() == want).all()
    assert int(cache.error) == 0


def test_bounds_nan_and_infinite_keys():
    torch = torch_cuda()
    cache = Cache([20], page=16, d=64, bounds=True)
    p, o = cache.at(0, [3, 5, 17])
    cache.keys[p[0], o[0], 0, 1] = float("nan")
    cache.keys[p[1], o[1], 0, 2] = float("inf")
    cache.keys[p[2], o[2], 0, 3] = -float("inf")
    bounds(cache)
    b = cache.bounds[p[0], 0]
    assert torch.isnan(b[:, 1]).all() and float(b[1, 2]) == math.inf and not torch.isnan(b[:, 2:]).any()
    assert float(cache.bounds[p[2], 0, 0, 3]) == -math.inf


# ------------------------------------------------------------------ select

@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("d,heads,kv,page,lengths,top,sink,recent", [
    (256, 4, 1, 16, [1000, 0, 1, 16, 700], 12, 1, 2), (128, 8, 2, 4, [2000, 1999], 100, 0, 0),
    (64, 15, 3, 8, [300, 50], 64, 3, 5), (256, 8, 1, 1, [5000], 257, 4, 4), (128, 2, 2, 16, [33, 90], 3, 1, 2),
    (64, 1, 1, 2, [20000], 1, 0, 0), (64, 5, 1, 1, [15000, 7], 300, 2, 2), (128, 16, 2, 1, [14000], 14000, 0, 9000)])
def test_select(type, d, heads, kv, page, lengths, top, sink, recent):
    cache = Cache(lengths, page=page, kv=kv, d=d, type=type, bounds=True, seed=top)
    bounds(cache)
    q = randn(len(lengths), heads, d, seed=3)
    blocks, scores = select(cache, q, top, sink, recent)
    blocks, scores = u32(blocks), scores.cpu().numpy()
    for s, n in enumerate(lengths):
        n = (n + page - 1) // page
        for h in range(kv):
            score = page_scores(cache, q, s, h)
            want = best(score, n, sink, recent, top)
            assert list(blocks[s, h, :len(want)]) == list(want)
            assert (blocks[s, h, len(want):] == NONE).all() and (scores[s, h, len(want):] == 0).all()
            # f32 accuracy: 32 additions of a chain within 2^-23 of the products' sizes each, 20 of f32 sums, the
            # parts of q to 2^-23 and to 2^-25 of its largest
            G = heads // kv
            x = q[s, h * G:(h + 1) * G].double().abs()
            size = (x.sum(-1) + d / 8 * x.amax(-1)).max() * cache.bounds.double().abs().max()
            assert np.abs(scores[s, h, :len(want)] - score[want]).max(initial=0) <= 88 * 2.0 ** -24 * float(size)


def test_select_ties_go_to_the_lower_page_and_nan_comes_first():
    torch = torch_cuda()
    cache = Cache([64 * 16], page=16, d=64, bounds=True)
    cache.bounds.fill_(1.0)
    q = torch.ones(1, 1, 64, device="cuda")
    assert list(u32(select(cache, q, 5, 1, 1)[0])[0, 0]) == [0, 1, 2, 3, 63]
    assert list(u32(select(cache, q, 4)[0])[0, 0]) == [0, 1, 2, 3]
    cache.bounds[int(cache.table_np[0, 40])] = 2.0
    cache.bounds[int(cache.table_np[0, 50]), 0, 1, 7] = float("nan")
    cache.bounds[int(cache.table_np[0, 50]), 0, 0, 7] = float("nan")
    blocks, scores = select(cache, q, 3)
    assert list(u32(blocks)[0, 0]) == [0, 40, 50]
    assert scores[0, 0, 0] == 64 and scores[0, 0, 1] == 128 and torch.isnan(scores[0, 0, 2])
    assert list(u32(select(cache, q, 1)[0])[0, 0]) == [50]


def test_select_reads_near_ties_in_64_bits():
    """Pages whose scores differ by less than f32 can hold: one key value 1 + 2^-10 among sums of 2^20."""
    torch = torch_cuda()
    cache = Cache([8 * 16], page=16, d=256, bounds=True)
    cache.bounds.zero_()
    q = torch.ones(1, 4, 256, device="cuda")
    for i in range(8):
        b = cache.bounds[int(cache.table_np[0, i]), 0]
        b[:, 0], b[:, 1] = 32768.0, 2.0 ** -10 * i
    q[:, :, 0] = 1024.0
    assert list(u32(select(cache, q, 3)[0])[0, 0]) == [5, 6, 7]


@pytest.mark.parametrize("pages,take", [(200, 50), (3000, 700), (13000, 1)])
def test_select_many_near_ties(pages, take):
    """Every page within f32's doubt of every other: a few, more than one CTA scores again, more than one CTA holds.
    Scores 2^20 + k 2^-10, k many times the same: the largest k first, then the lower page."""
    torch = torch_cuda()
    cache = Cache([pages * 2], page=2, d=64, bounds=True)
    k = np.random.default_rng(pages).integers(0, 40, pages)
    rows = torch.from_numpy(cache.table_np[0].astype(np.int64)).cuda()
    cache.bounds[rows] = torch.from_numpy(k / 1024.0).cuda().to(cache.dtype)[:, None, None, None]
    cache.bounds[:, :, :, 0] = 1024.0
    q = torch.zeros(1, 1, 64, device="cuda")
    q[0, 0, 0], q[0, 0, 1] = 1024.0, 1.0
    blocks, scores = select(cache, q, take)
    want = best(1048576.0 + k / 1024.0, pages, 0, 0, take)
    assert list(u32(blocks)[0, 0]) == list(want)
    assert (scores - 1048576.0).abs().max() <= 1.0


@pytest.mark.parametrize("capacity", [12000, 36000])
def test_select_largest_tables(capacity):
    """The most shared memory a selection takes: 8 bf16 heads of 256 over the longest tables, chosen by one CTA or by all."""
    cache = Cache([300, 7000], page=1, d=256, type="bf16", bounds=True, capacity=capacity, fill=0.0)
    cache.keys.copy_(randn(*cache.keys.shape, seed=1))
    bounds(cache)
    q = randn(2, 8, 256, seed=2)
    blocks = u32(select(cache, q, 500, 3, 3)[0])
    for s, n in enumerate(cache.lengths):
        want = best(page_scores(cache, q, s, 0), n, 3, 3, 500)
        assert list(blocks[s, 0, :len(want)]) == list(want)
    assert int(cache.error) == 0


@pytest.mark.parametrize("type,q_scale,bound", [
    ("bf16", 1e-5, 3e38), ("bf16", 1e-36, 3e38), ("bf16", 1.0, 3e38), ("bf16", 1e37, 1e-38), ("bf16", 1.0, 1e-38),
    ("bf16", 1e-6, 1e-38), ("bf16", 1e-41, 1.0), ("f16", 1e-41, 1.0), ("f16", 1e34, 6e4), ("f16", 1e34, 1e-6),
    ("f16", 1e-36, 1e-6)])
def test_select_at_the_ends_of_f32(type, q_scale, bound):
    """Sums that pass the largest f32 by the way, products and scores below the least normal one."""
    torch = torch_cuda()
    cache = Cache([600 * 16], page=16, d=256, type=type, bounds=True)
    b = torch.rand(cache.bounds.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 2 - 1
    cache.bounds.copy_(torch.sort(b, dim=2).values * bound)          # least keys below the greatest
    q = torch.clamp(randn(1, 3, 256, seed=6), -3, 3) * q_scale
    blocks, _ = select(cache, q, 60)
    assert list(u32(blocks)[0, 0]) == list(best(page_scores(cache, q, 0, 0), 600, 0, 0, 60))


def test_select_infinite_queries_and_bounds():
    """Scores of +-inf and NaN choose as their 64-bit values do."""
    torch = torch_cuda()
    cache = Cache([40 * 16], page=16, d=64, bounds=True)
    bounds(cache)
    q = randn(1, 2, 64)
    for change in ("q", "bounds"):
        if change == "q":
            q[0, 0, 3] = float("inf")
        else:
            q[0, 0, 3] = 1.0
            cache.bounds[int(cache.table_np[0, 7]), 0, 1, 3] = float("inf")
            cache.bounds[int(cache.table_np[0, 9]), 0, :, 5] = -float("inf")
        x, b = q[0].double()[:, None], cache.bounds[torch.from_numpy(cache.table_np[0].astype(np.int64)).cuda(), 0].double()
        score = torch.where(x < 0, x * b[:, 0], x * b[:, 1]).sum(-1)
        score = torch.where(torch.isnan(score).any(0), float("nan"), score.nan_to_num(-1e300, 1e308, -1e308).amax(0))
        assert list(u32(select(cache, q, 9)[0])[0, 0]) == list(best(score.cpu().numpy(), 40, 0, 0, 9))


@pytest.mark.parametrize("heads", [2, 8])
def test_select_a_query_head_of_nan(heads):
    """Every page scores NaN by the first head, whatever the others: the lowest pages, after what is forced."""
    cache = Cache([40 * 16], page=16, d=64, bounds=True)
    bounds(cache)
    q = randn(1, heads, 64)
    q[0, 0, 3] = float("nan")
    assert list(u32(select(cache, q, 9, 0, 2)[0])[0, 0]) == [0, 1, 2, 3, 4, 5, 6, 38, 39]


@pytest.mark.parametrize("take", [7, 8, 9, 10])
def test_select_bad_pages_with_an_infinite_bound(take):
    """Pages that are none come last in every case, and every word is written."""
    cache = Cache([11 * 16], page=16, d=64, bounds=True)
    bounds(cache)
    bad = cache.table.clone()
    bad[0, 4] = bad[0, 6] = bad[0, 9] = -1
    cache.desc.page_table = bad.data_ptr()
    cache.bounds[int(cache.table_np[0, 7]), 0, 1, 3] = float("inf")
    q = randn(1, 1, 64).abs()
    score = page_scores(cache, q, 0, 0)
    score[[4, 6, 9]] = -float("inf")
    blocks, _ = select(cache, q, take)
    assert list(u32(blocks)[0, 0]) == list(best(score, 11, 0, 0, take))
    assert int(cache.error) == 1


def test_select_bad_page_is_reported_and_last():
    cache = Cache([10 * 16], page=16, d=64, bounds=True)
    bounds(cache)
    bad = cache.table.clone()
    bad[0, 4] = -1
    cache.desc.page_table = bad.data_ptr()
    q = randn(1, 1, 64)
    blocks, _ = select(cache, q, 9)
    assert list(u32(blocks)[0, 0]) == [0, 1, 2, 3, 5, 6, 7, 8, 9]
    assert int(cache.error) == 1


# ------------------------------------------------------------------ attention

LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,page,order,window", [
    (4, 1, 16, "nhd", 0), (1, 1, 1, "nhd", 0), (2, 2, 24, "hnd", 0), (8, 1, 7, "hnd", 0), (6, 2, 64, "nhd", 20),
    (15, 3, 16, "hnd", 64), (12, 2, 5, "nhd", 1), (14, 2, 200, "hnd", 130)])
def test_attention_short(type, d, heads, kv, page, order, window):
    cache = Cache(LENGTHS, page=page, kv=kv, d=d, type=type, order=order, seed=heads).hide()
    q = randn(len(LENGTHS), heads, d, seed=heads, scale=2.0)
    scale = d ** -0.5
    got = attend(cache, q, scale, window)
    want, _, bound = attend_exact(cache, q, scale, window)
    check_out(got, want, bound)
    assert (got[0] == 0).all()
    assert int(cache.error) == 0


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,heads,kv,d,page,window", [
    ([5000], 4, 1, 256, 16, 0), ([33000], 4, 1, 256, 32, 0), ([3000, 0, 2999, 1, 4097], 8, 1, 256, 16, 0),
    ([2500] * 40 + [3] * 40, 4, 2, 128, 24, 512), ([9000, 20], 16, 2, 64, 64, 0), ([700] * 149, 1, 1, 64, 16, 0),
    ([1, 20000], 3, 1, 128, 13, 15000), ([4000] * 3, 12, 4, 256, 48, 0), ([600] * 70 + [0] * 10 + [5] * 20, 2, 1, 256, 16, 300),
    ([0] * 100 + [300] * 90 + [0, 1] * 60 + [5000] + [0] * 40, 4, 2, 64, 16, 0), ([0] * 300, 2, 1, 128, 16, 0)])
def test_attention_long(type, lengths, heads, kv, d, page, window):
    cache = Cache(lengths, page=page, kv=kv, d=d, type=type, seed=len(lengths)).hide()
    q = randn(len(lengths), heads, d, seed=1, scale=2.0)
    got = attend(cache, q, d ** -0.5, window)
    want, _, bound = attend_exact(cache, q, d ** -0.5, window)
    check_out(got, want, bound)
    again = attend(cache, q, d ** -0.5, window)
    assert (again == got).all()                                      # the same bits every time


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,page,lengths,window,decay", [
    (4, 1, 256, 16, [40, 0, 1000, 5], 0, 1.0), (8, 1, 128, 24, [300, 129], 100, 0.5), (3, 3, 64, 8, [2000], 0, 0.0),
    (10, 2, 256, 32, [5000, 1], 0, 1.0), (16, 2, 64, 16, [1000] * 30, 0, 1.0), (4, 1, 256, 16, [600, 0, 5] * 40, 300, 0.25),
    (5, 5, 128, 1, [90, 4000], 0, 1.0)])
def test_attention_weights(type, heads, kv, d, page, lengths, window, decay):
    torch = torch_cuda()
    cache = Cache(lengths, page=page, kv=kv, d=d, type=type, weights=True, seed=9).hide()
    if decay == 0.0:
        cache.weights.fill_(float("nan"))                            # the old value is not read
    q = randn(len(lengths), heads, d, seed=2, scale=2.0)
    old = cache.weights.clone().double()
    got = attend(cache, q, d ** -0.5, window, decay=decay)
    want, weights, bound = attend_exact(cache, q, d ** -0.5, window)
    check_out(got, want, bound)
    expect = old.clone()
    tol = torch.zeros_like(old)
    G = heads // kv
    for (s, h), (j, w) in weights.items():
        p, o = cache.at(s, j)
        base = decay * old[p, h, o] if decay else 0.0
        expect[p, h, o] = base + w
        x, k = q[s, h * G:(h + 1) * G].double(), cache.rows(cache.keys, s, j, h)
        delta = (d + 8) * 2.0 ** -24 * d ** -0.5 * (x.abs() @ k.abs().T).amax()
        tol[p, h, o] = w * (2 * delta + (len(j) + 64) * 2.0 ** -24) + 2.0 ** -23 * (w + base) + 1e-37
    same = torch.isnan(expect) & torch.isnan(cache.weights) | ((cache.weights.double() - expect).abs() <= tol)
    assert same.all(), float((cache.weights.double() - expect).abs().nan_to_num().max())


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,page,lengths,top,window", [
    (4, 1, 256, 16, [1000, 0, 5, 330], 8, 0), (8, 2, 128, 24, [3000, 100], 20, 0), (5, 1, 64, 8, [999], 200, 500),
    (4, 4, 256, 32, [2000, 31], 5, 0), (2, 1, 128, 1, [500, 7], 33, 0)])
def test_attention_selected(type, heads, kv, d, page, lengths, top, window):
    cache = Cache(lengths, page=page, kv=kv, d=d, type=type, weights=True, bounds=True, seed=4).hide()
    bounds(cache)
    q = randn(len(lengths), heads, d, seed=5, scale=2.0)
    blocks, _ = select(cache, q, top, sink=min(1, top), recent=1)
    old = cache.weights.clone()
    got = attend(cache, q, d ** -0.5, window, blocks=blocks, top=top, decay=1.0)
    want, weights, bound = attend_exact(cache, q, d ** -0.5, window, blocks)
    check_out(got, want, bound)
    assert int(cache.error) == 0
    touched = {}
    for (s, h), (j, w) in weights.items():
        p, o = cache.at(s, j)
        new = cache.weights[p, h, o].double() - old[p, h, o].double()
        assert (new - w).abs().max() < 1e-4 * (1 + w.abs().max())
        old[p, h, o] = cache.weights[p, h, o]
        touched[s, h] = len(j)
    assert (old == cache.weights).all()                              # nothing else was


def test_attention_selected_bad_blocks():
    """Unheld, descending and repeated pages, and one after a NONE, are left out and reported; NONE itself is skipped."""
    torch = torch_cuda()
    cache = Cache([10 * 16 - 3], page=16, d=64)
    q = randn(1, 2, 64)
    for words, good, bit in [([2, NONE, 5], [2], 8), ([2, 2, 5], [2, 5], 8), ([2, 5, 3], [2, 5], 8),
                             ([1, 10, NONE], [1], 8), ([NONE, NONE, NONE], [], 0)]:
        blocks = Cache.u32(np.array([[words]]))
        cache.error.zero_()
        got = attend(cache, q, 0.125, blocks=blocks, top=3)
        want, _, bound = attend_exact(cache, q, 0.125, blocks=Cache.u32(np.array([[good + [NONE] * (3 - len(good))]])))
        assert ((got.double() - want).abs() <= bound + 1e-30).all(), words
        assert int(cache.error) == bit, words


@pytest.mark.parametrize("q_scale", [1e-38, 1e-5, 1e-2])
def test_attention_largest_bf16_keys(q_scale):
    """Keys about the largest f32 and queries that leave the scores in range: a head whose products all have one sign."""
    torch = torch_cuda()
    cache = Cache([500], page=16, d=256, type="bf16")
    p, o = cache.at(0, [17])
    cache.keys[p, o, 0] = 3.3e38
    q = randn(1, 4, 256, seed=8).abs().clamp(0.5, 2.0) * q_scale
    q[0, 1] *= -1.0                                                   # the key's score far below the others' at 1e-2
    scale = 1e-4
    got = attend(cache, q, scale)
    want, _, _ = attend_exact(cache, q, scale)
    # the key's weight is 0 or 1, or every score's products sum to less than 0.2: delta <= 264 2^-24 0.2
    bound = cache.values.double().abs().max() * (2 * 264 * 0.2 + 500 + 64) * 2.0 ** -24
    assert ((got.double() - want).abs() <= bound).all()


def test_attention_peaky_tiny_and_huge_scores():
    """One key takes nearly all the weight over many small ones; queries of 1e-30 and 1e4; keys of the type's largest values."""
    torch = torch_cuda()
    for type in ("f16", "bf16"):
        cache = Cache([6000, 6000, 300, 300], page=16, d=256, type=type)
        q = randn(4, 4, 256, seed=8)
        p, o = cache.at(0, [17])
        cache.keys[p, o, 0] = (q[0, 0] * 1.3).to(cache.dtype)        # 16 to 20 above the others' scores in log2
        cache.values[p, o, 0] = 0.0
        q[1] *= 1e-30
        q[2] *= 1e4
        p, o = cache.at(3, [5])
        cache.keys[p, o, 0] = 65504.0 if type == "f16" else 3e30
        q[3] = q[3].abs() * -1.0                                     # that key's score is far below every other
        got = attend(cache, q, 1.0 / 16)
        want, _, bound = attend_exact(cache, q, 1.0 / 16)
        err = (got.double() - want).abs()
        assert torch.isfinite(got).all()
        assert (err <= bound).all(), (type, [float((err[s] / bound[s]).max()) for s in range(4)])
        small = want[0, 0].norm() / want[1, 0].norm()
        assert small < 0.5                                           # (sequence 0's output is its small weights' alone)
        assert float((got[0, 0].double() - want[0, 0]).norm() / want[0, 0].norm()) < 1e-4


def test_attention_infinite_scores_give_zero_weight_not_nan():
    """Keys whose every score is -inf in one warp's entries, then in all of them."""
    torch = torch_cuda()
    cache = Cache([64, 40], page=16, d=64, type="bf16", weights=True)
    q = torch.zeros(2, 1, 64, device="cuda")
    q[:, :, 0] = 1.0
    for s, js in ((0, range(0, 48)), (1, range(40))):
        p, o = cache.at(s, list(js))
        cache.keys[p, o, 0] = 0.0
        cache.keys[p, o, 0, 0] = -3e38
    got = attend(cache, q, 1e38)                                      # scale x product overflows to -inf
    assert torch.isfinite(got[0]).all()
    assert (got[1] == 0).all()


def test_attention_strided_rows_and_padded_cache():
    """q and out as parts of wider rows (what lies between is left as it was), cache rows with gaps between heads."""
    torch = torch_cuda()
    cache = Cache([100, 37], page=16, kv=2, d=128, pad=8)
    wide = randn(2, 4 * 128 + 64, seed=6)
    q = wide[:, :512].unflatten(1, (4, 128))
    store = torch.full((3, 600), 5.0, device="cuda")
    out = store[:2, 40:552].unflatten(1, (4, 128))
    attend(cache, q, 0.1, out=out)
    want, _, bound = attend_exact(cache, q, 0.1)
    check_out(out, want, bound)
    assert (store[2] == 5).all() and (store[:, :40] == 5).all() and (store[:, 552:] == 5).all()


def test_attention_reports_bad_pages_and_lengths():
    torch = torch_cuda()
    cache = Cache([100, 60], page=16, d=64)
    q = randn(2, 1, 64)
    table = cache.table.clone()
    table[0, 2] = cache.pages + 7
    cache.desc.page_table = table.data_ptr()
    got = attend(cache, q, 0.125)
    assert int(cache.error) == 1
    b = np.array([[[0, 1, 3, 4, 5, 6]], [[0, 1, 2, 3, NONE, NONE]]])
    want, _, bound = attend_exact(cache, q, 0.125, blocks=Cache.u32(b))
    check_out(got, want, bound)
    cache.desc.page_table = cache.table.data_ptr()
    cache.error.zero_()
    cache.len.copy_(Cache.u32(np.array([100, 1 << 31])))
    got = attend(cache, q, 0.125)
    assert int(cache.error) == 2
    cache.lengths[1] = cache.desc.table_stride * 16                  # cut to the table
    want, _, bound = attend_exact(cache, q, 0.125)
    check_out(got, want, bound)


def test_attention_far_offsets():
    """A pool past 2^32 elements: pages whose element offsets need 64 bits."""
    torch = torch_cuda()
    cache = Cache([64], page=16, d=256, type="f16")
    pages = (1 << 32) // (16 * 256) + 8
    pool = torch.empty(pages, 16, 1, 256, dtype=torch.float16, device="cuda")
    table = Cache.u32(np.array([[pages - 1, 3, pages - 5, 0]]))
    for i, p in enumerate(u32(table)[0]):
        pool[int(p)] = cache.keys[int(cache.table_np[0, i])]
    cache.desc.keys = cache.desc.values = pool.data_ptr()
    cache.desc.pages, cache.desc.page_table = pages, table.data_ptr()
    cache.values = cache.keys
    q = randn(1, 4, 256)
    got = attend(cache, q, 0.0625)
    want, _, bound = attend_exact(cache, q, 0.0625)
    check_out(got, want, bound)


# ------------------------------------------------------------------ eviction

@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("d,kv,page,to_page,order,lengths,budget,sink,recent", [
    (256, 1, 16, 16, "nhd", [1000, 0, 100, 64, 1], 64, 4, 10), (128, 3, 24, 7, "hnd", [500, 499], 200, 0, 0),
    (64, 2, 1, 16, "nhd", [40, 3], 1, 0, 0), (256, 1, 32, 32, "hnd", [9000], 4000, 16, 512),
    (64, 4, 16, 64, "nhd", [70, 300, 20], 128, 64, 64), (128, 1, 16, 16, "nhd", [40], 100, 3, 3),
    (64, 2, 16, 16, "nhd", [5000, 0, 40000, 3], 777, 0, 100)])
def test_evict(type, d, kv, page, to_page, order, lengths, budget, sink, recent):
    torch = torch_cuda()
    a = Cache(lengths, page=page, kv=kv, d=d, type=type, order=order, weights=True, seed=budget).hide()
    a.weights.copy_(torch.where(a.weights < 0.3, 0.0, (a.weights * 32).round() / 32))   # many equal weights
    b = Cache([min(n, budget) for n in lengths], page=to_page, kv=kv, d=d, type=type, order=order, weights=True, fill=7.0,
              seed=1)
    b.len.fill_(77)
    b.weights.fill_(7.0)
    keys0, weights0 = a.keys.clone(), a.weights.clone()
    kept = u32(evict(a, b, budget, sink, recent))
    want_k, want_v, want_w = (torch.full_like(t, 7.0) for t in (b.keys, b.values, b.weights))
    for s, n in enumerate(lengths):
        for h in range(kv):
            i = best(a.weight(s, np.arange(n), h).cpu().numpy(), n, sink, recent, budget)
            assert list(kept[s, h, :len(i)]) == list(i)
            assert (kept[s, h, len(i):] == NONE).all()
            (p, o), (tp, to) = a.at(s, i), b.at(s, np.arange(len(i)))
            want_k[tp, to, h], want_v[tp, to, h] = a.keys[p, o, h], a.values[p, o, h]
            want_w[tp, h, to] = a.weights[p, h, o]
    assert (b.keys == want_k).all() and (b.values == want_v).all() and (b.weights == want_w).all()
    assert list(u32(b.len)) == [min(n, budget) for n in lengths]
    assert (a.keys == keys0)[~torch.isnan(keys0)].all() and (a.weights == weights0).all()
    assert list(u32(a.len)) == lengths and int(a.error) == 0 and int(b.error) == 0


def test_evict_longest_table():
    """The most shared memory an eviction takes."""
    a = Cache([70000, 10], page=16, d=64, weights=True, capacity=400000)
    b = Cache([5000, 10], page=16, d=64, weights=True, seed=2)
    kept = u32(evict(a, b, 5000, 1, 1))
    want = best(a.weight(0, np.arange(70000), 0).cpu().numpy(), 70000, 1, 1, 5000)
    assert list(kept[0, 0]) == list(want)
    (p, o), (tp, to) = a.at(0, want), b.at(0, np.arange(5000))
    assert (b.keys[tp, to, 0] == a.keys[p, o, 0]).all() and (b.weights[tp, 0, to] == a.weights[p, 0, o]).all()


def test_evict_nan_weights_come_first_and_lengths_may_be_shared():
    torch = torch_cuda()
    a = Cache([50], page=16, d=64, weights=True)
    b = Cache([50], page=16, d=64, weights=True, seed=5)
    p, o = a.at(0, [30, 31, 10])
    a.weights[p, 0, o] = torch.tensor([float("nan"), float("inf"), -1.0], device="cuda")
    b.desc.lengths = a.desc.lengths
    kept = u32(evict(a, b, 2))
    assert list(kept[0, 0]) == [30, 31]
    assert int(a.len) == 2


def test_evict_reports_bad_pages():
    a = Cache([64], page=16, d=64, weights=True)
    b = Cache([64], page=16, d=64, weights=True, seed=5, fill=7.0)
    bad = b.table.clone()
    bad[0, 1] = b.pages
    b.desc.page_table = bad.data_ptr()
    evict(a, b, 32)
    assert int(b.error) == 1 and int(a.error) == 0
    bad = a.table.clone()
    bad[0, 0] = -1
    a.desc.page_table = bad.data_ptr()
    b.desc.page_table = b.table.data_ptr()
    kept = u32(evict(a, b, 48))
    assert int(a.error) == 1
    assert list(kept[0, 0]) == list(range(16, 64))                   # what cannot be read is kept last


# ------------------------------------------------------------------ together

def step(cache, rows, q_view, scale, top, blocks, scores, query, lib, s):
    _native.check(lib.fz_paged_append(cache.desc, rows.desc, s))
    _native.check(lib.fz_paged_bounds(cache.desc, None, s))
    _native.check(lib.fz_paged_select(cache.desc, q_view.data_ptr(), q_view.stride(0), q_view.shape[1], top, 1, 2,
                                      blocks.data_ptr(), scores.data_ptr(), s))
    _native.check(lib.fz_paged_attention(cache.desc, query, s))


@pytest.mark.parametrize("type,d,heads,kv", [("f16", 256, 4, 1), ("bf16", 128, 16, 2)])
def test_decode_steps_captured_and_replayed(type, d, heads, kv):
    """Decode steps as a server runs them: a step (append, bounds, select, attention of the selected pages with its
    weights) captured once and replayed with other rows, positions and lengths, then an eviction and attention over
    what it kept, all against the definitions."""
    torch = torch_cuda()
    lib = _native.load()
    lengths = [200, 0, 77]
    cache = Cache(lengths, page=16, kv=kv, d=d, type=type, capacity=256, weights=True, bounds=True, seed=3).hide()
    cache.weights.zero_()
    rows = Rows(cache, heads, [0, 1, 2], lengths, seed=1)
    top, S = 6, 3
    q_view = rows.q_out.view(S, heads, d)
    out = torch.empty(S, heads, d, device="cuda")
    blocks = torch.zeros(S, kv, top, dtype=torch.int32, device="cuda")
    scores = torch.zeros(S, kv, top, device="cuda")
    r = _native.PagedQuery()
    r.q, r.out, r.q_stride, r.out_stride = q_view.data_ptr(), out.data_ptr(), heads * d, heads * d
    r.heads, r.scale, r.decay, r.blocks, r.top = heads, d ** -0.5, 1.0, blocks.data_ptr(), top
    r.workspace_bytes = lib.fz_paged_attention_workspace(cache.desc, heads)
    workspace = torch.empty(max(256, r.workspace_bytes), dtype=torch.uint8, device="cuda")
    r.workspace = workspace.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(cache, rows, q_view, r.scale, top, blocks, scores, r, lib, torch.cuda.current_stream().cuda_stream)
    total = cache.weights.double()
    for t in range(4):
        fresh = Rows(cache, heads, [0, 1, 2], [n + t for n in lengths], seed=10 + t)
        rows.qkv.copy_(fresh.qkv)
        rows.dev[1].copy_(fresh.dev[1])
        rows.index = rows.position = fresh.index
        graph.replay()
        torch.cuda.synchronize()
        cache.lengths = [n + t + 1 for n in lengths]
        assert list(u32(cache.len)) == cache.lengths
        q, qe = rows.exact(cache)[:2]
        assert (np.abs(q_view.double().cpu().numpy() - q) <= qe).all()
        for s in range(S):
            n = (cache.lengths[s] + 15) // 16
            for h in range(kv):
                want = best(page_scores(cache, q_view, s, h), n, 1, 2, top)
                assert list(u32(blocks)[s, h, :len(want)]) == list(want)
        want, weights, bound = attend_exact(cache, q_view, r.scale, blocks=blocks)
        check_out(out, want, bound)
        for (s, h), (j, w) in weights.items():
            p, o = cache.at(s, j)
            total[p, h, o] += w
    for s in range(S):
        for h in range(kv):
            j = np.arange(cache.lengths[s])
            p, o = cache.at(s, j)
            assert (cache.weights[p, h, o].double() - total[p, h, o]).abs().max() < 1e-4
    to = Cache([min(n, 40) for n in cache.lengths], page=16, kv=kv, d=d, type=type, capacity=64, weights=True, seed=8).hide()
    kept = u32(evict(cache, to, 40, 2, 8))
    q = randn(S, heads, d, seed=77)
    got = attend(to, q, r.scale)
    want, _, bound = attend_exact(to, q, r.scale)
    check_out(got, want, bound)
    for s, n in enumerate(cache.lengths):
        if n <= 40:
            assert list(kept[s, 0, :n]) == list(range(n))
    assert int(cache.error) == 0


@pytest.mark.parametrize("window", [0, 37])
def test_many_steps_without_a_pause(window):
    """Forty steps queued at once (append, bounds, selection, attention of the selection with its weights, attention of
    everything): each sees what the ones before it left, lengths, bounds, selections and weights among it."""
    torch = torch_cuda()
    lib = _native.load()
    lengths, heads, kv, d, top, T = [150, 0, 33], 4, 1, 128, 5, 40
    cache = Cache(lengths, page=8, kv=kv, d=d, capacity=200, weights=True, bounds=True, seed=5).hide()
    cache.weights.zero_()
    s = stream()
    steps = []
    for t in range(T):
        rows = Rows(cache, heads, [0, 1, 2], [n + t for n in lengths], seed=100 + t)
        q = rows.q_out.view(3, heads, d)
        blocks, out, full = (torch.zeros(3, kv, top, dtype=torch.int32, device="cuda"), torch.empty_like(q), torch.empty_like(q))
        steps.append((rows, q, blocks, out, full))
    space = torch.empty(lib.fz_paged_attention_workspace(cache.desc, heads), dtype=torch.uint8, device="cuda")
    plain = _native.PagedKv.from_buffer_copy(cache.desc)
    plain.weights = None
    bounds(cache)
    torch.cuda.synchronize()
    first = None
    for rows, q, blocks, out, full in steps:
        _native.check(lib.fz_paged_append(cache.desc, rows.desc, s))
        _native.check(lib.fz_paged_bounds(cache.desc, first, s))
        first = rows.dev[1].data_ptr()                   # (this step's entries: the page's other ones are in its bounds' page)
        _native.check(lib.fz_paged_select(cache.desc, q.data_ptr(), heads * d, heads, top, 1, 1, blocks.data_ptr(), None, s))
        attend(cache, q, 0.1, window, blocks=blocks, top=top, decay=1.0, workspace=space, out=out)
        keep, cache.desc = cache.desc, plain
        attend(cache, q, 0.1, window, workspace=space, out=full)
        cache.desc = keep
    torch.cuda.synchronize()
    total = torch.zeros_like(cache.weights, dtype=torch.float64)
    for t, (rows, q, blocks, out, full) in enumerate(steps):
        cache.lengths = [n + t + 1 for n in lengths]
        want, weights, bound = attend_exact(cache, q, 0.1, window, blocks)
        check_out(out, want, bound)
        check_out(full, *[attend_exact(cache, q, 0.1, window)[i] for i in (0, 2)])
        for (i, h), (j, w) in weights.items():
            p, o = cache.at(i, j)
            total[p, h, o] += w
        for i in range(3):
            n = (cache.lengths[i] + 7) // 8
            got = u32(blocks)[i, 0]
            assert n - 1 in got[got != NONE] and 0 in got and len(set(got[got != NONE])) == min(top, n)
    assert (cache.weights.double() - total).abs().max() < T * 1e-5
    assert list(u32(cache.len)) == cache.lengths and int(cache.error) == 0


def test_two_graphs_share_a_workspace():
    """Graphs of two caches over one workspace, replayed in turn on one stream."""
    torch = torch_cuda()
    lib = _native.load()
    caches = [Cache([2000, 3], page=16, d=256, weights=True, seed=1).hide(), Cache([700] * 5, page=32, d=256, weights=True, seed=2)]
    qs = [randn(len(c.lengths), 4, 256, seed=i) for i, c in enumerate(caches)]
    outs = [torch.zeros_like(q) for q in qs]
    space = torch.empty(max(lib.fz_paged_attention_workspace(c.desc, 4) for c in caches), dtype=torch.uint8, device="cuda")
    graphs = []
    for c, q, out in zip(caches, qs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(c, q, 0.0625, decay=0.0, workspace=space, out=out)
        graphs.append(graph)
    for _ in range(10):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for c, q, out in zip(caches, qs, outs):
        want, weights, bound = attend_exact(c, q, 0.0625)
        check_out(out, want, bound)
        for (s, h), (j, w) in weights.items():
            p, o = c.at(s, j)
            assert (c.weights[p, h, o].double() - w).abs().max() < 1e-5


def test_two_streams_with_their_own_workspaces():
    torch = torch_cuda()
    caches = [Cache([3000, 10], page=16, d=256, seed=i).hide() for i in range(2)]
    qs = [randn(2, 4, 256, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    spaces = [torch.empty(_native.load().fz_paged_attention_workspace(c.desc, 4), dtype=torch.uint8, device="cuda") for c in caches]
    outs = [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                attend(caches[i], qs[i], 0.0625, workspace=spaces[i], out=outs[i])
    torch.cuda.synchronize()
    for i in range(2):
        want, _, bound = attend_exact(caches[i], qs[i], 0.0625)
        check_out(outs[i], want, bound)


def test_host_memory_is_refused():
    torch = torch_cuda()
    cache = Cache([5], page=16, d=64)
    q = torch.zeros(1, 1, 64)
    r = _native.PagedQuery()
    out = torch.zeros(1, 1, 64, device="cuda")
    r.q, r.out, r.heads, r.scale = q.data_ptr(), out.data_ptr(), 1, 1.0
    r.workspace_bytes = _native.load().fz_paged_attention_workspace(cache.desc, 1)
    w = torch.empty(r.workspace_bytes, dtype=torch.uint8, device="cuda")
    r.workspace = w.data_ptr()
    assert _native.load().fz_paged_attention(cache.desc, r, stream()) == 1
    assert b"current device" in _native.load().fz_last_error()

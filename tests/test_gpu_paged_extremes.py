"""The paged cache's operators at the ends of their ranges, against the definitions in 64 bits: scores and values about
the largest the types hold, queries of very unlike dimensions, pages that are none, and calls from two host threads."""
import threading

import numpy as np
import pytest

from frizzle_b200 import _native

from paged_cases import NONE, Cache, attend, attend_exact, bounds, evict, page_scores, select, torch_cuda

pytestmark = pytest.mark.gpu


def u32(t):
    return t.cpu().numpy().view(np.uint32)


def randn(*shape, seed=0):
    torch = torch_cuda()
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("score", [1.6777316e7, 2.0 ** 27, -(2.0 ** 30), 2.0 ** 40])
@pytest.mark.parametrize("heads,lengths", [(1, [1, 2, 40]), (8, [7000, 1, 0, 300])])
def test_weights_at_large_scores(type, score, heads, lengths):
    """Entries of one key share a sequence's weight evenly, whatever their score: heads / n each.  A weight's error: the
    sum of n ones (n 2^-24), its reciprocal, its product and the sum over the heads (a unit each)."""
    torch = torch_cuda()
    cache = Cache(lengths, page=16, d=64, type=type, weights=True).hide()
    for s, n in enumerate(lengths):
        p, o = cache.at(s, np.arange(n))
        cache.keys[p, o] = 0.0
        cache.keys[p, o, 0, 0] = 1024.0
    q = torch.zeros(len(lengths), heads, 64, device="cuda")
    q[:, :, 0] = score / 1024.0
    got = attend(cache, q, 1.0)
    want, _, _ = attend_exact(cache, q, 1.0)
    for s, n in enumerate(lengths):
        if not n:
            continue
        p, o = cache.at(s, np.arange(n))
        w = cache.weights[p, 0, o].double()
        assert ((w - heads / n).abs() <= heads / n * (n + heads + 4) * 2.0 ** -24).all(), (n, float(w[0]))
        # (the scores are equal, so the output's error is the weights')
        bound = cache.rows(cache.values, s, np.arange(n), 0).abs().max() * (n + 64) * 2.0 ** -24
        assert ((got[s].double() - want[s]).abs() <= bound).all()


@pytest.mark.parametrize("size", [3.3895e38, 1e38, 1.0, 1e-30])
@pytest.mark.parametrize("heads,d,lengths,alike", [
    (4, 256, [1, 2, 3, 16, 300], True), (8, 128, [5000, 2, 70], True), (3, 64, [40000], True), (4, 256, [9000, 33], False),
    (16, 64, [500] * 20, False)])
def test_bf16_values_of_any_size(size, heads, d, lengths, alike):
    """Values about the largest bf16 (an average of them is no larger) and about the least: `alike`, one key and one
    value a sequence, so that every partial sum grows with the entries; else random ones."""
    torch = torch_cuda()
    kv = heads // 8 or 1
    cache = Cache(lengths, page=16, kv=kv, d=d, type="bf16", weights=True, seed=d)
    if alike:
        cache.keys.fill_(0.5)
        sign = torch.where(torch.arange(d, device="cuda") % 3 == 0, -1.0, 1.0)
        cache.values.copy_((sign * size).to(cache.dtype).expand_as(cache.values))
    else:
        v = cache.values.float().clamp(-1.0, 1.0) * size
        cache.values.copy_(v)
    q = randn(len(lengths), heads, d, seed=3)
    got = attend(cache, q, d ** -0.5)
    want, weights, bound = attend_exact(cache, q, d ** -0.5)
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= bound).all()
    for (s, h), (j, w) in weights.items():
        p, o = cache.at(s, j)
        assert ((cache.weights[p, h, o].double() - w).abs() <= w * 1e-3).all()


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("heads,d", [(4, 256), (8, 64), (7, 128)])
@pytest.mark.parametrize("outlier", [1e4, 1e6, 1e8])
def test_attention_query_with_one_large_dimension(type, heads, d, outlier):
    """One dimension far above a head's others, which the keys have at zero: the others count as they do without it."""
    cache = Cache([1, 30, 700, 3000], page=16, d=d, type=type, seed=heads)
    cache.keys[..., 5] = 0.0
    q = randn(4, heads, d, seed=4) * 4.0
    q[..., 5] = outlier
    got = attend(cache, q, d ** -0.5)
    want, _, bound = attend_exact(cache, q, d ** -0.5)
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() / bound).max())


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_sums_of_products_within_the_units_assumed(type):
    """The tensor cores' f32 sums, which the margin of fz_paged_select and the bounds of attend_exact rest on: each of the
    32 additions of two steps of 16 products within 2^-23 of the products' sizes.  Products of every size that cancel to
    nothing, in the dimensions that one of the attention's sums takes, read from the weight of a key against one of
    zero: out[1] / out[0] = e^(scale q k)."""
    torch = torch_cuda()
    S, d, G = 400, 256, 4
    rng = np.random.default_rng(7)
    steps = np.r_[0:16, 64:80]                                       # step 0 and step 4, of one sum
    k = np.zeros((S, d))
    for s in range(S):
        spread = rng.choice([2, 8, 14, 20])                          # (f16 holds them all as normal numbers)
        half = (1.0 + rng.integers(0, 128, 16) / 128.0) * 2.0 ** (14 - rng.integers(0, spread + 1, 16)) * rng.choice([-1, 1], 16)
        k[s, steps] = rng.permutation(np.concatenate([half, -half]))
    cache = Cache([2] * S, page=2, d=d, type=type)
    cache.keys.zero_()
    cache.values.zero_()
    rows = torch.from_numpy(cache.table_np[:, 0].astype(np.int64)).cuda()
    cache.keys[rows, 1, 0] = torch.from_numpy(k).cuda().to(cache.dtype)
    cache.values[rows, 0, 0, 0] = 1.0
    cache.values[rows, 1, 0, 1] = 1.0
    assert (cache.keys[rows, 1, 0].double().cpu().numpy() == k).all()
    size = float(np.abs(k).sum(1).max())
    scale = 2.0 ** 18 / size                                         # a unit of 32 x 2^-23 of the largest size: 1
    out = attend(cache, torch.ones(S, G, d, device="cuda"), scale).double()
    score = torch.log(out[..., 1] / out[..., 0]).abs().amax(1).cpu().numpy()
    # (the weights are within 2^-20, and the factor of the scores within 2^-23 of their size)
    assert (score <= 32 * 2.0 ** -23 * np.abs(k).sum(1) * scale + 2.0 ** -19).all(), score.max()


# ------------------------------------------------------------------ selection

def check_scores(cache, q, blocks, scores, size=None):
    """Every listed page's score as the 64-bit sum rounded to f32 (half a unit, or half of 2^-149), that sum in any order:
    (d + 8) 2^-53 of the page's products' sizes."""
    torch = torch_cuda()
    blocks, scores = u32(blocks), scores.double().cpu().numpy()
    G = q.shape[1] // cache.kv
    for s, n in enumerate(cache.lengths):
        n = (n + cache.page - 1) // cache.page
        for h in range(cache.kv):
            at = blocks[s, h][blocks[s, h] != NONE].astype(np.int64)
            assert len(at) == min(n, blocks.shape[2]) and (scores[s, h, len(at):] == 0).all()
            want = page_scores(cache, q, s, h)[at]
            b = cache.bounds[torch.from_numpy(cache.table_np[s, at].astype(np.int64)).cuda(), h].double()
            x = q[s, h * G:(h + 1) * G].double()[:, None]
            sizes = torch.where(x < 0, x * b[:, 0], x * b[:, 1]).abs().sum(-1).amax(0).cpu().numpy()
            with np.errstate(invalid="ignore", over="ignore"):
                got, rounded = scores[s, h, :len(at)], want.astype(np.float32).astype(np.float64)
                near = np.abs(got - want) <= np.abs(want) * 2.0 ** -24 + sizes * (cache.d + 8) * 2.0 ** -53 + 2.0 ** -150
            same = near | (got == rounded) | (np.isnan(got) & np.isnan(want))
            assert same.all(), (s, h, got[~same][:4], want[~same][:4])


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("d,heads,kv,page,lengths,top,sink,recent,capacity", [
    (256, 4, 1, 16, [1000, 0, 1, 16, 700], 12, 1, 2, None), (128, 8, 2, 4, [2000, 1999], 100, 0, 0, None),
    (64, 15, 3, 8, [300, 50], 64, 3, 5, None), (256, 8, 1, 1, [5000], 257, 4, 4, None), (128, 2, 2, 16, [33, 90], 3, 1, 2, None),
    (64, 1, 1, 2, [20000], 1, 0, 0, None), (128, 16, 2, 1, [14000], 14000, 0, 9000, None), (256, 8, 4, 16, [9000] * 16, 200, 2, 8, None),
    (64, 5, 1, 1, [7000, 300], 500, 3, 3, 36000)])
def test_select_scores_are_the_64_bit_ones(type, d, heads, kv, page, lengths, top, sink, recent, capacity):
    cache = Cache(lengths, page=page, kv=kv, d=d, type=type, bounds=True, seed=top, capacity=capacity)
    bounds(cache)
    q = randn(len(lengths), heads, d, seed=3)
    check_scores(cache, q, *select(cache, q, top, sink, recent))


@pytest.mark.parametrize("pages,take", [(200, 50), (3000, 700), (13000, 5)])
def test_select_scores_of_near_ties(pages, take):
    """Scores that f32 sums cannot tell apart, but f32 can hold: 2^13 + k 2^-10."""
    torch = torch_cuda()
    cache = Cache([pages * 2], page=2, d=64, bounds=True)
    k = np.random.default_rng(pages).integers(0, 40, pages)
    rows = torch.from_numpy(cache.table_np[0].astype(np.int64)).cuda()
    cache.bounds[rows] = torch.from_numpy(k / 1024.0).cuda().to(cache.dtype)[:, None, None, None]
    cache.bounds[:, :, :, 0] = 1024.0
    cache.bounds[:, :, :, 2] = 1000.0
    q = torch.zeros(1, 1, 64, device="cuda")
    q[0, 0, 0], q[0, 0, 1], q[0, 0, 2] = 1024.0, 1.0, -1024 * 1.016
    blocks, scores = select(cache, q, take)
    check_scores(cache, q, blocks, scores)


@pytest.mark.parametrize("heads,lengths", [(2, [40 * 16]), (8, [3000 * 16]), (1, [5 * 16])])
def test_select_scores_with_bounds_infinite_on_the_side_not_picked(heads, lengths):
    """q < 0 with a greatest key of inf, q > 0 with a least of -inf: the score is finite."""
    torch = torch_cuda()
    cache = Cache(lengths, page=16, d=64, bounds=True)
    bounds(cache)
    q = randn(1, heads, 64)
    q[:, :, 3], q[:, :, 4] = -1.5, 2.0
    cache.bounds[int(cache.table_np[0, 2]), 0, 1, 3] = float("inf")
    cache.bounds[int(cache.table_np[0, 4]), 0, 0, 4] = -float("inf")
    cache.bounds[int(cache.table_np[0, 3]), 0, 1, 4] = float("inf")   # picked: inf
    for top in (len(cache.table_np[0]), 4):
        blocks, scores = select(cache, q, top)
        check_scores(cache, q, blocks, scores)
    blocks, scores = select(cache, q, 5, 5, 0)
    check_scores(cache, q, blocks, scores)
    assert torch.isfinite(scores[0, 0, [2, 4]]).all() and scores[0, 0, 3] == float("inf")


@pytest.mark.parametrize("type,q_scale,bound", [
    ("bf16", 1e-5, 3e38), ("bf16", 1e37, 1e-38), ("bf16", 1e-41, 1.0), ("bf16", 1e-41, 1e38), ("bf16", 1e38, 3e38), ("bf16", 1.0, 1e-39),
    ("f16", 1e-41, 1.0), ("f16", 1e34, 6e4), ("f16", 1e-36, 1e-6), ("f16", 1e-43, 1e-7)])
def test_select_scores_at_the_ends_of_f32(type, q_scale, bound):
    """Queries and bounds below the least normal f32, scores past the largest and below the least."""
    torch = torch_cuda()
    cache = Cache([600 * 16, 40], page=16, d=128, kv=2, type=type, bounds=True)
    b = torch.rand(cache.bounds.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 2 - 1
    cache.bounds.copy_(torch.sort(b, dim=2).values * bound)
    q = torch.clamp(randn(2, 6, 128, seed=6), -3, 3) * q_scale
    check_scores(cache, q, *select(cache, q, 60))


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_select_scores_of_queries_without_a_number(heads, value):
    """Beside pages whose bounds are infinite, NaN or zero."""
    cache = Cache([100 * 16], page=16, d=256, bounds=True)
    bounds(cache)
    q = randn(1, heads, 256)
    q[0, heads // 2, 3] = value
    cache.bounds[int(cache.table_np[0, 2]), 0, 1, 3] = float("inf")
    cache.bounds[int(cache.table_np[0, 4]), 0, :, 4] = float("nan")
    cache.bounds[int(cache.table_np[0, 6]), 0, :, 3] = 0.0
    check_scores(cache, q, *select(cache, q, 100))
    check_scores(cache, q, *select(cache, q, 9, 7, 1))


@pytest.mark.parametrize("pages,take", [(11, 11), (11, 6), (3000, 40)])
def test_select_score_of_a_page_that_is_none(pages, take):
    """-infinity, below every other page's."""
    cache = Cache([pages * 16], page=16, d=64, bounds=True)
    bounds(cache)
    bad = cache.table.clone()
    bad[0, 1] = bad[0, pages - 2] = -1
    cache.desc.page_table = bad.data_ptr()
    q = randn(1, 3, 64)
    blocks, scores = select(cache, q, take, 2, 3)
    at = u32(blocks)[0, 0]
    got = scores[0, 0].cpu().numpy()
    none = (at == 1) | (at == pages - 2)
    assert none.sum() == 2 and (got[none] == -np.inf).all() and np.isfinite(got[~none]).all()
    assert int(cache.error) == 1


# ------------------------------------------------------------------ eviction

@pytest.mark.parametrize("kv,lengths,bad,budget,sink,recent", [
    (1, [64], [0], 48, 4, 8), (2, [64, 50], [3, 0], 64, 0, 0), (1, [64], [0, 3], 20, 20, 0), (1, [64], [1, 3], 20, 0, 20),
    (2, [64, 3, 0], [0, 1, 2, 3], 64, 5, 5), (1, [20000, 100], [0, 700, 1249], 15000, 30, 30),
    (1, [20000, 64], [0, 700, 1249], 20000, 0, 0), (3, [9000], [562, 3], 9000, 16, 16), (1, [6000], [5], 100, 90, 10)])
def test_evict_leaves_out_entries_of_bad_pages(kv, lengths, bad, budget, sink, recent):
    """Logical pages `bad` of every sequence are no pages: what they hold is left out even where it is forced or the
    budget has room for it, so that every slot the new cache holds was written."""
    torch = torch_cuda()
    a = Cache(lengths, page=16, kv=kv, d=64, weights=True, seed=1)
    b = Cache([max(1, min(n, budget)) for n in lengths], page=16, kv=kv, d=64, weights=True, seed=2, fill=float("nan"))
    b.weights.fill_(float("nan"))
    b.len.fill_(77)
    table = u32(a.table).copy()
    table[:, [i for i in bad if i < table.shape[1]]] = a.pages + 5
    words = Cache.u32(table)
    a.desc.page_table = words.data_ptr()
    kept = u32(evict(a, b, budget, sink, recent))
    new = []
    for s, n in enumerate(lengths):
        good = np.array([i for i in range(n) if i // 16 not in bad], dtype=np.int64)
        take = min(budget, len(good))
        new.append(take)
        for h in range(kv):
            w = a.weight(s, good, h).double().cpu().numpy() if len(good) else np.zeros(0)
            forced = (good < sink) | (good + recent >= n)
            want = np.sort(good[np.lexsort((good, -w, ~forced))[:take]])
            assert np.array_equal(kept[s, h, :take], want), (s, h)
            assert (kept[s, h, take:] == NONE).all()
            if take:
                (p, o), (tp, to) = a.at(s, want), b.at(s, np.arange(take))
                assert (b.keys[tp, to, h] == a.keys[p, o, h]).all() and (b.values[tp, to, h] == a.values[p, o, h]).all()
                assert (b.weights[tp, h, to] == a.weights[p, h, o]).all()
    assert list(u32(b.len)) == new
    assert int(b.error) == 0 and int(a.error) == (1 if any(i * 16 < n for i in bad for n in lengths) else 0)
    q = randn(len(lengths), kv, 64)
    b.lengths = new
    got = attend(b, q, 0.125)
    want, _, bound = attend_exact(b, q, 0.125)
    assert ((got.double() - want).abs() <= bound).all()


# ------------------------------------------------------------------ host threads

@pytest.mark.parametrize("op", ["select", "evict"])
def test_two_host_threads_with_tables_of_unlike_widths(op):
    """Calls of caches with long and short tables from two threads at once: each call's need of shared memory is its own."""
    torch = torch_cuda()
    lib = _native.load()
    jobs = []
    for i, capacity in enumerate([20000, 4500] if op == "select" else [400000, 40000]):
        cache = Cache([4], page=1 if op == "select" else 4, d=64, weights=True, bounds=True, seed=i, capacity=capacity)
        to = Cache([4], page=4, d=64, weights=True, seed=9)
        q = randn(1, 1, 64)
        blocks, kept = (torch.zeros(1, 1, 4, dtype=torch.int32, device="cuda") for _ in range(2))
        jobs.append((cache, to, q, blocks, kept, torch.cuda.Stream()))
    torch.cuda.synchronize()
    failed = [[], []]
    start = threading.Barrier(2)

    def calls(i):
        cache, to, q, blocks, kept, st = jobs[i]
        start.wait()
        for _ in range(3000):
            if op == "select":
                status = lib.fz_paged_select(cache.desc, q.data_ptr(), 64, 1, 4, 0, 0, blocks.data_ptr(), None, st.cuda_stream)
            else:
                status = lib.fz_paged_evict(cache.desc, to.desc, 4, 0, 0, kept.data_ptr(), st.cuda_stream)
            if status:
                failed[i].append((status, lib.fz_last_error()))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed[0] and not failed[1], (len(failed[0]), len(failed[1]), (failed[0] + failed[1])[0])


def test_one_long_list_among_many_short_ones():
    """The long sequence's list is cut over the GPU whatever else the batch holds: 147 short ones beside it cost less than
    four times its own time (on one SM it takes more than twenty times that)."""
    torch = torch_cuda()

    def run(lengths):
        cache = long_cache(lengths)
        q = randn(len(lengths), 4, 256, seed=1)
        space = torch.empty(_native.load().fz_paged_attention_workspace(cache.desc, 4), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        best = float("inf")
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                attend(cache, q, 0.0625, workspace=space, out=out)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        want, _, bound = attend_exact(cache, q, 0.0625)
        assert ((out.double() - want).abs() <= bound).all()
        return best

    def long_cache(lengths):
        """Tables of 32,768 entries over a pool that holds only what the sequences do."""
        cache = Cache([max(lengths)] + [200], page=16, d=256, seed=4)
        table = np.full((len(lengths), 32768 // 16), 0xFFFFFFFF, dtype=np.uint32)
        for s, n in enumerate(lengths):
            table[s, :(n + 15) // 16] = cache.table_np[0 if n == max(lengths) else 1, :(n + 15) // 16]
        cache.lengths, cache.table_np = lengths, table
        cache.table, cache.len = Cache.u32(table), Cache.u32(np.array(lengths, dtype=np.uint32))
        cache.desc.page_table, cache.desc.lengths = cache.table.data_ptr(), cache.len.data_ptr()
        cache.desc.sequences, cache.desc.table_stride = len(lengths), table.shape[1]
        return cache

    alone = run([32768])
    among = run([200] * 70 + [32768] + [200] * 77)
    assert among < 4 * alone, (among, alone)

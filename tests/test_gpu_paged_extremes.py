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

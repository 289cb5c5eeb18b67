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

"""The paged key/value cache's operators as measured work: appending rows (QK-norm and rotation in the
same pass), the pages' key bounds, selecting pages for a query, attention of one new token, and
eviction by accumulated attention weight.

`own` False computes each in plain torch operations; True makes the library's calls.  Slots no
sequence holds carry NaN wherever an operator must not read them."""
import math
import random

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------ cases

def listed():
    return [
        # One decode step of 16 sequences, the most a batch of the engine takes, deep in a 32,768-token context.
        {"name": "append-step-16", "op": "append", "sequences": 16, "rows": 16, "length": 32768, "heads": 4, "kv": 1,
         "d": 256, "page": 32, "type": "f16", "order": "nhd", "mix": 1},
        # Prompt tokens of three sequences packed into one step, head-major pages.
        {"name": "append-prompt-4095", "op": "append", "sequences": 3, "rows": 4095, "length": 4096, "heads": 8, "kv": 2,
         "d": 256, "page": 16, "type": "bf16", "order": "hnd", "mix": 2},
        # After a decode step: only each sequence's last page changed.
        {"name": "bounds-step-16", "op": "bounds", "sequences": 16, "length": 32768, "kv": 1, "d": 256, "page": 64,
         "type": "f16", "order": "nhd", "last": True, "mix": 3},
        # After long prompts: every page.
        {"name": "bounds-prompt-32512", "op": "bounds", "sequences": 4, "length": 32512, "kv": 2, "d": 256, "page": 32,
         "type": "bf16", "order": "hnd", "last": False, "mix": 4},
        # One long conversation, small pages.
        {"name": "select-one-32512", "op": "select", "sequences": 1, "length": 32512, "heads": 4, "kv": 1, "d": 256,
         "page": 16, "type": "f16", "top": 128, "sink": 1, "recent": 4, "mix": 5},
        # A batch of conversations of different lengths.
        {"name": "select-batch-32768", "op": "select", "sequences": 16, "length": 32768, "heads": 8, "kv": 4, "d": 256,
         "page": 16, "type": "bf16", "top": 200, "sink": 2, "recent": 8, "mix": 6},
        # The first decode steps after a short prompt: latency.
        {"name": "attend-one-36", "op": "attend", "sequences": 1, "length": 36, "heads": 4, "kv": 1, "d": 256, "page": 16,
         "type": "f16", "order": "nhd", "window": 0, "top": 0, "weights": False, "mix": 7},
        # A window layer of a ragged batch, eight query heads a KV head, one sequence empty.
        {"name": "attend-window-64", "op": "attend", "sequences": 64, "length": 2500, "heads": 16, "kv": 2, "d": 128,
         "page": 24, "type": "bf16", "order": "hnd", "window": 512, "top": 0, "weights": False, "mix": 8},
        # Eight long contexts on a global layer, the attention weights kept for eviction.
        {"name": "attend-weights-8x32768", "op": "attend", "sequences": 8, "length": 32768, "heads": 4, "kv": 1, "d": 256,
         "page": 32, "type": "f16", "order": "nhd", "window": 0, "top": 0, "weights": True, "mix": 9},
        # The same contexts through selected pages.
        {"name": "attend-selected-8x2048", "op": "attend", "sequences": 8, "length": 32512, "heads": 4, "kv": 1, "d": 256,
         "page": 16, "type": "f16", "order": "nhd", "window": 0, "top": 128, "weights": False, "mix": 10},
        # One sequence cut back to a window's worth.
        {"name": "evict-one-1500", "op": "evict", "sequences": 1, "length": 1500, "kv": 1, "d": 256, "page": 32,
         "type": "f16", "order": "nhd", "budget": 512, "sink": 4, "recent": 64, "mix": 11},
        # A batch of long contexts cut back to an eighth.
        {"name": "evict-batch-32640", "op": "evict", "sequences": 8, "length": 32640, "kv": 2, "d": 256, "page": 16,
         "type": "bf16", "order": "hnd", "budget": 4080, "sink": 16, "recent": 512, "mix": 12},
    ]


def _between(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "bounds", "select", "attend", "attend", "evict"])
    kv = rng.choice([1, 1, 2, 4])
    case = {"op": op, "kv": kv, "d": rng.choice([64, 128, 256, 256]), "page": rng.choice([8, 16, 24, 32, 64]),
            "type": rng.choice(["f16", "bf16"]), "mix": rng.randrange(1, 1 << 20)}
    if op != "select":
        case["order"] = rng.choice(["nhd", "hnd"])
    if op in ("append", "select", "attend"):
        case["heads"] = kv * rng.choice([1, 2, 3, 4, 8] if kv < 4 else [1, 2])
    case["length"] = _between(rng, 4, 32768)
    most = {"append": 64, "bounds": 16, "select": 16, "attend": 64, "evict": 16}[op]
    case["sequences"] = _between(rng, 1, max(1, min(most, 8 * 32768 // (case["length"] * kv))))
    if op == "append":
        case["rows"] = _between(rng, case["sequences"], 4095 if kv < 4 else 2047)
    elif op == "bounds":
        case["last"] = rng.random() < 0.3
    elif op == "select":
        case["top"] = _between(rng, 1, 256)
        case["sink"] = rng.randrange(0, max(1, min(4, case["top"] // 2)))
        case["recent"] = rng.randrange(0, max(1, min(8, case["top"] // 2)))
    elif op == "attend":
        case["window"] = rng.choice([0, 0, _between(rng, 1, case["length"])])
        case["top"] = rng.choice([0, 0, _between(rng, 1, min(256, 3 + _pages(case["length"], case["page"])))])
        case["weights"] = rng.random() < 0.4
    else:
        case["budget"] = _between(rng, 1, max(1, case["length"] // 3))
        case["sink"] = rng.randrange(0, max(1, case["budget"] // 4))
        case["recent"] = rng.randrange(0, max(1, case["budget"] // 2))
    return case


def _lengths(case):
    """Tokens each sequence holds: the first the whole length, the others spread over 40 to 100 % of it,
    every 16th empty (a padded batch)."""
    r = random.Random(case["mix"])
    n = [case["length"]] + [max(1, int(case["length"] * r.uniform(0.4, 1.0))) for _ in range(case["sequences"] - 1)]
    return [0 if s % 16 == 15 else x for s, x in enumerate(n)]


def _starts(case):
    """Where each sequence's appended rows begin, and how many it appends."""
    S, R = case["sequences"], case["rows"]
    share = [R // S + (1 if s < R % S else 0) for s in range(S)]
    r = random.Random(case["mix"])
    return [r.randrange(0, case["length"]) for _ in range(S)], share


def _pages(n, page):
    return (n + page - 1) // page


# ------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float16 if case["type"] == "f16" else torch.bfloat16


def _pool(case, pages, fill, seed, order):
    """A pool of pages, [page][slot][head][d] ("nhd") or [page][head][slot][d] ("hnd") in memory, as the
    logical [page][slot][head][d]."""
    P, kv, d = case["page"], case["kv"], case["d"]
    shape = (pages, P, kv, d) if order == "nhd" else (pages, kv, P, d)
    if fill == "zeros":
        t = torch.zeros(shape, dtype=_dtype(case), device=DEVICE)
    else:
        g = torch.Generator(device=DEVICE).manual_seed(seed)
        t = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(_dtype(case))
    return t if order == "nhd" else t.permute(0, 2, 1, 3)


def _table(case, lengths, seed, spare=3):
    """Each sequence's pages: a shuffle of the pool, -1 past the ones it holds."""
    counts = [_pages(n, case["page"]) for n in lengths]
    width, total = max(1, max(counts)), sum(counts)
    order = torch.randperm(total + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    return table.to(DEVICE), total + spare


def _hide(case, st, lengths):
    """NaN in the slots past each sequence's end."""
    P = case["page"]
    for s, n in enumerate(lengths):
        if n % P:
            p = int(st["table"][s, n // P])
            st["keys"][p, n % P:] = float("nan")
            st["values"][p, n % P:] = float("nan")


def _kv(st, case, keys, values, table, lengths, pages, weights=None, bounds=None):
    """The library's description of the cache, which a user's program keeps beside it."""
    from frizzle_b200 import _native
    kv = _native.PagedKv()
    if keys is not None:
        kv.keys, kv.values = keys.data_ptr(), values.data_ptr()
        kv.page_stride, kv.slot_stride, kv.head_stride = keys.stride(0), keys.stride(1), keys.stride(2)
    kv.page_table, kv.lengths = table.data_ptr(), lengths.data_ptr()
    kv.weights = weights.data_ptr() if weights is not None else None
    kv.bounds = bounds.data_ptr() if bounds is not None else None
    kv.error = st["error"].data_ptr()
    kv.sequences, kv.table_stride, kv.pages = table.shape[0], table.shape[1], pages
    kv.page_slots, kv.kv_heads, kv.head_dim = case["page"], case["kv"], case["d"]
    kv.type = 0 if case["type"] == "f16" else 1
    return kv


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    op, P, kv, d, S = case["op"], case["page"], case["kv"], case["d"], case["sequences"]
    st = {"case": case, "error": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    if op == "append":
        starts, share = _starts(case)
        ends = [a + n for a, n in zip(starts, share)]
        st["table"], pages = _table(case, ends, seed)
        st["keys"] = _pool(case, pages, "zeros", seed, case["order"])
        st["values"] = _pool(case, pages, "zeros", seed, case["order"])
        st["lengths"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        H, R = case["heads"], case["rows"]
        st["qkv"] = randn(R, (H + 2 * kv) * d) * 3.0
        st["q_gain"], st["k_gain"] = 1.0 + 0.3 * randn(d), 1.0 + 0.3 * randn(d)
        turns = [10000.0 ** (-2.0 * i / d) / (2.0 * math.pi) for i in range(d // 2)]
        st["turns"] = torch.tensor(turns, dtype=torch.float64, device=DEVICE)
        st["sequence"] = torch.tensor([s for s in range(S) for _ in range(share[s])], dtype=torch.int32, device=DEVICE)
        st["index"] = torch.tensor([starts[s] + i for s in range(S) for i in range(share[s])], dtype=torch.int32,
                                   device=DEVICE)
        st["q_out"] = torch.empty(R, H * d, dtype=torch.float32, device=DEVICE)
        if own:
            from frizzle_b200 import _native
            st["kv"] = _kv(st, case, st["keys"], st["values"], st["table"], st["lengths"], pages)
            r = _native.PagedRows()
            qkv, w = st["qkv"].data_ptr(), (H + 2 * kv) * d
            r.q, r.k, r.v, r.q_out = qkv, qkv + H * d * 4, qkv + (H + kv) * d * 4, st["q_out"].data_ptr()
            r.q_stride = r.k_stride = r.v_stride = w
            r.q_out_stride = H * d
            r.q_gain, r.k_gain, r.turns = st["q_gain"].data_ptr(), st["k_gain"].data_ptr(), st["turns"].data_ptr()
            r.sequence, r.index = st["sequence"].data_ptr(), st["index"].data_ptr()
            r.rows, r.heads, r.eps = R, H, EPS
            st["rows"] = r
        return st

    lengths = _lengths(case)
    st["table"], pages = _table(case, lengths, seed)
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    if op == "select":
        # Bounds of random keys: the least and the greatest of a page's, which differ from page to page.
        mid, half = randn(pages + 1, kv, 1, d) * 0.7, randn(pages + 1, kv, 1, d).abs() + 0.3
        st["bounds"] = torch.cat([mid - half, mid + half], 2).to(_dtype(case)).contiguous()
        st["q"] = randn(S, case["heads"] * d) * 2.0
        st["blocks"] = torch.empty(S, kv, case["top"], dtype=torch.int32, device=DEVICE)
        st["scores"] = torch.empty(S, kv, case["top"], dtype=torch.float32, device=DEVICE)
        if own:
            st["kv"] = _kv(st, case, None, None, st["table"], st["lengths"], pages, bounds=st["bounds"])
        return st

    st["keys"] = _pool(case, pages, "randn", seed + 1, case["order"])
    st["values"] = _pool(case, pages, "randn", seed + 2, case["order"])
    _hide(case, st, lengths)
    if op == "bounds":
        st["bounds"] = torch.zeros(pages + 1, kv, 2, d, dtype=_dtype(case), device=DEVICE)
        st["first"] = torch.tensor([max(0, n - 1) if case["last"] else 0 for n in lengths], dtype=torch.int32, device=DEVICE)
        if own:
            st["kv"] = _kv(st, case, st["keys"], st["values"], st["table"], st["lengths"], pages, bounds=st["bounds"])
        return st

    # Weights as a heavy-tailed sum leaves them, a tenth of the entries never looked at (ties at zero).
    w = torch.exp(2.0 * randn(pages + 1, kv, P))
    st["weights"] = torch.where(torch.rand(pages + 1, kv, P, generator=g, device=DEVICE) < 0.1, torch.zeros_like(w), w)
    if op == "attend":
        H = case["heads"]
        st["weights"].zero_()
        st["q"] = randn(S, H * d) * 2.0
        st["out"] = torch.empty(S, H * d, dtype=torch.float32, device=DEVICE)
        if case["top"]:
            held = torch.tensor([_pages(n, P) for n in lengths], device=DEVICE)[:, None, None]
            width = st["table"].shape[1]
            score = torch.rand(S, kv, width, generator=g, device=DEVICE)
            score = torch.where(torch.arange(width, device=DEVICE) < held, score, -1.0)
            take = min(case["top"], width)
            best, at = score.topk(take, -1)
            at = torch.where(best < 0, torch.full_like(at, 1 << 30), at).sort(-1).values
            at = torch.where(at == 1 << 30, -1, at).to(torch.int32)
            st["blocks"] = torch.full((S, kv, case["top"]), -1, dtype=torch.int32, device=DEVICE)
            st["blocks"][:, :, :take] = at
        if own:
            from frizzle_b200 import _native
            lib = _native.load()
            st["kv"] = _kv(st, case, st["keys"], st["values"], st["table"], st["lengths"], pages,
                           weights=st["weights"] if case["weights"] else None)
            r = _native.PagedQuery()
            r.q, r.out, r.q_stride, r.out_stride = st["q"].data_ptr(), st["out"].data_ptr(), H * d, H * d
            r.blocks = st["blocks"].data_ptr() if case["top"] else None
            r.top, r.heads, r.window = case["top"], H, case["window"]
            r.scale, r.decay = 1.0 / math.sqrt(d), 0.0
            r.workspace_bytes = lib.fz_paged_attention_workspace(st["kv"], H)
            st["workspace"] = torch.empty(max(16, r.workspace_bytes), dtype=torch.uint8, device=DEVICE)
            r.workspace = st["workspace"].data_ptr()
            st["query"] = r
        return st

    kept = [min(n, case["budget"]) for n in lengths]
    st["to_table"], to_pages = _table(case, kept, seed + 3)
    st["to_keys"] = _pool(case, to_pages + 1, "zeros", seed, case["order"])
    st["to_values"] = _pool(case, to_pages + 1, "zeros", seed, case["order"])
    st["to_weights"] = torch.zeros(to_pages + 1, kv, P, dtype=torch.float32, device=DEVICE)
    st["to_lengths"] = torch.zeros(S, dtype=torch.int32, device=DEVICE)
    st["kept"] = torch.empty(S, kv, case["budget"], dtype=torch.int32, device=DEVICE)
    if own:
        st["kv"] = _kv(st, case, st["keys"], st["values"], st["table"], st["lengths"], pages, weights=st["weights"])
        st["to"] = _kv(st, case, st["to_keys"], st["to_values"], st["to_table"], st["to_lengths"], to_pages,
                       weights=st["to_weights"])
    return st


# ------------------------------------------------------------------ one pass

def run(st):
    op = st["case"]["op"]
    if own:
        _calls(st)
    else:
        {"append": _append, "bounds": _bounds, "select": _select, "attend": _attend, "evict": _evict}[op](st)
    if op == "append":
        return {"q": st["q_out"], "keys": st["keys"], "values": st["values"], "lengths": st["lengths"]}
    if op == "bounds":
        return {"bounds": st["bounds"][:-1]}
    if op == "select":
        return {"blocks": st["blocks"], "scores": st["scores"]}
    if op == "attend":
        return {"out": st["out"], "weights": st["weights"][:-1]} if st["case"]["weights"] else {"out": st["out"]}
    return {"kept": st["kept"], "lengths": st["to_lengths"], "keys": st["to_keys"][:-1], "values": st["to_values"][:-1],
            "weights": st["to_weights"][:-1]}


def _calls(st):
    from frizzle_b200 import _native
    lib, case = _native.load(), st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    op = case["op"]
    if op == "append":
        status = lib.fz_paged_append(st["kv"], st["rows"], stream)
    elif op == "bounds":
        status = lib.fz_paged_bounds(st["kv"], st["first"].data_ptr(), stream)
    elif op == "select":
        status = lib.fz_paged_select(st["kv"], st["q"].data_ptr(), case["heads"] * case["d"], case["heads"], case["top"],
                                     case["sink"], case["recent"], st["blocks"].data_ptr(), st["scores"].data_ptr(), stream)
    elif op == "attend":
        status = lib.fz_paged_attention(st["kv"], st["query"], stream)
    else:
        status = lib.fz_paged_evict(st["kv"], st["to"], case["budget"], case["sink"], case["recent"],
                                    st["kept"].data_ptr(), stream)
    _native.check(status)


def _store(x, like):
    """f32 to the cache's type: f16 saturates at its largest value."""
    return x.clamp(-65504.0, 65504.0).to(like.dtype) if like.dtype == torch.float16 else x.to(like.dtype)


def _append(st):
    c = st["case"]
    H, kv, d, P, R = c["heads"], c["kv"], c["d"], c["page"], c["rows"]
    q, k, v = (x.reshape(R, -1, d) for x in st["qkv"].split([H * d, kv * d, kv * d], 1))
    turn = st["index"].double()[:, None] * st["turns"]
    angle = 2.0 * math.pi * (turn - turn.round())
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, gain):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    st["q_out"].copy_(rotated(q, st["q_gain"]).reshape(R, H * d))
    seq, index = st["sequence"].long(), st["index"].long()
    page, slot = st["table"][seq, index // P].long(), index % P
    st["keys"][page, slot] = _store(rotated(k, st["k_gain"]), st["keys"])
    st["values"][page, slot] = _store(v, st["values"])
    st["lengths"].scatter_reduce_(0, seq, st["index"] + 1, "amax")


def _bounds(st):
    c, b = st["case"], st["bounds"]
    S, P, width = c["sequences"], c["page"], st["table"].shape[1]
    n = st["lengths"][:, None].long()
    p = ((n - 1) // P).clamp_min(0) if c["last"] else torch.arange(width, device=DEVICE).expand(S, width)
    page = torch.gather(st["table"].long(), 1, p)
    k = st["keys"][page.clamp_min(0)].float()                                         # [S][pages][slot][head][d]
    held = (p[..., None] * P + torch.arange(P, device=DEVICE) < n[..., None])[..., None, None]
    low, high = torch.where(held, k, math.inf).amin(2), torch.where(held, k, -math.inf).amax(2)
    touched = (p * P < n) & ((p + 1) * P > st["first"][:, None])
    b[torch.where(touched, page, b.shape[0] - 1)] = torch.stack([low, high], 3).to(b.dtype)


def _ranked(score, held, forced, take):
    """The `take` best of the last axis, ascending, -1 past the ones held: forced ones first, then the
    largest scores, ties to the lower index."""
    n = score.shape[-1]
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices
    tier = torch.where(forced, 2, 1) * held
    tier = torch.gather(tier.expand(score.shape), -1, best)
    best = torch.gather(best, -1, torch.sort(tier, dim=-1, descending=True, stable=True).indices)[..., :take]
    ok = torch.gather(held.expand(score.shape), -1, best)
    best = torch.where(ok, best, n).sort(-1).values
    return torch.where(best == n, -1, best).to(torch.int32)


def _select(st):
    c = st["case"]
    S, kv, d, G = c["sequences"], c["kv"], c["d"], c["heads"] // c["kv"]
    q = st["q"].double().reshape(S, kv, G, d)
    b = st["bounds"][st["table"].long().clamp_min(0)].double().permute(0, 2, 3, 4, 1)  # [S][kv][2][d][pages]
    score = torch.matmul(q.clamp(max=0.0), b[:, :, 0]) + torch.matmul(q.clamp(min=0.0), b[:, :, 1])
    score = score.amax(2)
    n = ((st["lengths"] + c["page"] - 1) // c["page"])[:, None, None]
    p = torch.arange(score.shape[-1], device=DEVICE)
    best = _ranked(score, p < n, (p < c["sink"]) | (p >= n - c["recent"]), c["top"])
    st["blocks"].fill_(-1)
    st["blocks"][..., :best.shape[-1]] = best
    st["scores"].zero_()
    chosen = torch.gather(score, -1, best.long().clamp_min(0))
    st["scores"][..., :best.shape[-1]] = torch.where(best >= 0, chosen, 0.0).float()


def _attend(st):
    c = st["case"]
    S, kv, d, P, G = c["sequences"], c["kv"], c["d"], c["page"], c["heads"] // c["kv"]
    n, table = st["lengths"][:, None, None].long(), st["table"].long()[:, None].expand(S, kv, -1)
    width = table.shape[2] * P
    if c["top"]:
        chosen = st["blocks"].long().repeat_interleave(P, 2)                          # [S][kv][entry]
        j = chosen.clamp_min(0) * P + torch.arange(P, device=DEVICE).repeat(c["top"])
        valid = (chosen >= 0) & (j < n)
        if c["window"]:
            valid = valid & (j >= n - c["window"])
    else:
        most = min(width, c["window"] or width)
        j = ((n - most).clamp_min(0) + torch.arange(most, device=DEVICE)).expand(S, kv, most)
        valid = j < n
    j = j.clamp_max(width - 1)
    page, slot = torch.gather(table, 2, j // P).clamp_min(0), j % P
    head = torch.arange(kv, device=DEVICE)[None, :, None].expand_as(page)
    k = torch.where(valid[..., None], st["keys"][page, slot, head].float(), 0.0)
    v = torch.where(valid[..., None], st["values"][page, slot, head].float(), 0.0)
    s = torch.matmul(st["q"].reshape(S, kv, G, d), k.transpose(2, 3)) / math.sqrt(d)
    s = torch.where(valid[:, :, None], s, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3e38))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-38)
    st["out"].copy_(torch.matmul(p, v).reshape(S, c["heads"] * d))
    if c["weights"]:
        st["weights"][torch.where(valid, page, st["weights"].shape[0] - 1), head, slot] = p.sum(2)


def _evict(st):
    c = st["case"]
    S, kv, P, B = c["sequences"], c["kv"], c["page"], c["budget"]
    table, to_table = (t.long()[:, None].expand(S, kv, -1) for t in (st["table"], st["to_table"]))
    head = torch.arange(kv, device=DEVICE)[None, :, None]
    n = st["lengths"][:, None, None].long()
    j = torch.arange(table.shape[2] * P, device=DEVICE)
    score = st["weights"][table[..., j // P].clamp_min(0), head, j % P]
    best = _ranked(score, j < n, (j < c["sink"]) | (j >= n - c["recent"]), B)
    st["kept"].fill_(-1)
    st["kept"][..., :best.shape[-1]] = best
    st["to_lengths"].copy_(st["lengths"].clamp_max(B))
    src, t = best.long().clamp_min(0), torch.arange(best.shape[-1], device=DEVICE)
    page, slot, h = torch.gather(table, 2, src // P).clamp_min(0), src % P, head.expand_as(src)
    to_page = to_table[..., (t // P).clamp_max(to_table.shape[2] - 1)]
    to = (torch.where(best >= 0, to_page, st["to_weights"].shape[0] - 1), h, (t % P).expand_as(src))
    st["to_keys"][to[0], to[2], h] = st["keys"][page, slot, h]
    st["to_values"][to[0], to[2], h] = st["values"][page, slot, h]
    st["to_weights"][to] = st["weights"][page, h, slot]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op, kv, d, P = case["op"], case["kv"], case["d"], case["page"]
    row = kv * d * 2                                     # one entry's keys, bytes
    if op == "append":
        H, R = case["heads"], case["rows"]
        return {"bytes": R * ((H + 2 * kv) * d * 4 + H * d * 4 + 2 * row + 8), "flops": R * (H + kv) * d * 7}
    lengths = _lengths(case)
    pages = [_pages(n, P) for n in lengths]
    if op == "bounds":
        read = [n - (p - 1) * P if n and case["last"] else n for n, p in zip(lengths, pages)]
        made = [min(p, 1) if case["last"] else p for p in pages]
        return {"bytes": sum(read) * row + sum(made) * 2 * row, "flops": 2 * sum(read) * kv * d}
    if op == "select":
        H = case["heads"]
        return {"bytes": sum(pages) * (2 * row + 4) + len(lengths) * (H * d * 4 + kv * case["top"] * 4),
                "flops": 2 * sum(pages) * H * d}
    if op == "attend":
        H, S = case["heads"], case["sequences"]
        n = [min(x, case["window"]) if case["window"] else x for x in lengths]
        n = [min(x, case["top"] * P) if case["top"] else x for x in n]
        if case["top"] and case["window"]:               # selected pages are spread evenly over the sequence's
            n = [x * min(1.0, case["window"] / max(1, y)) for x, y in
                 zip([min(y, case["top"] * P) for y in lengths], lengths)]
        moved = sum(n) * (2 * row + (4 * kv if case["weights"] else 0)) + 2 * S * H * d * 4
        return {"bytes": int(moved), "flops": int(4 * sum(n) * H * d)}
    kept = [min(n, case["budget"]) for n in lengths]
    return {"bytes": sum(lengths) * kv * 4 + sum(kept) * (4 * row + kv * 8), "flops": 0}


# ------------------------------------------------------------------ the definitions, in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    op, P, kv, d = case["op"], case["page"], case["kv"], case["d"]
    f64 = {k: v.double() for k, v in st.items() if k in ("keys", "values", "qkv", "q", "q_gain", "k_gain")}
    if op == "append":
        H, R = case["heads"], case["rows"]
        x = f64["qkv"].reshape(R, H + 2 * kv, d)
        z = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                        2 * math.pi * torch.remainder(st["index"].double()[:, None] * st["turns"], 1.0))

        def turned(y, gain):
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * gain
            y = torch.complex(y[..., :d // 2], y[..., d // 2:]) * z[:, None]
            return torch.cat([y.real, y.imag], -1)

        q = turned(x[:, :H], f64["q_gain"]).reshape(R, H * d)
        k, v = turned(x[:, H:H + kv], f64["k_gain"]), x[:, H + kv:]
        s, i = st["sequence"].long(), st["index"].long()
        at = (st["table"][s, i // P].long(), i % P)
        keys, values = f64["keys"], f64["values"]
        keys[at], values[at] = k, v
        lengths = None
        return {"q": q, "keys": keys, "values": values, "lengths": lengths}
    if op == "attend":
        H, G = case["heads"], case["heads"] // kv
        out = torch.zeros(case["sequences"], H, d, dtype=torch.float64, device=DEVICE)
        weights = st["weights"].double()
        for s, n in enumerate(_lengths(case)):
            for h in range(kv if n else 0):
                j = torch.arange(n, device=DEVICE)
                if case["top"]:
                    blocks = st["blocks"][s, h]
                    j = j[torch.isin(j // P, blocks[blocks >= 0].long())]
                if case["window"]:
                    j = j[j >= n - case["window"]]
                if not len(j):
                    continue
                p, o = st["table"][s, j // P].long(), j % P
                k, v = st["keys"][p, o, h].double(), st["values"][p, o, h].double()
                w = torch.softmax(f64["q"].reshape(-1, H, d)[s, h * G:(h + 1) * G] @ k.T / math.sqrt(d), -1)
                out[s, h * G:(h + 1) * G] = w @ v
                weights[p, h, o] = w.sum(0)
        out = out.reshape(case["sequences"], H * d)
        return {"out": out, "weights": weights[:-1]} if case["weights"] else {"out": out}
    if op == "bounds":
        b = torch.zeros(st["bounds"].shape, dtype=torch.float64, device=DEVICE)
        for s, n in enumerate(_lengths(case)):
            for p in range(int(st["first"][s]) // P if case["last"] else 0, _pages(n, P)):
                at = int(st["table"][s, p])
                k = f64["keys"][at, :min(P, n - p * P)]
                b[at, :, 0], b[at, :, 1] = k.min(0).values, k.max(0).values
        return {"bounds": b[:-1]}
    import numpy as np
    if op == "select":
        H, G = case["heads"], case["heads"] // kv
        q, b = st["q"].double().reshape(-1, kv, G, 1, d), st["bounds"].double()
        out = torch.zeros(case["sequences"], kv, case["top"], dtype=torch.float64, device=DEVICE)
        for s, n in enumerate(_pages(n, P) for n in _lengths(case)):
            for h in range(kv if n else 0):
                low, high = b[st["table"][s, :n].long(), h].unbind(1)
                score = torch.where(q[s, h] < 0, q[s, h] * low, q[s, h] * high).sum(-1).amax(0)
                p = np.arange(n)
                forced = (p < case["sink"]) | (p >= n - case["recent"])
                best = np.lexsort((p, -score.cpu().numpy(), ~forced))[:case["top"]]
                out[s, h, :len(best)] = score[torch.from_numpy(np.sort(best)).to(DEVICE)]
        return {"blocks": None, "scores": out}
    keys, values, weights = st["to_keys"].double(), st["to_values"].double(), st["to_weights"].double()
    for s, n in enumerate(_lengths(case)):
        for h in range(kv if n else 0):
            i = np.arange(n)
            at = torch.from_numpy(i).to(DEVICE)
            p, o = st["table"][s, at // P].long(), at % P
            forced = (i < case["sink"]) | (i >= n - case["recent"])
            best = np.sort(np.lexsort((i, -st["weights"][p, h, o].cpu().numpy(), ~forced))[:case["budget"]])
            best = torch.from_numpy(best).to(DEVICE)
            t = torch.arange(len(best), device=DEVICE)
            to, slot = st["to_table"][s, t // P].long(), t % P
            keys[to, slot, h] = st["keys"][p[best], o[best], h].double()
            values[to, slot, h] = st["values"][p[best], o[best], h].double()
            weights[to, h, slot] = st["weights"][p[best], h, o[best]].double()
    return {"kept": None, "lengths": None, "keys": keys[:-1], "values": values[:-1], "weights": weights[:-1]}

"""Paged caches for the paged operators' tests, and the operators' definitions in 64 bits."""
import numpy as np

from frizzle_b200 import _native

NONE = 0xFFFFFFFF
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # a rounding's most, relative


def torch_cuda():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a CUDA device"
    return torch


class Cache:
    """A pool of pages on the GPU and its description; `order` nhd or hnd, `pad` elements between heads' rows."""

    def __init__(self, lengths, page=16, kv=1, d=256, type="f16", order="nhd", seed=0, spare=3, capacity=None,
                 weights=False, bounds=False, fill="randn", pad=0):
        torch = torch_cuda()
        self.lengths = [int(n) for n in lengths]
        self.page, self.kv, self.d, self.type = page, kv, d, type
        self.dtype = torch.float16 if type == "f16" else torch.bfloat16
        width = max(1, max((max(n, capacity or 0) + page - 1) // page for n in self.lengths or [0]))
        g = np.random.default_rng(seed)
        self.pages = len(self.lengths) * width + spare
        self.table_np = g.permutation(self.pages)[:len(self.lengths) * width].reshape(-1, width).astype(np.uint32)
        shape = (self.pages, page, kv, d + pad) if order == "nhd" else (self.pages, kv, page, d + pad)
        gen = torch.Generator(device="cuda").manual_seed(seed + 1)

        def pool():
            t = torch.randn(shape, generator=gen, device="cuda") if fill == "randn" else torch.full(shape, fill, device="cuda")
            t = t.to(self.dtype)[..., :d]
            return t if order == "nhd" else t.permute(0, 2, 1, 3)

        self.keys, self.values = pool(), pool()
        self.table = self.u32(self.table_np)
        self.len = self.u32(np.array(self.lengths, dtype=np.uint32))
        self.weights = torch.rand(self.pages, kv, page, generator=gen, device="cuda") if weights else None
        self.bounds = torch.zeros(self.pages, kv, 2, d, device="cuda", dtype=self.dtype) if bounds else None
        self.error = torch.zeros(1, dtype=torch.int32, device="cuda")
        c = _native.PagedKv()
        c.keys, c.values, c.page_table, c.lengths = (t.data_ptr() for t in (self.keys, self.values, self.table, self.len))
        c.weights = self.weights.data_ptr() if weights else None
        c.bounds = self.bounds.data_ptr() if bounds else None
        c.error = self.error.data_ptr()
        c.page_stride, c.slot_stride, c.head_stride = (self.keys.stride(i) for i in range(3))
        c.sequences, c.table_stride, c.pages, c.page_slots = len(self.lengths), width, self.pages, page
        c.kv_heads, c.head_dim, c.type = kv, d, 0 if type == "f16" else 1
        self.desc = c

    @staticmethod
    def u32(a):
        torch = torch_cuda()
        return torch.from_numpy(np.ascontiguousarray(a).astype(np.uint32).view(np.int32)).cuda()

    def hide(self, value=float("nan")):
        """`value` in every slot that no sequence holds."""
        torch = torch_cuda()
        free = torch.ones(self.pages, self.page, dtype=torch.bool)
        for s, n in enumerate(self.lengths):
            j = np.arange(n)
            free[self.table_np[s, j // self.page].astype(np.int64), j % self.page] = False
        free = free.cuda()
        self.keys[free] = value
        self.values[free] = value
        return self

    def at(self, s, j):
        """(page, slot) index arrays of sequence s's entries j, on the GPU."""
        torch = torch_cuda()
        j = np.asarray(j, dtype=np.int64)
        return (torch.from_numpy(self.table_np[s, j // self.page].astype(np.int64)).cuda(),
                torch.from_numpy(j % self.page).cuda())

    def rows(self, t, s, j, h):
        p, o = self.at(s, j)
        return t[p, o, h].double()

    def weight(self, s, j, h):
        p, o = self.at(s, j)
        return self.weights[p, h, o]


def stream():
    return torch_cuda().cuda.current_stream().cuda_stream


def attend(cache, q, scale, window=0, blocks=None, top=0, decay=0.0, workspace=None, out=None):
    """fz_paged_attention's out, with the call's own workspace unless one is given."""
    torch = torch_cuda()
    lib = _native.load()
    heads = q.shape[1]
    r = _native.PagedQuery()
    out = torch.full_like(q, float("nan")) if out is None else out
    r.q, r.out, r.q_stride, r.out_stride = q.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0)
    r.heads, r.window, r.scale, r.decay = heads, window, scale, decay
    if blocks is not None:
        r.blocks, r.top = blocks.data_ptr(), top
    r.workspace_bytes = lib.fz_paged_attention_workspace(cache.desc, heads)
    if workspace is None:
        # (filled: a workspace's earlier contents must not matter)
        workspace = torch.full((max(256, r.workspace_bytes),), 0xFF, dtype=torch.uint8, device="cuda")
    assert workspace.numel() >= r.workspace_bytes
    r.workspace = workspace.data_ptr()
    _native.check(lib.fz_paged_attention(cache.desc, r, stream()))
    return out


def chosen(cache, s, h, window=0, blocks=None):
    """The entries a query of sequence s and KV head h attends to."""
    n = cache.lengths[s]
    j = np.arange(max(0, n - window) if window else 0, n)
    if blocks is not None:
        b = blocks[s, h].cpu().numpy().view(np.uint32)
        j = j[np.isin(j // cache.page, b[b != NONE])]
    return j


def attend_exact(cache, q, scale, window=0, blocks=None):
    """(out, per (s, KV head): entries and summed weights, per-row error bound) in 64 bits.

    The bound, for f32 arithmetic: a score is off by at most delta = (d + 8) 2^-24 scale max_j sum|q k| (d products
    and sums, each rounded once at most), which moves each softmax weight by a factor within e^(2 delta); exp2 and the
    fold factors add a few units of 2^-22, and summing n weights in order n 2^-24; so |out - exact| <= max|v| times
    2 delta + (n + 64) 2^-24."""
    torch = torch_cuda()
    S, H, d = q.shape
    G = H // cache.kv
    out = torch.zeros(S, H, d, dtype=torch.float64, device="cuda")
    bound = torch.zeros(S, H, 1, dtype=torch.float64, device="cuda")
    weights = {}
    for s in range(S):
        for h in range(cache.kv):
            j = chosen(cache, s, h, window, blocks)
            if not len(j):
                continue
            k, v = cache.rows(cache.keys, s, j, h), cache.rows(cache.values, s, j, h)
            x = q[s, h * G:(h + 1) * G].double()
            w = torch.softmax(scale * (x @ k.T), -1)
            out[s, h * G:(h + 1) * G] = w @ v
            weights[s, h] = (j, w.sum(0))
            delta = (d + 8) * 2.0 ** -24 * scale * (x.abs() @ k.abs().T).amax(-1, keepdim=True)
            bound[s, h * G:(h + 1) * G] = v.abs().max() * (2 * delta + (len(j) + 64) * 2.0 ** -24)
    return out, weights, bound


def best(score, n, sink, recent, take):
    """Indices of the `take` best of score[:n], ascending: forced ones, then the largest (NaN first), ties to the lower index."""
    i = np.arange(n)
    forced = (i < sink) | (i + recent >= n)
    score = np.asarray(score, dtype=np.float64)[:n] + 0.0
    return np.sort(np.lexsort((i, -np.where(np.isnan(score), np.inf, score), ~np.isnan(score), ~forced))[:take])


def select(cache, q, top, sink=0, recent=0, scores=True):
    torch = torch_cuda()
    lib = _native.load()
    shape = (len(cache.lengths), cache.kv, top)
    blocks = torch.full(shape, 7, dtype=torch.int32, device="cuda")
    out = torch.full(shape, 7.0, dtype=torch.float32, device="cuda") if scores else None
    _native.check(lib.fz_paged_select(cache.desc, q.data_ptr(), q.stride(0), q.shape[1], top, sink, recent,
                                      blocks.data_ptr(), out.data_ptr() if scores else None, stream()))
    return blocks, out


def page_scores(cache, q, s, h):
    """Each held page's score in 64 bits."""
    torch = torch_cuda()
    G = q.shape[1] // cache.kv
    n = (cache.lengths[s] + cache.page - 1) // cache.page
    b = cache.bounds[torch.from_numpy(cache.table_np[s, :n].astype(np.int64)).cuda(), h].double()   # [n][2][d]
    x = q[s, h * G:(h + 1) * G].double()[:, None]
    return torch.where(x < 0, x * b[:, 0], x * b[:, 1]).sum(-1).amax(0).cpu().numpy()


def bounds(cache, first=None):
    lib = _native.load()
    f = Cache.u32(np.array(first)) if first is not None else None
    _native.check(lib.fz_paged_bounds(cache.desc, f.data_ptr() if f is not None else None, stream()))


def evict(a, b, budget, sink=0, recent=0):
    torch = torch_cuda()
    kept = torch.full((len(a.lengths), a.kv, budget), 7, dtype=torch.int32, device="cuda")
    _native.check(_native.load().fz_paged_evict(a.desc, b.desc, budget, sink, recent, kept.data_ptr(), stream()))
    return kept


class Rows:
    """Appended rows' inputs, and their description."""

    def __init__(self, cache, heads, sequence, index, position=None, seed=0, gains=True, turns=True, base=10000.0,
                 eps=1e-6, fused=True, scale=2.0):
        torch = torch_cuda()
        g = torch.Generator(device="cuda").manual_seed(seed)
        R, kv, d = len(index), cache.kv, cache.d
        self.heads, self.eps = heads, eps
        self.qkv = torch.randn(R, (heads + 2 * kv) * d, generator=g, device="cuda") * scale
        self.q_out = torch.full((R, heads * d), float("nan"), device="cuda")
        self.q_gain = torch.randn(d, generator=g, device="cuda") if gains else None
        self.k_gain = torch.randn(d, generator=g, device="cuda") if gains else None
        t = base ** (-2.0 * np.arange(d // 2) / d) / (2 * np.pi)
        self.turns_np = t if turns else None
        self.turns = torch.from_numpy(t).cuda() if turns else None
        self.sequence, self.index = np.asarray(sequence, dtype=np.uint32), np.asarray(index, dtype=np.uint32)
        self.position = np.asarray(position if position is not None else index, dtype=np.uint32)
        self.dev = [Cache.u32(x) for x in (self.sequence, self.index, self.position)]
        r = _native.PagedRows()
        w = self.qkv.shape[1]
        r.q, r.k, r.v = (self.qkv.data_ptr() + 4 * d * i for i in (0, heads, heads + kv))
        r.q_stride = r.k_stride = r.v_stride = w
        r.q_out, r.q_out_stride = self.q_out.data_ptr(), heads * d
        r.q_gain = self.q_gain.data_ptr() if gains else None
        r.k_gain = self.k_gain.data_ptr() if gains else None
        r.turns = self.turns.data_ptr() if turns else None
        r.sequence, r.index = self.dev[0].data_ptr(), self.dev[1].data_ptr()
        r.position = self.dev[2].data_ptr() if position is not None else None
        r.rows, r.heads, r.eps = R, heads, eps
        self.desc = r

    def append(self, cache):
        _native.check(_native.load().fz_paged_append(cache.desc, self.desc, stream()))

    def exact(self, cache):
        """(q, k, v, bound of q's and k's f32 error) in 64 bits, [rows][heads][d].

        The bound, in units of 2^-24 of |a| + |b|, a and b the normed pair: the sum of squares and its square root (d / 32
        + 6 sums, halved: 7), the reciprocal root and gain (4), the angle (rounded once, its sine and cosine 2 each: 6
        of |a| + |b|) and the rotation's products and sum (3): 20; 32 taken."""
        R, kv, d, H = len(self.index), cache.kv, cache.d, self.heads
        x = self.qkv.double().reshape(R, H + 2 * kv, d).cpu().numpy()
        v = x[:, H + kv:]
        out = []
        for y, gain in ((x[:, :H], self.q_gain), (x[:, H:H + kv], self.k_gain)):
            if gain is not None:
                y = y / np.sqrt((y * y).mean(-1, keepdims=True) + self.eps) * gain.double().cpu().numpy()
            a, b = y[..., :d // 2], y[..., d // 2:]
            err = np.tile(np.abs(a) + np.abs(b), 2) * 32 * 2.0 ** -24
            if self.turns_np is not None:
                t = self.position.astype(np.longdouble)[:, None] * self.turns_np.astype(np.longdouble)
                angle = (2 * np.pi * (t - np.rint(t)).astype(np.float64))[:, None]
                a, b = a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)
            out += [np.concatenate([a, b], -1), err]
        return out[0], out[1], out[2], out[3], v

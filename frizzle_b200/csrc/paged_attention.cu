// Attention of one new token a sequence over a paged cache (fz_paged_attention).
#include "paged.cuh"

#include <algorithm>
#include <cmath>

namespace fz {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr uint32_t kCtas = 148;        // one an SM
constexpr int kHalf = 8192;            // bytes of a tile's keys, and of its values
constexpr int kSlots = 3;              // halves a warp holds
constexpr int kMerge = 8192;           // floats the warps exchange their outputs through
constexpr int kSmem = kWarps * kSlots * kHalf + kMerge * 4;

struct AttendArgs {
  PagedView kv;
  const float* q;
  float* out;
  uint64_t q_stride, out_stride;
  const uint32_t* blocks;
  uint32_t group, top, window;
  float scale_log2e, decay;
  uint32_t whole;          // items are never split
  uint64_t recip;          // floor(2^64 / CTAs) + 1
  // Workspace.
  float* part_o;           // [kCtas][2][group][D] unnormalised outputs of a CTA's first and last item
  float2* part_ml;         // [kCtas][2][8] their maximum and sum
  uint4* heads;            // [kCtas] the split item a CTA begins: {item, CTAs, its slot, 0}
  uint4* origin;           // [items] where an item's outputs are, for the weights: {first CTA, CTAs, its slot, 0}
  float2* stats;           // [items][8] an unsplit item's maximum and reciprocal sum of weights, for the weights
  float* scores;           // [items][group][score_stride] in log2 units, for the weights
  uint64_t score_stride;
};

// A sequence's list: the entries a query attends to, `count` of them, without
// selected pages those from `first` on, with them the pages' slots in order.
struct List {
  uint32_t n, first, count;
};
FZ_DEV List list_of(const AttendArgs& a, uint32_t s) {
  List l;
  l.n = held(a.kv, s);
  l.first = a.window && l.n > a.window ? l.n - a.window : 0;
  const uint32_t slots = a.kv.page_slots;
  l.count = a.blocks ? min(a.top, (l.n + slots - 1) / a.kv.slots) * slots : l.n - l.first;
  return l;
}

// Entry i of an item's list: its logical index, or FZ_PAGED_NONE.
FZ_DEV uint32_t listed(const AttendArgs& a, const uint32_t* blocks, uint32_t i, const List& l) {
  if (i >= l.count) return FZ_PAGED_NONE;
  if (!blocks) return l.first + i;
  const uint32_t slots = a.kv.page_slots, at = i / a.kv.slots, b = blocks[at];
  if (b == FZ_PAGED_NONE) return FZ_PAGED_NONE;
  if (b >= (l.n + slots - 1) / a.kv.slots || (at && blocks[at - 1] >= b)) {
    note(a.kv, FZ_PAGED_BAD_BLOCK);
    return FZ_PAGED_NONE;
  }
  const uint32_t j = b * slots + (i - at * slots);
  return j < l.n && j >= l.first ? j : FZ_PAGED_NONE;
}

// The table's word for entry i of (s, h)'s list and its slot in that page; slot
// FZ_PAGED_NONE where there is no entry.
FZ_DEV uint32_t look(const AttendArgs& a, uint32_t s, uint32_t h, uint32_t i, const List& l, uint32_t& slot) {
  const uint32_t* blocks = a.blocks ? a.blocks + ((size_t)s * a.kv.kv_heads + h) * a.top : nullptr;
  const uint32_t j = listed(a, blocks, i, l);
  slot = FZ_PAGED_NONE;
  if (j == FZ_PAGED_NONE) return FZ_PAGED_NONE;
  const uint32_t logical = j / a.kv.slots;
  slot = j - logical * a.kv.page_slots;
  return a.kv.table[(size_t)s * a.kv.table_stride + logical];
}
// Whether such a word and slot are an entry to read.
FZ_DEV bool usable(const AttendArgs& a, uint32_t page, uint32_t slot) {
  if (slot == FZ_PAGED_NONE) return false;
  if (page < a.kv.pages) return true;
  note(a.kv, FZ_PAGED_BAD_PAGE);
  return false;
}

constexpr uint32_t kBegin = 3 * kWarps;   // units that beginning an item costs
constexpr uint32_t kJoin = kWarps;        // units that adding up shared items costs

// A CTA's share of all items' units (`unit` entries a unit), in order of
// sequence and KV head: a contiguous run of ceil(all / CTAs) units, so that
// every CTA reads as much as the others whatever the lengths.  Where a CTA has
// several tiles a warp, `extra` units before each item stand for what beginning
// it costs: the warps' barriers and the refilling of the copies' pipeline (8 x
// 32,768 entries of one KV head: CTAs with two items ended 12 us after the
// others, 55 us in all; counted as 8, 16 and 24 units 43, 42 and 40 us; 200
// sequences of 500 entries 33, 30 and 29).  Where whole items, the same number a
// CTA, take no longer than that and the joining (many items of like length),
// items are not cut.  Called by the whole block.
struct Share {
  uint32_t units, items;   // this CTA's; the one that does not count is large
  uint32_t extra;
  uint32_t s, h;           // the first item
  int at;                  // where that item's entries begin, from the CTA's first unit
  List l;                  // its list
  uint64_t first, per;
};
// With up to 32 sequences every warp works it out for itself, without a barrier;
// beyond, the block together.
template <bool BLOCK>
FZ_DEV Share share_by(const AttendArgs& a, uint32_t unit, Share& found) {
  constexpr uint32_t THREADS = BLOCK ? kThreads : 32;
  const uint32_t t = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t S = a.kv.sequences, run = (S + THREADS - 1) / THREADS, s0 = min(S, t * run), s1 = min(S, s0 + run);
  const uint32_t ctas = gridDim.x, KV = a.kv.kv_heads;
  uint64_t tiles = 0;
  uint32_t some = 0, most = 0;
  List l{};
#pragma unroll 1
  for (uint32_t s = s0; s < s1; s++) {
    l = list_of(a, s);
    const uint32_t u = (l.count + unit - 1) / unit;
    tiles += u;
    some += u != 0;
    most = max(most, u);
  }
  uint64_t upto = tiles;
  uint32_t some_upto = some;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, upto, o);
    const uint32_t y = __shfl_up_sync(0xffffffffu, some_upto, o);
    if (lane >= o) upto += x, some_upto += y;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  uint64_t all = __shfl_sync(0xffffffffu, upto, 31), before = upto - tiles;
  uint32_t any = __shfl_sync(0xffffffffu, some_upto, 31), some_before = some_upto - some;
  if (t == 0) found.units = found.items = 0;
  if (BLOCK) {
    __shared__ uint64_t sums[kWarps];
    __shared__ uint2 counts[kWarps];
    if (lane == 31) sums[warp] = upto, counts[warp] = make_uint2(some_upto, most);
    __syncthreads();
    all = 0, any = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) before += sums[w], some_before += counts[w].x;
      all += sums[w];
      any += counts[w].x;
      most = max(most, counts[w].y);
    }
  } else {
    __syncwarp();
  }
  const uint64_t items = (uint64_t)any * KV;
  const uint32_t extra = all * KV >= 2ull * kWarps * ctas ? kBegin : 0u;
  all = all * KV + items * extra;
  // (Shares of a unit or an item more than needed do no harm, so a product with 2^64 / CTAs will do.)
  const uint64_t even = ctas == 1 ? all : __umul64hi(all + ctas - 1, a.recip);
  const uint64_t each = ctas == 1 ? items : __umul64hi(items + ctas - 1, a.recip);
  const uint64_t per = even > kWarps ? even : kWarps;
  const bool whole = each * (most + extra) <= per + kJoin;
  // This thread's sequences, in units or in items.
  const uint64_t from = whole ? (uint64_t)some_before * KV : (before + (uint64_t)some_before * extra) * KV;
  const uint64_t length = whole ? (uint64_t)some * KV : (tiles + (uint64_t)some * extra) * KV;
  const uint64_t first = blockIdx.x * (whole ? each : per);
  if (length && from <= first && first < from + length) {
    uint64_t base = from;
    uint32_t s = s0, u;
    for (;; s++) {
      if (run > 1) l = list_of(a, s);
      u = l.count ? (whole ? 1u : (l.count + unit - 1) / unit + extra) : 0u;
      if (first < base + (uint64_t)u * KV) break;
      base += (uint64_t)u * KV;
    }
    const uint64_t in = first - base;
    // (in / u: an estimate, put right.)
    uint32_t h = KV == 1 ? 0u : min(KV - 1, (uint32_t)((float)in / (float)u));
    while ((uint64_t)h * u > in) h--;
    while ((uint64_t)(h + 1) * u <= in) h++;
    found.h = h;
    found.at = whole ? 0 : (int)(extra + (int64_t)found.h * u - (int64_t)in);
    found.extra = extra;
    found.l = l;
    found.s = s;
    found.items = whole ? (uint32_t)min(each, items - first) : 0xFFFFFFFFu;
    found.units = whole ? 0x7FFFFFFFu : (uint32_t)min(per, all - first);
    found.first = first;
    found.per = per;
  }
  if (BLOCK) __syncthreads();
  else __syncwarp();
  return found;
}
FZ_DEV Share share_of(const AttendArgs& a, uint32_t unit) {
  __shared__ Share found[kWarps];
  return a.kv.sequences <= 32 ? share_by<false>(a, unit, found[threadIdx.x >> 5]) : share_by<true>(a, unit, found[0]);
}

// Walks a CTA's items that have entries: `at` is the item's first unit, counted
// from the CTA's first (negative where an earlier CTA has some of it).
struct Walk {
  uint32_t s, h, units;
  int at;
  uint32_t index;          // items before it in the CTA
  List l;
};
FZ_DEV void load(const AttendArgs& a, Walk& w, uint32_t unit) {
  w.l = list_of(a, w.s);
  w.units = (w.l.count + unit - 1) / unit;
}
// To the next item with entries; false past the last sequence.  Called by whole
// warps, which look at 32 sequences at a time (a padded batch ends in many
// empty ones).
FZ_DEV bool next(const AttendArgs& a, Walk& w, uint32_t unit, uint32_t extra) {
  w.at += (int)(w.units + extra);
  w.index++;
  if (++w.h < a.kv.kv_heads && w.units) return true;
  w.h = 0;
  w.units = 0;
  for (uint32_t s = w.s + 1; s < a.kv.sequences; s += 32) {
    const uint32_t mine = s + (threadIdx.x & 31);
    const uint32_t some = __ballot_sync(0xffffffffu, mine < a.kv.sequences && list_of(a, mine).count != 0);
    if (some) {
      w.s = s + __ffs(some) - 1;
      load(a, w, unit);
      return true;
    }
  }
  w.s = a.kv.sequences;
  return false;
}

// The item a share begins with.
FZ_DEV Walk begin(const Share& sh, uint32_t unit) {
  return Walk{sh.s, sh.h, (sh.l.count + unit - 1) / unit, sh.at, 0, sh.l};
}

FZ_DEV void matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
FZ_DEV void matrices_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
FZ_DEV uint32_t transpose(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// exp2 of a difference to the maximum of `m`'s side: 0 for a side without entries.
FZ_DEV float fold(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

// What the softmax weights of a list of `count` entries are multiplied by on the
// way to the output: f16 ones by 2^15, so that small ones keep their bits, bf16
// ones by at most 1 / (2 count), so that no partial sum of values about the
// largest f32 overflows where their average does not.
template <class T>
FZ_DEV float unit_of(uint32_t count) {
  return T::kType == FZ_KV_F16 ? 32768.f : __uint_as_float((94u + __clz(count - 1)) << 23);
}

// softmax(q k / sqrt d) v for one query a head over a paged list of entries.
//
// The products run on mma.sync m16n8k16 with the entries in the M axis and the
// KV head's query heads in N: scores (16 keys x 8) += K (16 x 16) q^T, out^T
// (16 dims x 8) += V^T p^T, so the cache is the A operand straight from shared
// memory (ldmatrix, transposed for V) and nothing is padded but N.  f32
// accuracy comes from the 8 columns: with 4 heads or fewer they hold the heads'
// f16 parts and remainders side by side (GP = 4, one MMA a step for f16); with
// more (GP = 8) one MMA a part.  q is scaled by a power of two a head, f16 parts so
// that its largest is about 2^14, and the remainders of f16 parts, q's and the
// weights', are times 2^11 more: q keeps 22 bits down to 2^-28 of a head's largest
// (one far larger dimension costs the others nothing) and 2^-50 of that below; the
// weights, at unit_of, 22 bits and 2^-51 of the largest.  (f32's own 24 bits would
// take one MMA more a step; 2^-22 of a score's products' sizes is less than its f32
// sum may be off by.)  A tile's product starts from zero and is added to the running
// output in f32 (the fold's multiply-add), so the tensor cores' own accumulation
// never runs along the sequence.
//
// Bound by HBM: 2 x d x 2 bytes an entry, G x 4 flops a byte.  So each warp is a
// stream of its own: it copies its tiles (8 KiB of keys, 8 of values: 4096 / d
// entries) by 16-byte cp.async, swizzled against bank conflicts, into three
// slots of 8 KiB, two in flight while one is used, 128 KiB in flight an SM, and
// keeps its own running maximum, sum and output; no barrier until an item ends,
// where the eight warps join in shared memory.  The copies run on into the next
// item meanwhile.  Items are cut at equal shares of all entries; what a CTA has
// of an item that others share goes to the workspace, and finish_kernel adds
// those up.
//
// Measured with it, d = 256, 4 heads, f16 (one CTA a sequence and KV head with
// f32 products: 13.3 ms for the first): 8 sequences of up to 32,768 entries, 193
// MB, 38 us (5.1 TB/s), 44 with their weights; up to 131,072 entries 125 us (6.2
// TB/s); 2,048 selected entries of each 10.9 us; one of 36 entries 5.7 us, of
// 4,096 9.4 us, some ten dependent reads, barriers and launches.
template <class T, int D, int GP>
__global__ void __launch_bounds__(kThreads, 1) attend_kernel(const AttendArgs a) {
  constexpr int KT = 4096 / D;                     // entries a tile
  constexpr int MS = KT / 16;                      // 16-entry steps a tile
  constexpr int KS = D / 16;                       // 16-dimension steps
  constexpr int TERMS = Parts<T>::N;
  constexpr int NT = (TERMS * GP + 7) / 8;         // column tiles
  constexpr int CHAINS = 4 / MS;                   // independent sums a score
  constexpr int CPR = D / 8, RPI = 32 / CPR;       // 16-byte pieces a row, rows a copy step
  constexpr float kLift = T::kType == FZ_KV_F16 ? 2048.f : 1.f;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ float2 ml[kWarps][8];
  __shared__ float qc[8];                          // the scores' factor of each head
  // The warps' exchange at an item's end; until then q's B operands.
  float* merge = reinterpret_cast<float*>(smem + kWarps * kSlots * kHalf);
  uint2* qf = reinterpret_cast<uint2*>(merge);     // [KS][NT][32], 12 KiB at most
  float4* raw = reinterpret_cast<float4*>(merge + 4096);   // [GP][D / 4]
  __shared__ float largest[16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t4 = lane & 3, g4 = lane >> 2;
  const uint32_t ring = smem_u32(smem) + warp * kSlots * kHalf;
  const PagedView& v = a.kv;
  const uint32_t G = a.group, KV = v.kv_heads;
  // While the kernel before this one ends: what is read first, from HBM into L2
  // (a hint, so it may still be written).
  {
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x, row = KV * G * (D / 32);   // (32 words a line)
    if (at * 32 < v.sequences) hint(v.lengths + at * 32);
    if (at * 32 < (uint64_t)v.sequences * v.table_stride) hint(v.table + at * 32);
    if (at * 32 < (uint64_t)v.sequences * KV * a.top && a.blocks) hint(a.blocks + at * 32);
    if (at < (uint64_t)v.sequences * row) hint(a.q + at / row * a.q_stride + at % row * 32);
  }
  pdl_wait();
  pdl_launch_dependents();

  // This CTA's items: a share of all units, or where lists are short (as the host
  // decides) whole items by their number alone.
  Walk seg{};
  uint32_t units = 0x7FFFFFFFu, items = 0xFFFFFFFFu, last_item = 0xFFFFFFFFu, extra = 0;
  uint64_t first = 0, per = 1;
  bool some;
  if (a.whole) {
    const uint64_t all = (uint64_t)v.sequences * KV;
    const uint32_t each = (uint32_t)(all + gridDim.x - 1) / gridDim.x, i0 = (uint32_t)min(all, (uint64_t)blockIdx.x * each);
    last_item = (uint32_t)min(all, (uint64_t)i0 + each);
    seg.s = i0 / KV, seg.h = i0 % KV;
    some = i0 < last_item;
    if (some) {
      load(a, seg, KT);
      if (!seg.units) some = next(a, seg, KT, 0);
    }
  } else {
    const Share sh = share_of(a, KT);
    units = sh.units, items = sh.items, extra = sh.extra;
    some = units != 0;
    first = sh.first, per = sh.per;
    if (some) seg = begin(sh, KT);
    if (threadIdx.x == 0) a.heads[blockIdx.x] = make_uint4(0, 0, 0, 0);
  }
  auto mine = [&](const Walk& w) { return w.at < (int)units && w.index < items && w.s * KV + w.h < last_item; };

  // An item's q, a few floats a thread, asked for an item ahead: a load waits
  // behind all the copies in flight, some 3 us.
  constexpr int QV = (GP * D + 4 * kThreads - 1) / (4 * kThreads);
  float4 q_next[QV];
  auto ask_q = [&](const Walk& w) {
    const float4* q = reinterpret_cast<const float4*>(a.q + w.s * a.q_stride + (size_t)w.h * G * D);
#pragma unroll
    for (int r = 0; r < QV; r++) {
      const int f = threadIdx.x + r * kThreads;
      q_next[r] = f < (int)(G * D / 4) ? __ldcg(q + f) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  // Its parts as B operands in shared memory.
  auto put_q = [&]() {
    constexpr int W = D / 4 < 32 ? D / 4 : 32, PER = D / 4 / W;     // lanes a group, groups a head
#pragma unroll
    for (int r = 0; r < QV; r++) {
      const int f = threadIdx.x + r * kThreads;
      const float4 x = q_next[r];
      float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (f < GP * D / 4) {
        raw[f] = x;
        if (f % W == 0) largest[f / W] = top;
      }
    }
    __syncthreads();
    const int g = g4 % GP;                         // the head of column g4 (all tiles)
    float top = largest[g * PER];
#pragma unroll
    for (int i = 1; i < PER; i++) top = fmaxf(top, largest[g * PER + i]);
    uint32_t e = query_exponent<T>(top);
    if (T::kType == FZ_KV_F16) e = max(e, 15u) - 14;   // (the largest in [2^14, 2^15))
    // (With a scale about the largest f32 the room for keys of that size is given up: the factor stays finite.)
    if (T::kType != FZ_KV_F16 && !(__uint_as_float(e << 23) * a.scale_log2e < INFINITY)) e -= 10;
    const float down = __uint_as_float((254 - e) << 23), up = __uint_as_float(e << 23);
    const float2* q = reinterpret_cast<const float2*>(raw) + g * (D / 2) + t4;
    for (int k = warp; k < KS; k += kWarps) {
      const float2 x = q[8 * k], y = q[8 * k + 4];
      const Parts<T> p0 = parts<T>(x.x * down, x.y * down, kLift), p1 = parts<T>(y.x * down, y.y * down, kLift);
#pragma unroll
      for (int n = 0; n < NT; n++)
        qf[(k * NT + n) * 32 + lane] = GP == 8 ? make_uint2(p0.w[n], p1.w[n])
                                               : (g4 < 4 ? make_uint2(p0.w[2 * n], p1.w[2 * n])
                                                         : make_uint2(p0.w[2 * n + 1], p1.w[2 * n + 1]));
    }
    // (An infinite q has no parts: NaN.)
    if (warp == 0 && t4 == 0 && g4 < GP) qc[g4] = top == INFINITY ? NAN : up * a.scale_log2e;
    __syncthreads();
  };
  if (some) ask_q(seg);                            // (before the copies)

  // The copies' side: tile k of this warp is unit warp + 8 k of the CTA.
  Walk ahead = seg;
  bool more = some;
  constexpr int ROWS = (KT + 31) / 32;             // a lane's rows of a tile
  struct Ask {
    uint32_t page[ROWS], slot[ROWS], h;
    bool any;                                      // a tile
  };
  struct Where {
    uint64_t off[ROWS];                            // elements
    uint64_t valid;                                // the tile's rows
    bool any;
  };
  int unit_ahead = warp;
  // The next tile's places: asked for before the products that hide the answer's way, made out after them.
  auto ask = [&]() {
    Ask w;
    w.any = more;
    while (w.any) {
      // (The units before an item's first hold nothing.)
      if (unit_ahead < ahead.at) unit_ahead += (ahead.at - unit_ahead + kWarps - 1) / kWarps * kWarps;
      w.any = mine(ahead) && unit_ahead < (int)units;
      if (!w.any || unit_ahead < ahead.at + (int)ahead.units) break;
      w.any = more = next(a, ahead, KT, extra);
    }
    w.h = ahead.h;
#pragma unroll
    for (int c = 0; c < ROWS; c++) {
      const uint32_t row = lane + 32 * c;
      w.page[c] = w.slot[c] = FZ_PAGED_NONE;
      if (w.any && row < KT)
        w.page[c] = look(a, ahead.s, ahead.h, (uint32_t)(unit_ahead - ahead.at) * KT + row, ahead.l, w.slot[c]);
    }
    unit_ahead += kWarps;
    return w;
  };
  auto find = [&](const Ask& k) {
    Where w;
    w.any = k.any;
    w.valid = 0;
#pragma unroll
    for (int c = 0; c < ROWS; c++) {
      const bool ok = usable(a, k.page[c], k.slot[c]);
      w.off[c] = ok ? element(v, k.page[c], k.slot[c], k.h) : 0;
      w.valid |= (uint64_t)__ballot_sync(0xffffffffu, ok) << (32 * c);
    }
    return w;
  };
  auto fetch = [&](const Where& w, const uint16_t* pool, int slot) {
    if (w.any) {
      // Row i RPI + sub, piece ^ (row & 7) of it (i RPI and sub have no bit in common).
      const int piece = lane % CPR, sub = lane / CPR;
      const uint32_t base = ring + slot * kHalf + sub * (2 * D), place = (piece ^ sub) << 4;
      const uint16_t* from = pool + piece * 8;
      const uint32_t low = (uint32_t)w.valid >> sub, high = (uint32_t)(w.valid >> 32) >> sub;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int row = i * RPI;
        const uint64_t off = __shfl_sync(0xffffffffu, ROWS == 1 || i < 8 ? w.off[0] : w.off[ROWS - 1], (row & 31) + sub);
        copy16(base + row * (2 * D) + (place ^ ((row & 7) << 4)), from + off, ((row < 32 ? low : high) >> (row & 31)) & 1);
      }
    }
    copy_commit();
  };
  const Ask ask0 = ask(), ask1 = ask();
  Where here = find(ask0), soon = find(ask1);
  fetch(here, v.keys, 0);
  fetch(here, v.values, 1);
  fetch(soon, v.keys, 2);
  uint64_t valid = here.valid, valid_soon = soon.valid;
  int slot = 0;                                    // of the next half to use
  int unit = warp;

  // Sequences without entries: zeros, a warp a sequence (while the first copies come).
  for (uint32_t s0 = (blockIdx.x * kWarps + warp) * 32; s0 < v.sequences; s0 += gridDim.x * kThreads) {
    const uint32_t s = s0 + lane;
    bool empty = false;
    if (s < v.sequences) {
      const List l = list_of(a, s);
      if (__ldcg(v.lengths + s) > l.n) note(v, FZ_PAGED_BAD_LENGTH);
      empty = l.count == 0;
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, empty); left; left &= left - 1) {
      float4* out = reinterpret_cast<float4*>(a.out + (s0 + __ffs(left) - 1) * a.out_stride);
      for (uint32_t i = lane; i < KV * G * D / 4; i += 32) out[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }

  while (some && mine(seg)) {
    const int from = max(seg.at, 0), to = min(seg.at + (int)seg.units, (int)units);
    if (unit < seg.at) unit += (seg.at - unit + kWarps - 1) / kWarps * kWarps;
    put_q();
    Walk after = seg;
    const bool then = next(a, after, KT, extra);
    if (then && mine(after)) ask_q(after);
    const float c0 = qc[(2 * t4) % GP], c1 = qc[(2 * t4 + 1) % GP], unit_w = unit_of<T>(seg.l.count);
    float o[KS][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[k][i] = 0.f;

    for (; unit < to; unit += kWarps) {
      // ---- scores
      copy_wait<kSlots - 1>();
      __syncwarp();
      float s[MS][4];
      {
        float sc[MS][CHAINS][NT][4];
#pragma unroll
        for (int x = 0; x < MS * CHAINS * NT * 4; x++) (&sc[0][0][0][0])[x] = 0.f;
        const uint32_t base = ring + slot * kHalf;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          uint2 b[NT];
#pragma unroll
          for (int n = 0; n < NT; n++) b[n] = qf[(k * NT + n) * 32 + lane];
#pragma unroll
          for (int ms = 0; ms < MS; ms++) {
            uint32_t f[4];
            const int row = ms * 16 + (lane & 15), piece = 2 * k + (lane >> 4);
            matrices(f, base + row * (2 * D) + ((piece ^ (row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; n++) mma<T>(sc[ms][k % CHAINS][n], f, b[n].x, b[n].y);
          }
        }
#pragma unroll
        for (int ms = 0; ms < MS; ms++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float x = 0.f;
#pragma unroll
            for (int n = NT - 1; n >= 0; n--) {
              if (kLift > 1.f && n == 0) x *= 1.f / kLift;
#pragma unroll
              for (int ch = 0; ch < CHAINS; ch++) x += sc[ms][ch][n][i];
            }
            if (kLift > 1.f && GP == 4) x = t4 < 2 ? x : x * (1.f / kLift);
            if (GP == 4) x += __shfl_xor_sync(0xffffffffu, x, 2);
            s[ms][i] = x;
          }
      }
      __syncwarp();
      fetch(soon, v.values, slot);
      const Ask asked = ask();
      slot = slot == kSlots - 1 ? 0 : slot + 1;
      float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
      for (int ms = 0; ms < MS; ms++) {
        const bool lo = (valid >> (ms * 16 + g4)) & 1, hi = (valid >> (ms * 16 + g4 + 8)) & 1;
        s[ms][0] = lo ? s[ms][0] * c0 : -INFINITY;
        s[ms][1] = lo ? s[ms][1] * c1 : -INFINITY;
        s[ms][2] = hi ? s[ms][2] * c0 : -INFINITY;
        s[ms][3] = hi ? s[ms][3] * c1 : -INFINITY;
        t0 = fmaxf(t0, fmaxf(s[ms][0], s[ms][2]));
        t1 = fmaxf(t1, fmaxf(s[ms][1], s[ms][3]));
      }
      if (v.weights && 2 * t4 < GP) {
        float* to = a.scores + ((seg.s * (uint64_t)KV + seg.h) * G + 2 * t4) * a.score_stride + (uint32_t)(unit - seg.at) * KT + g4;
#pragma unroll
        for (int x = 0; x < 2 * MS; x++)
#pragma unroll
          for (int c = 0; c < 2; c++)
            if ((valid >> (8 * x + g4)) & 1 && 2 * t4 + c < G)
              to[c * a.score_stride + 8 * x] = s[x / 2][2 * (x & 1) + c];
      }
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, x));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
      }
      t0 = fmaxf(t0, m0), t1 = fmaxf(t1, m1);
      const float b0 = t0 == -INFINITY ? 0.f : t0, b1 = t1 == -INFINITY ? 0.f : t1;
      const float f0 = exp2f(m0 - b0), f1 = exp2f(m1 - b1);
      m0 = t0, m1 = t1;
      l0 *= f0, l1 *= f1;
      uint32_t pf[MS][NT][2];
#pragma unroll
      for (int ms = 0; ms < MS; ms++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float p0 = exp2f(s[ms][2 * i] - b0) * unit_w, p1 = exp2f(s[ms][2 * i + 1] - b1) * unit_w;
          l0 += p0, l1 += p1;
          const Parts<T> p = parts<T>(p0, p1, kLift);
#pragma unroll
          for (int n = 0; n < NT; n++) pf[ms][n][i] = transpose(GP == 8 ? p.w[n] : (t4 < 2 ? p.w[2 * n] : p.w[2 * n + 1]));
        }
      // ---- output
      copy_wait<kSlots - 1>();
      __syncwarp();
      {
        const uint32_t base = ring + slot * kHalf;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          float r[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ms = 0; ms < MS; ms++) {
            uint32_t f[4];
            const int row = ms * 16 + (lane & 7) + ((lane >> 4) << 3), piece = 2 * k + ((lane >> 3) & 1);
            matrices_t(f, base + row * (2 * D) + ((piece ^ (row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; n++) mma<T>(kLift > 1.f && n ? low : r, f, pf[ms][n][0], pf[ms][n][1]);
          }
          if (kLift > 1.f && GP == 8)
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = fmaf(low[i], 1.f / kLift, r[i]);
          o[k][0] = fmaf(o[k][0], f0, r[0]);
          o[k][1] = fmaf(o[k][1], f1, r[1]);
          o[k][2] = fmaf(o[k][2], f0, r[2]);
          o[k][3] = fmaf(o[k][3], f1, r[3]);
        }
      }
      __syncwarp();
      soon = find(asked);
      fetch(soon, v.keys, slot);
      slot = slot == kSlots - 1 ? 0 : slot + 1;
      valid = valid_soon;
      valid_soon = soon.valid;
    }

    // ---- the item's end: the warps' sums, maxima and outputs
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (g4 == 0 && 2 * t4 < GP) ml[warp][2 * t4] = make_float2(m0, l0), ml[warp][2 * t4 + 1] = make_float2(m1, l1);
    if (GP == 4) {
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float x = t4 < 2 ? o[k][i] : o[k][i] * (1.f / kLift);
          o[k][i] = x + __shfl_xor_sync(0xffffffffu, x, 2);
        }
    }
    const bool is_whole = seg.at >= 0 && seg.at + (int)seg.units == to;
    const uint32_t part = blockIdx.x * 2 + (from > 0 ? 1 : 0);
    const uint64_t item = seg.s * (uint64_t)KV + seg.h;
    __syncthreads();                               // (every warp is done with q's operands)
    constexpr int DR = D * GP > 1024 ? 1024 / GP : D;    // dimensions a round
#pragma unroll
    for (int r = 0; r < D / DR; r++) {
      if (2 * t4 < GP) {
#pragma unroll
        for (int k = 0; k < DR / 16; k++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            merge[(warp * GP + 2 * t4 + (i & 1)) * DR + 16 * k + g4 + 8 * (i >> 1)] = o[r * (DR / 16) + k][i];
      }
      __syncthreads();
      const uint32_t g = threadIdx.x / (DR / 4), d = threadIdx.x % (DR / 4) * 4;
      if (g < G) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) top = fmaxf(top, ml[w][g].x);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
          const float2 y = ml[w][g];
          const float f = fold(y.x, top);
          const float4 z = *reinterpret_cast<const float4*>(merge + (w * GP + g) * DR + d);
          sum = fmaf(y.y, f, sum);
          x.x = fmaf(z.x, f, x.x), x.y = fmaf(z.y, f, x.y), x.z = fmaf(z.z, f, x.z), x.w = fmaf(z.w, f, x.w);
        }
        if (is_whole) {
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
          *reinterpret_cast<float4*>(a.out + seg.s * a.out_stride + (seg.h * (size_t)G + g) * D + r * DR + d) =
              make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
          if (v.weights && r == 0 && d == 0) a.stats[item * 8 + g] = make_float2(sum == 0.f ? 0.f : top, inv * unit_w);
        } else {
          *reinterpret_cast<float4*>(a.part_o + ((size_t)part * G + g) * D + r * DR + d) = x;
          if (r == 0 && d == 0) a.part_ml[part * 8 + g] = make_float2(top, sum);
        }
      }
      __syncthreads();
    }
    if (seg.at >= 0 && threadIdx.x == 0) {
      const uint32_t last = (uint32_t)seg.at + seg.units - 1;   // the item's last unit, from this CTA's first
      const uint32_t ctas = is_whole ? 0u : last / (uint32_t)per + 1;
      if (!is_whole) a.heads[blockIdx.x] = make_uint4((uint32_t)item, ctas, from > 0 ? 1u : 0u, 0u);
      if (v.weights) a.origin[item] = make_uint4(blockIdx.x, ctas, from > 0 ? 1u : 0u, 0u);
    }
    seg = after;
    some = then;
  }
  copy_wait<0>();
}

// What is left once every CTA of attend_kernel is done, by two kinds of CTAs.
//
// The first `joins` add up the outputs of the items that several of its `ctas`
// CTAs share: a task is 64 dimensions of a head of one of them, its parts added
// in a fixed order, so the sum never depends on who came first.
//
// The others make the entries' weights from the scores and the items' maxima
// and sums, exp2(score - maximum) / sum (the maximum as it is: one lifted with the
// weights' unit would be rounded from 2^24 on), 128 entries a warp at a time, four
// a lane, each entry written by the one lane it falls to.  (Without the bound on
// the CTAs an SM some forms were compiled to 80 registers and spilled: 10.8 -> 11.2
// us for 2,048 selected entries of 8 sequences.)
constexpr int kWeighed = 128;
template <class T, int D>
__global__ void __launch_bounds__(kThreads, 2) finish_kernel(const AttendArgs a, uint32_t ctas, uint32_t joins, uint32_t pieces) {
  constexpr int COLS = 16, LANES = kThreads / COLS, MOST = (kCtas + LANES - 1) / LANES;
  __shared__ float factor[kCtas];
  __shared__ float4 sums[kThreads];
  __shared__ float reduce[2][kWarps];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const PagedView& v = a.kv;
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x < joins) {
    // The split items, in order.
    __shared__ uint4 split[kCtas];
    __shared__ uint32_t below[kWarps + 1];
    uint4 h = make_uint4(0, 0, 0, 0);
    if (t < (int)ctas) h = __ldcg(a.heads + t);
    const uint32_t any = __ballot_sync(0xffffffffu, h.y != 0);
    if (lane == 0) below[warp + 1] = __popc(any);
    __syncthreads();
    uint32_t items = 0, at = __popc(any & ((1u << lane) - 1));
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) at += below[w + 1];
      items += below[w + 1];
    }
    if (h.y) split[at] = make_uint4(h.x, h.y, h.z, t);
    __syncthreads();
    for (uint32_t task = blockIdx.x; task < items * a.group * (D / 64); task += joins) {
      const uint32_t chunk = task % (D / 64), g = task / (D / 64) % a.group;
      const uint4 h = split[task / (D / 64 * a.group)];
      const uint32_t parts = h.y, c = h.w;
      auto part = [&](uint32_t i) { return (c + i) * 2 + (i == 0 ? h.z : 0u); };
      const int col = t % COLS;
      float4 x[MOST];
#pragma unroll
      for (int k = 0; k < MOST; k++) {
        const uint32_t i = t / COLS + k * LANES;
        if (i < parts)
          x[k] = __ldcg(reinterpret_cast<const float4*>(a.part_o + ((size_t)part(i) * a.group + g) * D + chunk * 64) + col);
      }
      const float2 ml = t < parts ? __ldcg(a.part_ml + part(t) * 8 + g) : make_float2(-INFINITY, 0.f);
      float top = warp_max(ml.x);
      if (lane == 0) reduce[0][warp] = top;
      __syncthreads();
      top = reduce[0][0];
#pragma unroll
      for (int w = 1; w < kWarps; w++) top = fmaxf(top, reduce[0][w]);
      const float f = fold(ml.x, top);
      if (t < parts) factor[t] = f;
      float sum = warp_sum(ml.y * f);
      if (lane == 0) reduce[1][warp] = sum;
      __syncthreads();
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < MOST; k++) {
        const uint32_t i = t / COLS + k * LANES;
        if (i < parts) {
          const float f = factor[i];
          y.x = fmaf(x[k].x, f, y.x), y.y = fmaf(x[k].y, f, y.y), y.z = fmaf(x[k].z, f, y.z), y.w = fmaf(x[k].w, f, y.w);
        }
      }
      sums[t] = y;
      __syncthreads();
      if (t < COLS) {
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) sum += reduce[1][w];
#pragma unroll
        for (int i = 1; i < LANES; i++) {
          const float4 z = sums[i * COLS + col];
          y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
        }
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        const uint32_t s = h.x / v.kv_heads, kvh = h.x % v.kv_heads;
        *(reinterpret_cast<float4*>(a.out + s * a.out_stride + (kvh * (size_t)a.group + g) * D + chunk * 64) + col) =
            make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      }
      __syncthreads();                             // (sums, factor and reduce are used again)
    }
    return;
  }
  uint64_t of = ~0ull;                             // the item whose maxima and sums this warp holds
  float m = 0.f, inv = 0.f;                        // lanes 4 g ..: head g's
  const uint64_t units = (uint64_t)v.sequences * v.kv_heads * pieces;
  for (uint64_t u = (blockIdx.x - joins) * kWarps + warp; u < units; u += (uint64_t)(gridDim.x - joins) * kWarps) {
    const uint64_t item = u / pieces;
    const uint32_t s = (uint32_t)(item / v.kv_heads), kvh = (uint32_t)(item % v.kv_heads);
    const List l = list_of(a, s);
    const uint32_t i0 = (uint32_t)(u - item * pieces) * kWeighed;
    if (i0 >= l.count) continue;
    const uint32_t i = i0 + 4 * lane;
    float* to[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
      uint32_t slot;
      const uint32_t page = look(a, s, kvh, i + c, l, slot);
      const bool ok = usable(a, page, slot);
      to[c] = ok ? v.weights + ((size_t)page * v.kv_heads + kvh) * v.page_slots + slot : nullptr;
    }
    float4 x[8];
    float old[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 8; g++)
      if (g < (int)a.group && i < l.count)
        x[g] = __ldcg(reinterpret_cast<const float4*>(a.scores + (item * a.group + g) * a.score_stride + i));
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (a.decay != 0.f && to[c]) old[c] = __ldcg(to[c]);
    if (item != of) {
      of = item;
      // Lanes 4 g .. 4 g + 3: every fourth of head g's parts (an unsplit item has its maximum and reciprocal sum).
      const uint4 o = __ldcg(a.origin + item);
      const uint32_t g = lane / 4;
      if (!o.y) {
        const float2 st = g < a.group ? __ldcg(a.stats + item * 8 + g) : make_float2(0.f, 0.f);
        m = st.x, inv = st.y;
      } else {
        float top = -INFINITY, sum = 0.f;
#pragma unroll 4
        for (uint32_t p = lane & 3; p < o.y; p += 4) {
          const float2 ml = g < a.group ? __ldcg(a.part_ml + ((o.x + p) * 2 + (p == 0 ? o.z : 0u)) * 8 + g)
                                        : make_float2(-INFINITY, 0.f);
          const float upper = fmaxf(top, ml.x);
          sum = fold(top, upper) * sum + ml.y * fold(ml.x, upper);
          top = upper;
        }
        __syncwarp();
        float upper = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        upper = fmaxf(upper, __shfl_xor_sync(0xffffffffu, upper, 2));
        sum *= fold(top, upper);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        m = sum == 0.f ? 0.f : upper, inv = sum == 0.f ? 0.f : unit_of<T>(l.count) / sum;
      }
    }
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 8; g++) {
      const float mg = __shfl_sync(0xffffffffu, m, 4 * g), ig = __shfl_sync(0xffffffffu, inv, 4 * g);
      if (g < (int)a.group) {
        sum[0] = fmaf(exp2f(x[g].x - mg), ig, sum[0]);
        sum[1] = fmaf(exp2f(x[g].y - mg), ig, sum[1]);
        sum[2] = fmaf(exp2f(x[g].z - mg), ig, sum[2]);
        sum[3] = fmaf(exp2f(x[g].w - mg), ig, sum[3]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (to[c]) *to[c] = fmaf(a.decay, old[c], sum[c]);
    __syncwarp();
  }
}

template <class T, int D>
const void* attend_of(uint32_t group) {
  return group <= 4 ? (const void*)attend_kernel<T, D, 4> : (const void*)attend_kernel<T, D, 8>;
}
template <class T>
const void* attend_of(uint32_t d, uint32_t group) {
  return d == 64 ? attend_of<T, 64>(group) : d == 128 ? attend_of<T, 128>(group) : attend_of<T, 256>(group);
}
template <class T>
const void* finish_of(uint32_t d) {
  return d == 64    ? (const void*)finish_kernel<T, 64>
         : d == 128 ? (const void*)finish_kernel<T, 128>
                    : (const void*)finish_kernel<T, 256>;
}

// Where each part of the workspace begins; returns its whole size, kTooLarge
// from 2^62 bytes on.
constexpr size_t kTooLarge = ~(size_t)0;
size_t layout(const fz_paged_kv* kv, uint32_t heads, size_t (&at)[6]) {
  const uint64_t group = heads / std::max(1u, kv->kv_heads), items = (uint64_t)kv->sequences * kv->kv_heads;
  const double scores = (double)items * ((double)kv->table_stride * kv->page_slots + kWeighed) * group * 4;
  if ((kv->weights && scores >= 0x1p62) || (double)group * kv->head_dim >= 0x1p40) return kTooLarge;
  const uint64_t entries = ((uint64_t)kv->table_stride * kv->page_slots + kWeighed - 1) / kWeighed * kWeighed;
  const uint64_t bytes[6] = {kCtas * 2ull * group * kv->head_dim * 4, kCtas * 2ull * 8 * 8, kCtas * 16ull,
                             kv->weights ? items * 16 : 0, kv->weights ? items * 64 : 0,
                             kv->weights ? items * entries * group * 4 : 0};
  size_t end = 0;
  for (int i = 0; i < 6; i++) {
    at[i] = end;
    end += (bytes[i] + 255) / 256 * 256;
  }
  return end;
}

}  // namespace
}  // namespace fz

extern "C" size_t fz_paged_attention_workspace(const fz_paged_kv* kv, uint32_t heads) {
  size_t at[6];
  return kv ? fz::layout(kv, heads, at) : 0;
}

extern "C" fz_status fz_paged_attention(const fz_paged_kv* kv, const fz_paged_query* query, void* stream) {
  using namespace fz;
  AttendArgs a{};
  fz_status st = paged_view(kv, kNeedKeys, &a.kv);
  if (st) return st;
  if (!query || !query->q || !query->out) return paged_refuse(FZ_ERR_ARGUMENT, "null query, q or out");
  if ((reinterpret_cast<uintptr_t>(query->q) | reinterpret_cast<uintptr_t>(query->out)) & 15u)
    return paged_refuse(FZ_ERR_ARGUMENT, "q or out not 16-byte aligned");
  if ((query->q_stride | query->out_stride) & 3u)
    return paged_refuse(FZ_ERR_ARGUMENT, "q and out strides must be multiples of 4 floats");
  const uint32_t heads = query->heads;
  if (heads == 0 || heads % kv->kv_heads || heads / kv->kv_heads > 8)
    return paged_refuse(FZ_ERR_ARGUMENT, "heads must be 1 to 8 times kv_heads");
  const uint64_t width = (uint64_t)heads * kv->head_dim;
  if (kv->sequences > 1 && (query->q_stride < width || query->out_stride < width))
    return paged_refuse(FZ_ERR_ARGUMENT, "a q or out stride shorter than its heads");
  if (!(query->scale > 0.f) || std::isinf(query->scale)) return paged_refuse(FZ_ERR_ARGUMENT, "scale must be positive and finite");
  if (!(query->decay >= 0.f) || std::isinf(query->decay))
    return paged_refuse(FZ_ERR_ARGUMENT, "decay must be finite and not negative");
  if (query->blocks && query->top == 0) return paged_refuse(FZ_ERR_ARGUMENT, "selected pages need top nonzero");
  if (reinterpret_cast<uintptr_t>(query->blocks) & 3u) return paged_refuse(FZ_ERR_ARGUMENT, "blocks not 4-byte aligned");
  const size_t need = fz_paged_attention_workspace(kv, heads);
  if (need == kTooLarge || !query->workspace || (reinterpret_cast<uintptr_t>(query->workspace) & 255u) || query->workspace_bytes < need)
    return paged_refuse(FZ_ERR_ARGUMENT, "workspace null, not 256-byte aligned, or shorter than fz_paged_attention_workspace");
  const uint64_t items = (uint64_t)kv->sequences * kv->kv_heads;
  if (items == 0) return FZ_OK;
  const void* p[] = {kv->keys, kv->values, kv->page_table, kv->lengths, kv->weights, kv->error,
                     query->q, query->out, query->blocks,  query->workspace};
  if ((st = paged_on_device(p, 10, "fz_paged_attention"))) return st;
  a.q = query->q, a.out = query->out, a.q_stride = query->q_stride, a.out_stride = query->out_stride;
  a.blocks = query->blocks, a.group = heads / kv->kv_heads, a.top = query->top, a.window = query->window;
  a.scale_log2e = (float)((double)query->scale * 1.4426950408889634);
  a.decay = query->decay;
  size_t at[6];
  layout(kv, heads, at);
  char* w = static_cast<char*>(query->workspace);
  a.part_o = reinterpret_cast<float*>(w + at[0]);
  a.part_ml = reinterpret_cast<float2*>(w + at[1]);
  a.heads = reinterpret_cast<uint4*>(w + at[2]);
  a.origin = reinterpret_cast<uint4*>(w + at[3]);
  a.stats = reinterpret_cast<float2*>(w + at[4]);
  a.scores = reinterpret_cast<float*>(w + at[5]);
  const uint64_t entries = (uint64_t)kv->table_stride * kv->page_slots;
  a.score_stride = (entries + kWeighed - 1) / kWeighed * kWeighed;
  uint64_t most = entries;
  if (a.blocks) most = std::min<uint64_t>(most, (uint64_t)a.top * kv->page_slots);
  else if (a.window) most = std::min<uint64_t>(most, a.window);
  const uint32_t tile = 4096 / kv->head_dim;
  const uint64_t tiles = (most + tile - 1) / tile;
  // Items stay whole, by their number alone (no CTA needs every length, and
  // nothing is left to add up), where they have at most a tile a warp, or where a
  // CTA's whole items are at most eight tiles a warp and an even share would save
  // less than the joining costs.  The longest list there may be decides that, not
  // the lengths there are, so it holds only as far as whole items are no slower for
  // one list that long beside short ones either: 148 sequences of d = 256 over tables
  // of 512 entries, all full 13.2 us whole, 16.3 cut by their lengths, one full
  // beside others of 20 entries 12.3 and 19.9; 296 of them 30.3 and 34.2, 16.2 and
  // 20.3; 148 of 1,024 entries 28.7 and 32.3, 19.1 and 19.8; of 2,048 52 and 55, but
  // 32.5 and 19.9 (of 32,768 more than twenty times as long); 64 sequences of 2 KV
  // heads and a window of 512 9.5 and 12.4, one of them full 9.0 and 12.0.  At most a
  // tile a warp: 1,184 sequences over tables of 128 entries, all full 45 and 49, an
  // eighth full beside others of 2 entries 41 and 65; beside empty ones 58 and 28,
  // which is the one kind of batch that loses.
  const uint64_t rounds = (items + kCtas - 1) / kCtas;
  a.whole = tiles <= kWarps || (rounds * tiles <= 8 * kWarps &&
                                (rounds * kCtas - items) * (tiles + kWarps) <= 2ull * kJoin * kCtas);
  const uint32_t grid =
      (uint32_t)std::min<uint64_t>(kCtas, a.whole ? items : (items * tiles + kWarps - 1) / kWarps);
  a.recip = grid > 1 ? ~0ull / grid + 1 : 0;
  void* args[] = {&a};
  const bool f16 = kv->type == FZ_KV_F16;
  const uint32_t d = kv->head_dim;
  if ((st = paged_launch(f16 ? attend_of<F16>(d, a.group) : attend_of<Bf16>(d, a.group), dim3(grid), dim3(kThreads), kSmem,
                         kSmem, 1, args, stream)))
    return st;
  uint32_t joins = a.whole ? 0u : std::min(4 * kCtas, grid * a.group * (d / 64)), weighs = 0, ctas = grid;
  uint32_t pieces = (uint32_t)((most + kWeighed - 1) / kWeighed);
  if (a.kv.weights) weighs = (uint32_t)std::min<uint64_t>(8 * kCtas, (items * pieces + kWarps - 1) / kWarps);
  if (!joins && !weighs) return FZ_OK;
  void* left[] = {&a, &ctas, &joins, &pieces};
  return paged_launch(f16 ? finish_of<F16>(d) : finish_of<Bf16>(d), dim3(joins + weighs), dim3(kThreads), 0, 0, 1, left, stream);
}

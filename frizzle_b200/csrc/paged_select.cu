// Choosing among what a paged cache holds: the pages a query attends to
// (fz_paged_select) and the entries an eviction keeps (fz_paged_evict).
//
// Both take the best `take` of a (sequence, KV head)'s n scores, ties to the
// lower index.  A cluster of CTAs takes one (sequence, KV head): each CTA holds
// the keys of a contiguous slice in shared memory, order-preserving unsigned
// integers of the scores, and the cluster finds the take-th largest digit by
// digit from the first bit in which they differ: a histogram a CTA, summed by the
// cluster's first CTA through distributed shared memory, the digit that the
// take-th falls into, and on with that digit's keys only.  One pass over the
// slice at the end writes the chosen indices in ascending order, each at its
// rank.
#include "paged.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace fz {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 2048;           // 11 bits a digit
constexpr int kMaxCluster = 8;

// A CTA's shared memory in a cluster.  What CTAs tell one another they write
// into all the others' boxes before a cluster barrier, so that after it every
// thread reads its own shared memory: a remote load costs most of a microsecond.
struct Shared {
  alignas(16) uint32_t bins[kBins];
  uint32_t warp[2][kThreads / 32];
  uint64_t range[2][kThreads / 32];
  uint32_t more, equal;               // this CTA's totals of the last block_scan
  uint4 step;                         // the digit, the keys above it and at it
  uint4 count[kMaxCluster];           // a CTA's keys, and of those the ones taken beforehand
  ulonglong2 span[kMaxCluster];       // its free keys' least and greatest
  uint2 taken[kMaxCluster];           // its keys above the threshold, and equal to it
  uint2 zones[kMaxCluster];           // its pages surely in, and near the threshold
  float bound[kMaxCluster];           // its greatest |bound|
};
// `value` into the box of this CTA's rank in every CTA; by the first warp.
template <class V>
FZ_DEV void tell(cg::cluster_group& cluster, V* boxes, V value) {
  const uint32_t c = threadIdx.x;
  if (c < cluster.num_blocks()) *cluster.map_shared_rank(boxes + cluster.block_rank(), c) = value;
}

// Order-preserving unsigned keys, -0 as +0, every NaN above +inf; 0 is no key.
FZ_DEV uint32_t order(float x) { return topk_key(__float_as_uint(x)); }
FZ_DEV uint64_t order(double x) {
  uint64_t b = (uint64_t)__double_as_longlong(x);
  if ((b << 1) == 0) b = 0;
  if ((b & 0x7FFFFFFFFFFFFFFFull) > 0x7FF0000000000000ull) return ~0ull;
  return (b >> 63) ? ~b : b | (1ull << 63);
}

// An exclusive sum over the block's threads of two counts; the totals in sh.more, sh.equal.
FZ_DEV uint2 block_scan(Shared& sh, uint2 c) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint2 s = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s.x += a, s.y += b;
  }
  if (lane == 31) sh.warp[0][w] = s.x, sh.warp[1][w] = s.y;
  __syncthreads();
  uint2 before = make_uint2(0, 0);
  for (int i = 0; i < kThreads / 32; i++) {
    const uint32_t a = sh.warp[0][i], b = sh.warp[1][i];
    if (i < w) before.x += a, before.y += b;
  }
  if (threadIdx.x == kThreads - 1) sh.more = before.x + s.x, sh.equal = before.y + s.y;
  __syncthreads();
  return make_uint2(before.x + s.x - c.x, before.y + s.y - c.y);
}

// Where the take-th largest of a cluster's free keys lies (free: not taken
// beforehand): keys above `prefix` under `mask` are taken, and of those equal
// to it the first `ties`.
template <class K>
struct Threshold {
  K prefix, mask;
  uint32_t ties, want;     // want: the free keys taken in all
  bool none, every;        // no free key is taken; all are
};

// `keys[0 .. n)`: this CTA's, of indices first ..; `forced(index)` ones are
// taken beforehand and count to `take`.  The digits, 11 bits each, begin at the
// highest bit in which the keys differ, so that scores of like size take one
// or two.
template <class K, class Forced>
FZ_DEV Threshold<K> find(cg::cluster_group& cluster, Shared& sh, const K* keys, uint32_t n, uint32_t first, uint32_t take,
                         Forced forced) {
  const uint32_t size = cluster.num_blocks();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  Threshold<K> r{0, 0, 0, 0, false, false};
  // How many are free, and the bits in which they differ.
  uint32_t pinned = 0;
  K least = ~(K)0, most = 0;
  for (uint32_t i = t; i < n; i += kThreads) {
    if (forced(first + i)) {
      pinned++;
    } else {
      least = keys[i] < least ? keys[i] : least;
      most = keys[i] > most ? keys[i] : most;
    }
  }
  pinned = __reduce_add_sync(0xffffffffu, pinned);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const K a = __shfl_xor_sync(0xffffffffu, least, o), b = __shfl_xor_sync(0xffffffffu, most, o);
    least = a < least ? a : least;
    most = b > most ? b : most;
  }
  if (lane == 0) sh.warp[0][warp] = pinned, sh.range[0][warp] = least, sh.range[1][warp] = most;
  for (uint32_t i = t; i < kBins / 4; i += kThreads) reinterpret_cast<uint4*>(sh.bins)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (warp == 0) {
    uint32_t p = lane < kThreads / 32 ? sh.warp[0][lane] : 0u;
    K a = lane < kThreads / 32 ? (K)sh.range[0][lane] : ~(K)0, b = lane < kThreads / 32 ? (K)sh.range[1][lane] : (K)0;
    p = __reduce_add_sync(0xffffffffu, p);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const K x = __shfl_xor_sync(0xffffffffu, a, o), y = __shfl_xor_sync(0xffffffffu, b, o);
      a = x < a ? x : a;
      b = y > b ? y : b;
    }
    tell(cluster, sh.count, make_uint4(n, p, 0, 0));
    tell(cluster, sh.span, make_ulonglong2(a, b));
  }
  cluster.sync();
  uint32_t all = 0, all_pinned = 0;
  least = ~(K)0, most = 0;
  for (uint32_t c = 0; c < size; c++) {
    all += sh.count[c].x, all_pinned += sh.count[c].y;
    least = (K)sh.span[c].x < least ? (K)sh.span[c].x : least;
    most = (K)sh.span[c].y > most ? (K)sh.span[c].y : most;
  }
  all -= all_pinned;
  uint32_t want = take > all_pinned ? take - all_pinned : 0u;
  r.want = want;
  if (want >= all) {
    r.every = true, r.ties = all;        // (mask 0: every key has the prefix)
    return r;
  }
  if (!want) {
    r.none = true;
    return r;
  }
  int high = least == most ? 0 : 8 * (int)sizeof(K) - (sizeof(K) == 8 ? __clzll((long long)(least ^ most)) : __clz((int)(least ^ most)));
  r.mask = high == 8 * (int)sizeof(K) ? (K)0 : ~(K)0 << high;
  r.prefix = most & r.mask;
  r.ties = want;
  while (high > 0) {
    const int bits = high < 11 ? high : 11, shift = high - bits;
    const uint32_t digits = (1u << bits) - 1;
    for (uint32_t i = t; i < n; i += kThreads) {
      const K k = keys[i];
      if ((k & r.mask) == r.prefix && !forced(first + i)) atomicAdd(&sh.bins[(uint32_t)(k >> shift) & digits], 1u);
    }
    cluster.sync();
    if (cluster.block_rank() == 0) {
      // Thread t: four bins from the top, summed over the cluster.
      const uint32_t at = kBins / 4 - 1 - t;
      uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (uint32_t c = 0; c < kMaxCluster; c++)
        if (c < size) {
          const uint4 b = reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.bins, c))[at];
          sum.x += b.x, sum.y += b.y, sum.z += b.z, sum.w += b.w;
        }
      const uint32_t count[4] = {sum.w, sum.z, sum.y, sum.x};
      uint32_t before = block_scan(sh, make_uint2(sum.x + sum.y + sum.z + sum.w, 0u)).x;
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) {
        if (before < want && want <= before + count[i])
          for (uint32_t c = 0; c < size; c++)
            *cluster.map_shared_rank(&sh.step, c) = make_uint4(4 * at + 3 - i, before, count[i], 0);
        before += count[i];
      }
    }
    cluster.sync();
    const uint4 step = sh.step;
    for (uint32_t i = t; i < kBins / 4; i += kThreads) reinterpret_cast<uint4*>(sh.bins)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    want -= step.y;
    r.prefix |= (K)step.x << shift;
    r.mask |= (K)digits << shift;
    r.ties = want;
    high = shift;
    if (want == step.z) break;           // the digit's keys are all taken
  }
  return r;
}

// emit(i, taken, rank) for every entry i of the CTA's n, the taken ones ranked in
// ascending order over the cluster: state(i) 2 taken, 1 a tie, of which the cluster's first `ties`
// are taken, 0 not.  Each thread takes a run of the slice.
template <class State, class Emit>
FZ_DEV void emit_taken(cg::cluster_group& cluster, Shared& sh, uint32_t n, uint32_t ties, State state, Emit emit) {
  const uint32_t rank = cluster.block_rank(), run = (n + kThreads - 1) / kThreads;
  const uint32_t i0 = min(n, threadIdx.x * run), i1 = min(n, i0 + run);
  uint2 mine = make_uint2(0, 0);
  for (uint32_t i = i0; i < i1; i++) {
    const int s = state(i);
    mine.x += s == 2, mine.y += s == 1;
  }
  uint2 at = block_scan(sh, mine);
  if (threadIdx.x < 32) tell(cluster, sh.taken, make_uint2(sh.more, sh.equal));
  cluster.sync();                        // (its arrival is the last thing a CTA does in another's shared memory)
  for (uint32_t c = 0; c < rank; c++) at.x += sh.taken[c].x, at.y += sh.taken[c].y;
  for (uint32_t i = i0; i < i1; i++) {
    const int s = state(i);
    emit(i, s == 2 || (s == 1 && at.y < ties), at.x + min(at.y, ties));
    at.x += s == 2, at.y += s == 1;
  }
}
template <class K>
FZ_DEV int state_of(const Threshold<K>& r, K key, bool forced) {
  if (forced) return 2;
  if (r.none) return 0;
  const K k = key & r.mask;
  return k > r.prefix ? 2 : k == r.prefix ? 1 : 0;
}

// ------------------------------------------------------------ pages

struct SelectArgs {
  PagedView kv;
  const float* q;
  uint64_t q_stride;
  uint32_t group;
  uint32_t top, sink, recent;
  uint32_t* blocks;
  float* scores;
};

// sum over d of q x (q < 0 ? least : greatest) in f64 (each product exact: 24
// + 11 bits), a warp a page, the largest over the group's heads.
template <class T, int D>
FZ_DEV double page_score(const SelectArgs& a, const float* q, uint32_t page, uint32_t h, int lane) {
  constexpr int P = D / 64;
  const uint32_t* b = reinterpret_cast<const uint32_t*>(a.kv.bounds + ((size_t)page * a.kv.kv_heads + h) * 2 * D);
  uint32_t lo[P], hi[P];
#pragma unroll
  for (int c = 0; c < P; c++) lo[c] = b[lane + 32 * c], hi[c] = b[D / 2 + lane + 32 * c];
  double best = 0.0;
  for (uint32_t g = 0; g < a.group; g++) {
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < P; c++) {
      const float2 l = T::unpack(lo[c]), u = T::unpack(hi[c]);
      const float2 x = reinterpret_cast<const float2*>(q + g * D)[lane + 32 * c];
      s = fma((double)x.x, (double)(x.x < 0.f ? l.x : u.x), s);
      s = fma((double)x.y, (double)(x.y < 0.f ? l.y : u.y), s);
      if (l.x != l.x || l.y != l.y) s = (double)NAN;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    best = (g == 0 || order(s) > order(best)) ? s : best;
  }
  return best;
}

// The scores are wanted in 64 bits, and 64-bit conversions run at an eighth of
// the rate of f32 arithmetic or less, so they are made for few pages only.
// First every page's score in f32, off by at most
//   E = 16 x 2^-24 x max_g sum |q| x max |bound|
// (8 fused products a lane and 5 sums over lanes, each within 2^-24 of the sum
// of the products' sizes), and the threshold T among those.  The take-th
// largest true score is then within E of T: pages more than 2 E above T are in,
// pages more than 2 E below are out, and only where more pages lie in between
// than are wanted are those scored in f64 and chosen among by that.  With a
// score or a bound that is not finite, E is not either, and every page is.
//
// f32: D / 8 lanes a page, 8 dimensions a lane, four pages at a time, their
// loads first, each head's q from shared memory once for the four; their sums
// over the lanes are halved page by page (6 shuffles for four pages, not 20).
template <class T, int D>
__global__ void __launch_bounds__(kThreads, 1) select_kernel(const SelectArgs a, uint32_t slice) {
  constexpr int LANES = D / 8, PW = 32 / LANES, BATCH = 4;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  __shared__ float norm[8], bound[kThreads / 32];
  uint64_t* exact = reinterpret_cast<uint64_t*>(dyn);                  // f64 scores of the pages in between
  uint32_t* keys = reinterpret_cast<uint32_t*>(exact + slice);
  float* q = reinterpret_cast<float*>(keys + slice);
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                        // (waited for before the first word to another CTA)
  pdl_wait();
  pdl_launch_dependents();
  const PagedView& v = a.kv;
  const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
  const uint64_t item = blockIdx.x / size;
  const uint32_t s = (uint32_t)(item / v.kv_heads), h = (uint32_t)(item % v.kv_heads);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const float4* q4 = reinterpret_cast<const float4*>(a.q + s * a.q_stride + (size_t)h * a.group * D);
  for (uint32_t i = t; i < a.group * D / 4; i += kThreads) reinterpret_cast<float4*>(q)[i] = __ldcg(q4 + i);
  const uint32_t entries = held(v, s);
  if (t == 0 && rank == 0 && v.lengths[s] > entries) note(v, FZ_PAGED_BAD_LENGTH);
  const uint32_t pages = (entries + v.page_slots - 1) / v.page_slots;
  uint32_t* out = a.blocks + item * a.top;
  float* scores = a.scores ? a.scores + item * a.top : nullptr;
  for (uint32_t i = min(pages, a.top) + rank * kThreads + t; i < a.top; i += size * kThreads) {
    out[i] = FZ_PAGED_NONE;
    if (scores) scores[i] = 0.f;
  }
  const uint32_t per = (pages + size - 1) / size, first = min(pages, rank * per), n = min(pages, first + per) - first;
  const uint32_t* table = v.table + (size_t)s * v.table_stride + first;
  __syncthreads();
  if (warp < (int)a.group) {
    float x = 0.f;
    for (int i = lane; i < D; i += 32) x += fabsf(q[warp * D + i]);
    x = warp_sum(x);
    if (lane == 0) norm[warp] = x;
  }

  // Every page in f32.
  const int part = lane % LANES, sub = lane / LANES;
  float largest = 0.f;
  constexpr uint32_t STEP = kThreads / 32 * BATCH * PW;
  uint32_t base = warp * BATCH * PW;
  uint32_t word = lane < BATCH * PW && base + lane < n ? table[base + lane] : FZ_PAGED_NONE;
  for (; base < n; base += STEP) {
    uint4 lo[BATCH], hi[BATCH];
    uint32_t page[BATCH];
#pragma unroll
    for (int p = 0; p < BATCH; p++) {
      page[p] = __shfl_sync(0xffffffffu, word, p * PW + sub);
      const uint4* b = reinterpret_cast<const uint4*>(v.bounds + ((size_t)(page[p] < v.pages ? page[p] : 0u) * v.kv_heads + h) * 2 * D);
      lo[p] = __ldcg(b + part);
      hi[p] = __ldcg(b + LANES + part);
    }
    word = lane < BATCH * PW && base + STEP + lane < n ? table[base + STEP + lane] : FZ_PAGED_NONE;
    float x[BATCH][8], y[BATCH][8], best[BATCH];
#pragma unroll
    for (int p = 0; p < BATCH; p++) {
      const uint32_t l[4] = {lo[p].x, lo[p].y, lo[p].z, lo[p].w}, u[4] = {hi[p].x, hi[p].y, hi[p].z, hi[p].w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = T::unpack(l[i]), g = T::unpack(u[i]);
        x[p][2 * i] = f.x, x[p][2 * i + 1] = f.y, y[p][2 * i] = g.x, y[p][2 * i + 1] = g.y;
        if (page[p] < v.pages) largest = fmaxf(largest, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(g.x), fabsf(g.y))));
      }
      best[p] = -INFINITY;
    }
    float top = 0.f;
    const bool half = lane & (LANES / 2), quarter = lane & (LANES / 4);
    for (uint32_t g = 0; g < a.group; g++) {
      const float4 qa = reinterpret_cast<const float4*>(q + g * D)[2 * part], qb = reinterpret_cast<const float4*>(q + g * D)[2 * part + 1];
      const float qs[8] = {qa.x, qa.y, qa.z, qa.w, qb.x, qb.y, qb.z, qb.w};
      float sum[BATCH] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int p = 0; p < BATCH; p++) sum[p] = fmaf(qs[i], qs[i] < 0.f ? x[p][i] : y[p][i], sum[p]);
      // (a lane's page is 2 half + quarter from here on)
      const float u0 = (half ? sum[2] : sum[0]) + __shfl_xor_sync(0xffffffffu, half ? sum[0] : sum[2], LANES / 2);
      const float u1 = (half ? sum[3] : sum[1]) + __shfl_xor_sync(0xffffffffu, half ? sum[1] : sum[3], LANES / 2);
      float u = (quarter ? u1 : u0) + __shfl_xor_sync(0xffffffffu, quarter ? u0 : u1, LANES / 4);
#pragma unroll
      for (int o = LANES / 8; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      top = g == 0 || order(u) > order(top) ? u : top;
    }
    const int p = (half ? 2 : 0) + (quarter ? 1 : 0);
    const uint32_t i = base + p * PW + sub;
    const bool ok = (p == 0 ? page[0] : p == 1 ? page[1] : p == 2 ? page[2] : page[3]) < v.pages;
    if (part % (LANES / 4) == 0 && i < n) {
      keys[i] = ok ? order(top) : 0u;
      if (!ok) note(v, FZ_PAGED_BAD_PAGE);
    }
  }
  largest = warp_max(largest);
  if (lane == 0) bound[warp] = largest;
  __syncthreads();
  cluster.barrier_wait();
  if (warp == 0) {
    for (int w = 1; w < kThreads / 32; w++) largest = fmaxf(largest, bound[w]);
    tell(cluster, sh.bound, largest);
  }

  // The threshold among them (its first barrier makes the bounds seen).  A free page's zone: 2 in, 1 near T, 0 out.
  const uint32_t take = min(a.top, pages);
  auto forced = [&](uint32_t i) { return i < a.sink || i + a.recent >= pages; };
  const Threshold<uint32_t> r = find(cluster, sh, keys, n, first, take, forced);
  bool refine = false;
  float above = 0.f, below = 0.f;
  auto zone = [&](uint32_t key) {
    const float x = __uint_as_float(topk_bits(key));
    return key == 0u || x < below ? 0 : x > above || x != x ? 2 : 1;
  };
  if (!r.every && !r.none) {
    float m = 0.f, norms = 0.f;
    for (uint32_t c = 0; c < size; c++) m = fmaxf(m, sh.bound[c]);
    for (uint32_t g = 0; g < a.group; g++) norms = norm[g] > norms || norm[g] != norm[g] ? norm[g] : norms;
    const float e = 2.f * 16.f * 5.9604645e-8f * norms * m;
    const uint32_t low = r.prefix, high = r.prefix | ~r.mask;
    // The ends' scores, as topk_key orders them.  (A NaN threshold: ties by the index, as in f64.)
    const float tl = __uint_as_float(topk_bits(low)), th = __uint_as_float(topk_bits(high));
    below = tl - e, above = th == th ? th + e : INFINITY;
    uint32_t in = 0, near = 0;
    for (uint32_t i = t; i < n; i += kThreads) {
      const int z = forced(first + i) ? 0 : zone(keys[i]);
      in += z == 2, near += z == 1;
    }
    in = __reduce_add_sync(0xffffffffu, in), near = __reduce_add_sync(0xffffffffu, near);
    __syncthreads();
    if (lane == 0) sh.warp[0][warp] = in, sh.warp[1][warp] = near;
    __syncthreads();
    if (warp == 0) {
      in = lane < kThreads / 32 ? sh.warp[0][lane] : 0u, near = lane < kThreads / 32 ? sh.warp[1][lane] : 0u;
      in = __reduce_add_sync(0xffffffffu, in), near = __reduce_add_sync(0xffffffffu, near);
      tell(cluster, sh.zones, make_uint2(in, near));
    }
    cluster.sync();
    in = near = 0;
    for (uint32_t c = 0; c < size; c++) in += sh.zones[c].x, near += sh.zones[c].y;
    refine = tl == tl && in + near != r.want;
  }
  Threshold<uint64_t> r64{};
  auto taken_first = [&](uint32_t i) { return forced(i) || zone(keys[i - first]) == 2; };
  if (refine) {
    for (uint32_t i = warp; i < n; i += kThreads / 32) {
      double d = 0.0;
      const bool near = !forced(first + i) && zone(keys[i]) == 1;
      if (near) d = page_score<T, D>(a, q, table[i], h, lane);
      if (lane == 0) exact[i] = near ? order(d) : 0ull;
    }
    __syncthreads();
    r64 = find(cluster, sh, exact, n, first, take, taken_first);
  }
  emit_taken(
      cluster, sh, n, refine ? r64.ties : r.ties,
      [&](uint32_t i) {
        return refine ? state_of(r64, exact[i], taken_first(first + i)) : state_of(r, keys[i], forced(first + i));
      },
      [&](uint32_t i, bool taken, uint32_t at) {
        if (taken) out[at] = first + i;
        if (scores) exact[i] = taken ? at + 1 : 0;
      });
  if (scores) {
    __syncthreads();
    for (uint32_t i0 = warp * 32; i0 < n; i0 += kThreads) {
      const uint32_t at = i0 + lane < n ? (uint32_t)exact[i0 + lane] : 0u;
      for (uint32_t left = __ballot_sync(0xffffffffu, at != 0); left; left &= left - 1) {
        const int l = __ffs(left) - 1;
        const uint32_t page = table[i0 + l], to = __shfl_sync(0xffffffffu, at, l) - 1;
        const double d = page < v.pages ? page_score<T, D>(a, q, page, h, lane) : 0.0;
        if (lane == 0) scores[to] = (float)d;
      }
    }
  }
}

// ------------------------------------------------------------ eviction

struct EvictArgs {
  PagedView from, to;
  uint32_t budget, sink, recent;
  uint32_t* kept;
};

__global__ void __launch_bounds__(kThreads) keep_kernel(const EvictArgs a, uint32_t slice) {
  constexpr int BATCH = 8;                         // entries a thread asks for at once
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint32_t* keys = reinterpret_cast<uint32_t*>(dyn);
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                        // (waited for before the first word to another CTA)
  pdl_wait();
  pdl_launch_dependents();
  const PagedView& v = a.from;
  const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
  const uint64_t item = blockIdx.x / size;
  const uint32_t s = (uint32_t)(item / v.kv_heads), h = (uint32_t)(item % v.kv_heads);
  const uint32_t entries = held(v, s);
  if (threadIdx.x == 0 && rank == 0 && v.lengths[s] > entries) note(v, FZ_PAGED_BAD_LENGTH);
  uint32_t* out = a.kept + item * a.budget;
  for (uint32_t i = min(entries, a.budget) + rank * kThreads + threadIdx.x; i < a.budget; i += size * kThreads)
    out[i] = FZ_PAGED_NONE;
  const uint32_t per = (entries + size - 1) / size, first = min(entries, rank * per), n = min(entries, first + per) - first;
  const uint32_t* table = v.table + (size_t)s * v.table_stride;
  for (uint32_t i0 = threadIdx.x; i0 < n; i0 += BATCH * kThreads) {
    uint32_t page[BATCH], slot[BATCH];
    float w[BATCH];
#pragma unroll
    for (int c = 0; c < BATCH; c++) {
      const uint32_t i = i0 + c * kThreads, j = first + i;
      page[c] = i < n ? table[j / v.page_slots] : FZ_PAGED_NONE;
      slot[c] = j % v.page_slots;
    }
#pragma unroll
    for (int c = 0; c < BATCH; c++)
      if (page[c] < v.pages) w[c] = __ldcg(v.weights + ((size_t)page[c] * v.kv_heads + h) * v.page_slots + slot[c]);
#pragma unroll
    for (int c = 0; c < BATCH; c++) {
      const uint32_t i = i0 + c * kThreads;
      if (i >= n) break;
      const bool ok = page[c] < v.pages;
      if (!ok) note(v, FZ_PAGED_BAD_PAGE);
      keys[i] = ok ? order(w[c]) : 0u;
    }
  }
  __syncthreads();
  cluster.barrier_wait();
  auto forced = [&](uint32_t i) { return i < a.sink || i + a.recent >= entries; };
  const Threshold<uint32_t> r = find(cluster, sh, keys, n, first, min(a.budget, entries), forced);
  emit_taken(
      cluster, sh, n, r.ties, [&](uint32_t i) { return state_of(r, keys[i], forced(first + i)); },
      [&](uint32_t i, bool taken, uint32_t at) {
        if (taken) out[at] = first + i;
      });
}

// The kept entries' keys and values, D / 8 lanes an entry, 16 bytes a lane, four
// steps' loads at once; their weights; and the new length.  Memory bound: 4 x D
// bytes read and written an entry.
template <int D>
__global__ void __launch_bounds__(256) move_kernel(const EvictArgs a) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES, STEPS = 4;
  pdl_wait();
  pdl_launch_dependents();
  const PagedView &f = a.from, &t = a.to;
  const int lane = threadIdx.x & 31, part = lane % LANES;
  const uint32_t h = blockIdx.y % f.kv_heads, s = blockIdx.y / f.kv_heads;
  const uint32_t* kept = a.kept + (size_t)blockIdx.y * a.budget;
  const uint32_t r0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (ROWS * STEPS);
  if (r0 >= a.budget) return;
  // Lane l: entry r0 + l's places (the first ROWS x STEPS lanes).
  const uint32_t r = r0 + lane;
  const uint32_t j = lane < ROWS * STEPS && r < a.budget ? __ldcg(kept + r) : FZ_PAGED_NONE;
  if (lane < ROWS * STEPS && r < a.budget && h == 0) {
    if (j == FZ_PAGED_NONE) {
      if (r == 0) t.lengths[s] = 0;
    } else if (r + 1 == a.budget || __ldcg(kept + r + 1) == FZ_PAGED_NONE) {
      t.lengths[s] = r + 1;
    }
  }
  uint64_t src = 0, dst = 0;
  bool ok = false;
  if (j != FZ_PAGED_NONE) {
    const uint32_t from = f.table[(size_t)s * f.table_stride + j / f.page_slots],
                   to = t.table[(size_t)s * t.table_stride + r / t.page_slots];
    ok = from < f.pages && to < t.pages;
    if (to >= t.pages) note(t, FZ_PAGED_BAD_PAGE);
    if (ok) {
      src = element(f, from, j % f.page_slots, h), dst = element(t, to, r % t.page_slots, h);
      if (t.weights)
        t.weights[((size_t)to * t.kv_heads + h) * t.page_slots + r % t.page_slots] =
            __ldcg(f.weights + ((size_t)from * f.kv_heads + h) * f.page_slots + j % f.page_slots);
    }
  }
  const uint32_t all = __ballot_sync(0xffffffffu, ok);
  if (!all) return;
  uint4 k[STEPS], x[STEPS];
#pragma unroll
  for (int c = 0; c < STEPS; c++) {
    const int e = c * ROWS + lane / LANES;
    const uint64_t at = __shfl_sync(0xffffffffu, src, e);
    if ((all >> e) & 1) {
      k[c] = __ldcs(reinterpret_cast<const uint4*>(f.keys + at) + part);
      x[c] = __ldcs(reinterpret_cast<const uint4*>(f.values + at) + part);
    }
  }
#pragma unroll
  for (int c = 0; c < STEPS; c++) {
    const int e = c * ROWS + lane / LANES;
    const uint64_t at = __shfl_sync(0xffffffffu, dst, e);
    if ((all >> e) & 1) {
      reinterpret_cast<uint4*>(t.keys + at)[part] = k[c];
      reinterpret_cast<uint4*>(t.values + at)[part] = x[c];
    }
  }
}

// CTAs a cluster: as many as fill the GPU once, at least enough that the
// slices fit shared memory; 0 when even the widest cluster's do not.
uint32_t cluster_for(uint64_t items, uint64_t longest, size_t key_bytes, size_t room) {
  uint32_t c = 1;
  while (c < kMaxCluster && ((longest + c - 1) / c * key_bytes > room || (items * c < 148 && longest / c > 256))) c *= 2;
  return (longest + c - 1) / c * key_bytes > room ? 0 : c;
}

constexpr size_t kRoom = 196 * 1024;

}  // namespace
}  // namespace fz

extern "C" fz_status fz_paged_select(const fz_paged_kv* kv, const float* q, uint64_t q_stride, uint32_t heads, uint32_t top,
                                     uint32_t sink, uint32_t recent, uint32_t* blocks, float* scores, void* stream) {
  using namespace fz;
  SelectArgs a{};
  fz_status st = paged_view(kv, kNeedBounds, &a.kv);
  if (st) return st;
  if (!q || !blocks) return paged_refuse(FZ_ERR_ARGUMENT, "null q or blocks");
  if ((reinterpret_cast<uintptr_t>(q) & 15u) || (q_stride & 3u))
    return paged_refuse(FZ_ERR_ARGUMENT, "q not 16-byte aligned, or its stride no multiple of 4 floats");
  if ((reinterpret_cast<uintptr_t>(blocks) | reinterpret_cast<uintptr_t>(scores)) & 3u)
    return paged_refuse(FZ_ERR_ARGUMENT, "blocks or scores not 4-byte aligned");
  if (heads == 0 || heads % kv->kv_heads || heads / kv->kv_heads > 8)
    return paged_refuse(FZ_ERR_ARGUMENT, "heads must be 1 to 8 times kv_heads");
  if (kv->sequences > 1 && q_stride < (uint64_t)heads * kv->head_dim)
    return paged_refuse(FZ_ERR_ARGUMENT, "a q stride shorter than its heads");
  if (top == 0 || (uint64_t)sink + recent > top) return paged_refuse(FZ_ERR_ARGUMENT, "top must be nonzero and at least sink + recent");
  const uint64_t items = (uint64_t)kv->sequences * kv->kv_heads;
  const uint32_t c = cluster_for(items, kv->table_stride, 12, kRoom);
  if (!c) return paged_refuse(FZ_ERR_NOT_SUPPORTED, "more pages a sequence than a cluster's shared memory holds scores of (133,000)");
  if (items * c > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many sequences");
  if (items == 0) return FZ_OK;
  const void* p[] = {kv->page_table, kv->lengths, kv->bounds, kv->error, q, blocks, scores};
  if ((st = paged_on_device(p, 7, "fz_paged_select"))) return st;
  a.q = q, a.q_stride = q_stride, a.group = heads / kv->kv_heads;
  a.top = top, a.sink = sink, a.recent = recent, a.blocks = blocks, a.scores = scores;
  uint32_t slice = (kv->table_stride + c - 1) / c;
  slice = (slice + 3) & ~3u;     // (q behind the keys is read 16 bytes at a time)
  void* args[] = {&a, &slice};
  const bool f16 = kv->type == FZ_KV_F16;
  const uint32_t d = kv->head_dim;
  const void* fn = f16 ? (d == 64    ? (const void*)select_kernel<F16, 64>
                          : d == 128 ? (const void*)select_kernel<F16, 128>
                                     : (const void*)select_kernel<F16, 256>)
                       : (d == 64    ? (const void*)select_kernel<Bf16, 64>
                          : d == 128 ? (const void*)select_kernel<Bf16, 128>
                                     : (const void*)select_kernel<Bf16, 256>);
  return paged_launch(fn, dim3((uint32_t)(items * c)), dim3(kThreads), slice * 12 + a.group * d * 4, c, args, stream);
}

extern "C" fz_status fz_paged_evict(const fz_paged_kv* from, const fz_paged_kv* to, uint32_t budget, uint32_t sink,
                                    uint32_t recent, uint32_t* kept, void* stream) {
  using namespace fz;
  EvictArgs a{};
  fz_status st = paged_view(from, kNeedKeys | kNeedWeights, &a.from);
  if (st || (st = paged_view(to, kNeedKeys, &a.to))) return st;
  if (!kept) return paged_refuse(FZ_ERR_ARGUMENT, "null kept");
  if (reinterpret_cast<uintptr_t>(kept) & 3u) return paged_refuse(FZ_ERR_ARGUMENT, "kept not 4-byte aligned");
  if (from->type != to->type || from->kv_heads != to->kv_heads || from->head_dim != to->head_dim ||
      from->sequences != to->sequences)
    return paged_refuse(FZ_ERR_ARGUMENT, "from and to differ in type, sequences, KV heads or head dimension");
  if (budget == 0 || (uint64_t)sink + recent > budget)
    return paged_refuse(FZ_ERR_ARGUMENT, "budget must be nonzero and at least sink + recent");
  const uint64_t longest = (uint64_t)from->table_stride * from->page_slots, room = (uint64_t)to->table_stride * to->page_slots;
  if (std::min<uint64_t>(budget, longest) > room) return paged_refuse(FZ_ERR_ARGUMENT, "budget past the destination's table");
  const uint64_t items = (uint64_t)from->sequences * from->kv_heads;
  if (items > 65535) return paged_refuse(FZ_ERR_ARGUMENT, "more than 65,535 sequences times KV heads");
  const uint32_t c = cluster_for(items, longest, 4, kRoom);
  if (!c) return paged_refuse(FZ_ERR_NOT_SUPPORTED, "more entries a sequence than a cluster's shared memory holds weights of (401,000)");
  if (items == 0) return FZ_OK;
  const void* p[] = {from->keys, from->values, from->page_table, from->lengths, from->weights, from->error,
                     to->keys,   to->values,   to->page_table,   to->lengths,   to->weights,   to->error, kept};
  if ((st = paged_on_device(p, 13, "fz_paged_evict"))) return st;
  a.budget = budget, a.sink = sink, a.recent = recent, a.kept = kept;
  uint32_t slice = (uint32_t)((longest + c - 1) / c);
  void* args[] = {&a, &slice};
  if ((st = paged_launch((const void*)keep_kernel, dim3((uint32_t)(items * c)), dim3(kThreads), slice * 4, c, args, stream)))
    return st;
  void* move[] = {&a};
  const uint32_t rows = 8 * 4 * (256 / from->head_dim);    // a CTA's entries
  const void* fn = from->head_dim == 64    ? (const void*)move_kernel<64>
                   : from->head_dim == 128 ? (const void*)move_kernel<128>
                                           : (const void*)move_kernel<256>;
  return paged_launch(fn, dim3((uint32_t)((std::min<uint64_t>(budget, longest) + rows - 1) / rows), (uint32_t)items), dim3(256), 0, 1,
                      move, stream);
}

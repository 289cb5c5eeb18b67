// Choosing among what a paged cache holds: the pages a query attends to
// (fz_paged_select) and the entries an eviction keeps (fz_paged_evict).
//
// Both take the best `take` of a (sequence, KV head)'s n scores, ties to the
// lower index.  A cluster of CTAs takes one (sequence, KV head): each CTA holds
// the keys of a contiguous slice in shared memory, order-preserving unsigned
// integers of the scores, and the cluster finds the take-th largest digit by
// digit from the first bit in which they differ: a histogram a CTA, summed by all
// through distributed shared memory, the digit that the take-th falls into, and
// on with that digit's keys only.  One pass over the
// slice at the end writes the chosen indices in ascending order, each at its
// rank.
#include "paged.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace fz {
namespace {

constexpr int kThreads = 512;
constexpr int kDigit = 9;             // bits a digit: a bin a thread
constexpr int kBins = 1 << kDigit;
static_assert(kBins == kThreads && 2 * kBins >= 4 * 256, "a bin a thread, and find_alone's four digits");
constexpr int kMaxCluster = 8;
constexpr uint32_t kNear = 256;       // pages near a threshold that the first CTA scores in f64
constexpr uint32_t kStages = 4;       // stages of 64 bytes of 32 rows in a warp's shared memory
constexpr size_t kRing = kThreads / 32 * kStages * 4 * 32 * 16;

// A CTA's shared memory in a cluster.  What CTAs tell one another they write
// into all the others' boxes before a cluster barrier, so that after it every
// thread reads its own shared memory: a remote load costs most of a microsecond.
struct Shared {
  alignas(16) uint32_t bins[2][kBins]; // (one digit's are read while the next one's are made)
  uint32_t warp[2][kThreads / 32];
  uint64_t range[2][kThreads / 32];
  uint32_t more, equal;               // this CTA's totals of the last block_scan
  uint4 step;                         // the digit, the keys above it and at it
  uint4 count[kMaxCluster];           // a CTA's keys, and of those the ones taken beforehand
  ulonglong2 span[kMaxCluster];       // its free keys' least and greatest
  uint2 taken[kMaxCluster];           // its keys above the threshold, and equal to it
  uint2 zones[kMaxCluster];           // its pages surely in, and near the threshold
  float bound[kMaxCluster];           // its greatest |bound|
  uint4 verdict;                      // the first CTA's word: whether to refine, and the range near the threshold
};
// The CTAs that choose together: a cluster, or one CTA alone.
struct Group {
  cg::cluster_group* cluster;
  uint32_t size, rank;
};
FZ_DEV void sync(const Group& g) {
  if (g.cluster) g.cluster->sync();
  else __syncthreads();
}
template <class V>
FZ_DEV V* theirs(const Group& g, V* mine, uint32_t c) {
  return g.cluster ? g.cluster->map_shared_rank(mine, c) : mine;
}
// `value` into the box of this CTA's rank in every CTA; by the first warp.
template <class V>
FZ_DEV void tell(const Group& g, V* boxes, V value) {
  if (threadIdx.x < g.size) *theirs(g, boxes + g.rank, threadIdx.x) = value;
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

// `keys[0 .. n)`: this CTA's, of indices first ..; `forced(index, key)` ones are
// taken beforehand and count to `take`.  The digits, 9 bits each, begin at the
// highest bit in which the keys differ, so that scores of like size take one
// or two.
template <class K, class Taken>
FZ_DEV Threshold<K> find(const Group& group, Shared& sh, const K* keys, uint32_t n, uint32_t first, uint32_t take,
                         Taken forced) {
  const uint32_t size = group.size;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  Threshold<K> r{0, 0, 0, 0, false, false};
  // How many are free, and the bits in which they differ.
  uint32_t pinned = 0;
  K least = ~(K)0, most = 0;
  for (uint32_t i = t; i < n; i += kThreads) {
    const K k = keys[i];
    if (forced(first + i, k)) {
      pinned++;
    } else {
      least = k < least ? k : least;
      most = k > most ? k : most;
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
  for (uint32_t i = t; i < 2 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(sh.bins)[i] = make_uint4(0, 0, 0, 0);
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
    tell(group, sh.count, make_uint4(n, p, 0, 0));
    tell(group, sh.span, make_ulonglong2(a, b));
  }
  sync(group);
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
  for (int digit = 0; high > 0; digit++) {
    const int bits = high < kDigit ? high : kDigit, shift = high - bits;
    const uint32_t digits = (1u << bits) - 1;
    uint32_t* bins = sh.bins[digit & 1];
    for (uint32_t i = t; i < n; i += kThreads) {
      const K k = keys[i];
      if ((k & r.mask) == r.prefix && !forced(first + i, k)) atomicAdd(&bins[(uint32_t)(k >> shift) & digits], 1u);
    }
    sync(group);
    // Thread t: a bin from the top, summed over the cluster.  Every CTA does so: telling the others what one found
    // would take another barrier.  (Of 2,048 bins, summed by all or by one, two digits took 12 and 9 us for 8 CTAs of 4,080
    // entries; three of 512 take 9; one sequence of 32,768 entries 16 us in all instead of 18.)
    const uint32_t at = kBins - 1 - t;
    uint32_t count = 0;
#pragma unroll
    for (uint32_t c = 0; c < kMaxCluster; c++)
      if (c < size) count += theirs(group, bins, c)[at];
    // (The other bins were read before this digit's barrier.)
    if (digit) sh.bins[~digit & 1][t] = 0;
    const uint32_t before = block_scan(sh, make_uint2(count, 0u)).x;
    if (before < want && want <= before + count) sh.step = make_uint4(at, before, count, 0);
    __syncthreads();
    const uint4 step = sh.step;
    want -= step.y;
    r.prefix |= (K)step.x << shift;
    r.mask |= (K)digits << shift;
    r.ties = want;
    high = shift;
    if (want == step.z) break;           // the digit's keys are all taken
  }
  return r;
}

// The same by one CTA with all the keys: 8 bits a digit, their 256 bins summed by
// one warp, so that a digit costs two barriers and little else.
template <class Taken>
FZ_DEV Threshold<uint32_t> find_alone(Shared& sh, const uint32_t* keys, uint32_t n, uint32_t take, Taken forced) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  Threshold<uint32_t> r{0, 0, 0, 0, false, false};
  uint32_t pinned = 0, least = ~0u, most = 0;
  for (uint32_t i = t; i < n; i += kThreads) {
    const uint32_t k = keys[i];
    if (forced(i, k)) pinned++;
    else least = min(least, k), most = max(most, k);
  }
  pinned = __reduce_add_sync(0xffffffffu, pinned);
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) sh.warp[0][warp] = pinned, sh.range[0][warp] = least, sh.range[1][warp] = most;
  for (int i = t; i < 4 * 256; i += kThreads) sh.bins[i / kBins][i % kBins] = 0;
  __syncthreads();
  pinned = 0, least = ~0u, most = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; w++) {
    pinned += sh.warp[0][w];
    least = min(least, (uint32_t)sh.range[0][w]);
    most = max(most, (uint32_t)sh.range[1][w]);
  }
  uint32_t want = take > pinned ? take - pinned : 0u;
  r.want = r.ties = want;
  if (want >= n - pinned) {
    r.every = true, r.ties = n - pinned;
    return r;
  }
  if (!want) {
    r.none = true;
    return r;
  }
  int high = least == most ? 0 : 32 - __clz((int)(least ^ most));
  r.mask = high == 32 ? 0u : ~0u << high;
  r.prefix = most & r.mask;
  for (uint32_t* bins = sh.bins[0]; high > 0; bins += 256) {
    const int bits = high < 8 ? high : 8, shift = high - bits;
    const uint32_t digits = (1u << bits) - 1;
    for (uint32_t i = t; i < n; i += kThreads) {
      const uint32_t k = keys[i];
      if ((k & r.mask) == r.prefix && !forced(i, k)) atomicAdd(&bins[(k >> shift) & digits], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // Lane l: eight bins from the top.
      uint32_t count[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) count[i] = bins[255 - (8 * lane + i)], sum += count[i];
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      uint32_t before = upto - sum;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (before < want && want <= before + count[i]) sh.step = make_uint4(255 - (8 * lane + i), before, count[i], 0);
        before += count[i];
      }
    }
    __syncthreads();
    const uint4 step = sh.step;
    want -= step.y;
    r.prefix |= step.x << shift;
    r.mask |= digits << shift;
    r.ties = want;
    high = shift;
    if (want == step.z) break;           // the digit's keys are all taken
  }
  return r;
}

// emit(i, rank) for every taken entry i of the CTA's n, ranked in ascending order
// over the cluster: state(i) 2 taken, 1 a tie, of which the cluster's first
// `ties` are taken, 0 not.  Each warp takes a run of the slice, 32 at a time.
template <class State, class Emit>
FZ_DEV void emit_taken(const Group& group, Shared& sh, uint32_t n, uint32_t ties, State state, Emit emit) {
  constexpr int W = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t run = (n + 32 * W - 1) / (32 * W) * 32, i0 = min(n, warp * run), i1 = min(n, i0 + run);
  uint32_t more = 0, equal = 0;
  for (uint32_t i = i0; i < i1; i += 32) {
    const int s = i + lane < i1 ? state(i + lane) : 0;
    more += __popc(__ballot_sync(0xffffffffu, s == 2)), equal += __popc(__ballot_sync(0xffffffffu, s == 1));
  }
  __syncthreads();                       // (sh.warp is read)
  if (lane == 0) sh.warp[0][warp] = more, sh.warp[1][warp] = equal;
  __syncthreads();
  more = equal = 0;
  uint32_t all_more = 0, all_equal = 0;
#pragma unroll
  for (int w = 0; w < W; w++) {
    if (w < warp) more += sh.warp[0][w], equal += sh.warp[1][w];
    all_more += sh.warp[0][w], all_equal += sh.warp[1][w];
  }
  if (group.size > 1) {
    if (warp == 0) tell(group, sh.taken, make_uint2(all_more, all_equal));
    sync(group);                         // (its arrival is the last thing a CTA does in another's shared memory)
    for (uint32_t c = 0; c < group.rank; c++) more += sh.taken[c].x, equal += sh.taken[c].y;
  }
  for (uint32_t i = i0; i < i1; i += 32) {
    const int s = i + lane < i1 ? state(i + lane) : 0;
    const uint32_t two = __ballot_sync(0xffffffffu, s == 2), one = __ballot_sync(0xffffffffu, s == 1), below = (1u << lane) - 1;
    const uint32_t m = more + __popc(two & below), e = equal + __popc(one & below);
    if (s == 2 || (s == 1 && e < ties)) emit(i + lane, m + min(e, ties));
    more += __popc(two), equal += __popc(one);
  }
}
// Keys above a range 2, in it 1, below it 0; a threshold's range is the keys with its prefix.
template <class K>
struct Range {
  K low, high;
  FZ_DEV int side(K key) const { return key > high ? 2 : key >= low ? 1 : 0; }
};
template <class K>
FZ_DEV Range<K> range_of(const Threshold<K>& r) {
  return r.none ? Range<K>{~(K)0, ~(K)0} : Range<K>{r.prefix, r.prefix | ~r.mask};
}
// The entries taken beforehand: the first `sink` of n and the last `recent`.
struct Forced {
  uint32_t sink, tail;
  FZ_DEV bool operator()(uint32_t i, uint32_t = 0) const { return i < sink || i >= tail; }
};
FZ_DEV Forced forced_of(uint32_t n, uint32_t sink, uint32_t recent) { return Forced{sink, n > recent ? n - recent : 0u}; }

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
// + 11 bits), a warp a page, the largest over the group's heads; four heads at a
// time, so that their loads and sums overlap.
template <class T, int D>
FZ_DEV double page_score(const SelectArgs& a, const float* q, uint32_t page, uint32_t h, int lane) {
  constexpr int P = D / 64, HEADS = 4;
  const uint32_t* b = reinterpret_cast<const uint32_t*>(a.kv.bounds + ((size_t)page * a.kv.kv_heads + h) * 2 * D);
  uint32_t lo[P], hi[P];
#pragma unroll
  for (int c = 0; c < P; c++) lo[c] = b[lane + 32 * c], hi[c] = b[D / 2 + lane + 32 * c];
  double best = 0.0;
  for (uint32_t g0 = 0; g0 < a.group; g0 += HEADS) {
    float2 x[HEADS][P];
    double s[HEADS];
#pragma unroll
    for (int g = 0; g < HEADS; g++)
#pragma unroll
      for (int c = 0; c < P; c++)
        x[g][c] = __ldcg(reinterpret_cast<const float2*>(q + min(g0 + g, a.group - 1) * D) + lane + 32 * c);
#pragma unroll
    for (int g = 0; g < HEADS; g++) {
      s[g] = 0.0;
#pragma unroll
      for (int c = 0; c < P; c++) {
        const float2 l = T::unpack(lo[c]), u = T::unpack(hi[c]);
        s[g] = fma((double)x[g][c].x, (double)(x[g][c].x < 0.f ? l.x : u.x), s[g]);
        s[g] = fma((double)x[g][c].y, (double)(x[g][c].y < 0.f ? l.y : u.y), s[g]);
        if (l.x != l.x || l.y != l.y) s[g] = (double)NAN;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int g = 0; g < HEADS; g++) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
#pragma unroll
    for (int g = 0; g < HEADS; g++) best = (g0 + g == 0 || order(s[g]) > order(best)) ? s[g] : best;
  }
  return best;
}

// A finite value of a 16-bit type as f64 times 2^-896: the exponent and leading
// bits of its f32 moved to f64's upper word (the lower one is zero), subnormal or
// not, by two integer instructions; a conversion runs at a fraction of their rate.
FZ_DEV uint32_t upper_word(float x) { return (uint32_t)((int)__float_as_uint(x) >> 3) & 0x8FFFFFFFu; }

// The greater sizes of two pairs, NaN kept; and whether one of a pair is no
// finite value.
template <class T>
FZ_DEV uint32_t greatest_size(uint32_t m, uint32_t x);
template <>
FZ_DEV uint32_t greatest_size<F16>(uint32_t m, uint32_t x) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&m), __habs2(*reinterpret_cast<__half2*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
FZ_DEV uint32_t greatest_size<Bf16>(uint32_t m, uint32_t x) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&m), __habs2(*reinterpret_cast<__nv_bfloat162*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <class T>
FZ_DEV bool not_finite(uint32_t word) {
  constexpr bool F = T::kType == FZ_KV_F16;
  return ((word & (F ? 0x7C007C00u : 0x7F807F80u)) + (F ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}

// q's values as f64 times 2^126, for a lane to read its eight of a head two at a
// time without bank conflicts: where value i of head g lies.
template <int D>
FZ_DEV uint32_t lifted_place(uint32_t g, uint32_t i) {
  return ((g * 4 + i % 8 / 2) * (D / 8) + i / 8) * 2 + i % 2;
}
constexpr int kLift = 126;               // (sums of products are times 2^-770 then, which keeps all that f32 could hold)

// The scores of the listed pages as their f64 sums rounded to f32 (rounding
// keeps the order, so the largest of the heads is taken of the rounded ones):
// D / 8 lanes a page and 16 bytes of each row a lane.  A page with an infinity or
// NaN by page_score.  Bound by the instructions of 16 warps an SM: 128 pages by 8
// SMs cost a selection of 2,032 pages 2.4 us, 200 pages by two of 16 x 4 7.0 (all
// by page_score 2.8 and 15; q's parts in registers instead of shared memory 3.6
// and 6.2, eight lanes a page 3.3 and 6.0).
template <class T, int D, int GP>
FZ_DEV void listed_scores(const SelectArgs& a, const float* q, const double* lifted, uint32_t h, const uint32_t* table,
                          const uint32_t* list, float* scores, uint32_t take, uint32_t w, uint32_t warps) {
  constexpr uint32_t LANES = D / 8, PER = 32 / LANES;                  // lanes a page, pages a step
  const uint32_t lane = threadIdx.x & 31, part = lane % LANES, sub = lane / LANES;
  const double2* x = reinterpret_cast<const double2*>(lifted) + part;
  const double back = __hiloint2double((1023 - kLift + 896) << 20, 0);
  for (uint32_t base = PER * w; base < take; base += 32 * warps) {
    // Lane l: the word of entry l mod PER of step l / PER.
    const uint32_t mine = base + lane / PER * PER * warps + lane % PER;
    const uint32_t words = mine < take ? table[__ldcg(list + mine)] : FZ_PAGED_NONE;
    const uint32_t steps = min(LANES, (take - base + PER * warps - 1) / (PER * warps));
    uint4 lo, hi;
    auto load = [&](uint32_t step) {
      const uint32_t page = __shfl_sync(0xffffffffu, words, PER * step + sub), at = page < a.kv.pages ? page : 0u;
      const uint4* b = reinterpret_cast<const uint4*>(a.kv.bounds + ((size_t)at * a.kv.kv_heads + h) * 2 * D) + part;
      lo = b[0], hi = b[LANES];
      return page;
    };
    uint32_t next = load(0);
#pragma unroll 1
    for (uint32_t step = 0; step < steps; step++) {
      const uint32_t l4[4] = {lo.x, lo.y, lo.z, lo.w}, u4[4] = {hi.x, hi.y, hi.z, hi.w}, page = next;
      if (step + 1 < steps) next = load(step + 1);
      uint32_t l[8], u[8], most = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 y = T::unpack(l4[i]), z = T::unpack(u4[i]);
        l[2 * i] = upper_word(y.x), l[2 * i + 1] = upper_word(y.y);
        u[2 * i] = upper_word(z.x), u[2 * i + 1] = upper_word(z.y);
        most = greatest_size<T>(greatest_size<T>(most, l4[i]), u4[i]);
      }
      // Two heads' chains at once (the second of an odd number is zeros).
      double s[GP];
#pragma unroll
      for (int g = 0; g < GP; g++) s[g] = 0.0;
#pragma unroll
      for (int g = 0; g < GP; g += 2)
        if (g < (int)a.group) {
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = g; k < g + 2; k++) {
              const double2 y = x[(k * 4 + i) * LANES];
              s[k] = fma(y.x, __hiloint2double(__double2hiint(y.x) < 0 ? l[2 * i] : u[2 * i], 0), s[k]);
              s[k] = fma(y.y, __hiloint2double(__double2hiint(y.y) < 0 ? l[2 * i + 1] : u[2 * i + 1], 0), s[k]);
            }
        }
      // Half the heads to half the lanes at each step, until a lane has one.
      uint32_t head = 0;
      int o = LANES / 2;
#pragma unroll
      for (int n = GP / 2; n > 0; n /= 2, o /= 2) {
        const bool upper = lane & o;
        head += upper ? n : 0;
#pragma unroll
        for (int i = 0; i < n; i++) s[i] = (upper ? s[i + n] : s[i]) + __shfl_xor_sync(0xffffffffu, upper ? s[i] : s[i + n], o);
      }
#pragma unroll
      for (; o > 0; o /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
      uint32_t best = head < a.group ? order((float)(s[0] * back)) : 0u;
#pragma unroll
      for (o = LANES / 2; o > (int)LANES / 2 / GP; o /= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
      for (uint32_t left = __ballot_sync(0xffffffffu, not_finite<T>(most)); left;) {
        const uint32_t first = (__ffs(left) - 1) / LANES * LANES, at = __shfl_sync(0xffffffffu, page, first);
        const uint32_t key = order((float)page_score<T, D>(a, q, at < a.kv.pages ? at : 0u, h, lane));
        if (sub == first / LANES) best = key;
        left &= ~((LANES == 32 ? ~0u : (1u << LANES % 32) - 1) << first);
      }
      const uint32_t e = base + step * PER * warps + sub;
      if (part == 0 && e < take) scores[e] = page < a.kv.pages ? __uint_as_float(topk_bits(best)) : -INFINITY;
    }
  }
}

template <class T>
FZ_DEV uint32_t greater_size(uint32_t m, uint32_t x);
template <>
FZ_DEV uint32_t greater_size<F16>(uint32_t m, uint32_t x) {
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&m), __habs2(*reinterpret_cast<__half2*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
FZ_DEV uint32_t greater_size<Bf16>(uint32_t m, uint32_t x) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&m), __habs2(*reinterpret_cast<__nv_bfloat162*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The choice is wanted by the scores in 64 bits, and 64-bit conversions run at an
// eighth of the rate of f32 arithmetic or less, so those are made for few pages
// only.  First every page's score to f32 accuracy, off by at most
//   E = 2^-24 x max_g (88 sum |q| + D / 2 max |q|) x max |bound|
// (below), and the threshold T among those.  The take-th largest true score is
// then within E of T: pages more than 2 E above T are in, pages more than 2 E
// below are out, and only where more pages lie in between than are wanted are
// those scored in f64 and chosen among by that (a page or two of two thousand,
// as a rule).  Where that product of sizes is not finite (an infinite bound, a
// NaN query, scores about the largest f32), every page is.
//
// The scores are products of the pages' rows of 2 D least and greatest keys with
// q's negative and positive parts: mma.sync m16n8k16 with 16 pages in M and the
// heads' parts of the cache's type in N, as attend_kernel has them (f16 22 bits
// of q, bf16 24).  The order of the 2 D products is free, so a lane takes 16
// bytes of a row as they lie for two steps' A operands; it copies them itself,
// by cp.async three stages ahead, and no barrier or ldmatrix comes between.  Two
// MMAs run into one f32 sum: 32 additions, each taken to be within 2^-23 of the
// products' sizes, which is an assumption (the instruction's rounding is not
// documented; over products of all sizes that cancel, all 32 together were off by
// 0.3 x 2^-23 of the sizes at most).  Those sums are added in f32 (2 D / 32 of them,
// and at most four of parts): 64 + 20 times 2^-24; what q's parts leave out is 2^-23
// of a value, or 2^-25 of the head's largest where a remainder is subnormal.
//
// A product may be lost below the least normal f32: the 3 D that are not zero are
// less than 2^-24 of a head's size with bounds of 10^-26, so E takes no smaller
// bound; a score itself is rounded at 2^-149, less than 10^-40, which E adds.
//
// Bound by HBM while it scores (4 D bytes a page), by barriers and single steps
// while it chooses: 16 sequences of up to 2,048 pages and 4 KV heads, 94 MB, 32.8
// us, 22 of them scoring the longest (all in f64: 90 us; f32 lanes and shuffles:
// 61); one sequence of 2,032 pages 14.8 us (59, 25.7).  With the listed pages'
// scores, which are f64's again, 39.8 and 17.2 us.
//
// Where one CTA's shared memory holds all the cluster's scores (`together`), the
// first CTA gets them all and chooses alone, two cluster barriers in all; beyond
// that the cluster does digit by digit.
template <class T, int D, int GP>
__global__ void __launch_bounds__(kThreads, 1) select_kernel(const SelectArgs a, uint32_t slice, uint32_t together) {
  constexpr int STEPS = D / 8, NT = (Parts<T>::N * GP + 7) / 8;        // 16-product steps a page; column tiles
  constexpr uint32_t STAGES = D / 32;                                  // stages (4 steps) a tile of 16 pages
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  __shared__ float norm[8], scale[8], bound[kThreads / 32];
  __shared__ uint32_t near_at[kNear], nears;
  __shared__ uint64_t near_key[kNear];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, t4 = lane & 3, g4 = lane >> 2;
  // [stage][piece][lane]: what a lane copies it alone reads.
  uint4* ring = reinterpret_cast<uint4*>(dyn) + warp * kStages * 4 * 32 + lane;
  uint2* qf = reinterpret_cast<uint2*>(dyn + kRing);                   // [STEPS][NT][32] q's B operands
  uint64_t* exact = reinterpret_cast<uint64_t*>(qf + STEPS * NT * 32); // f64 scores of the pages in between
  uint32_t* keys = reinterpret_cast<uint32_t*>(exact + slice);         // this CTA's, in the first CTA all with `together`
  uint32_t* chosen = keys + (together ? together : slice);             // a bit a page: near the threshold and taken
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                        // (waited for before the first word to another CTA)
  const PagedView& v = a.kv;
  // While the kernel before this one ends: what is read first, from HBM into L2.
  if (t == 0) hint(v.lengths + blockIdx.x / cluster.num_blocks() / v.kv_heads);
  for (uint32_t i = t * 32; i < slice; i += kThreads * 32)
    hint(v.table + blockIdx.x / cluster.num_blocks() / v.kv_heads * (size_t)v.table_stride +
         min(cluster.block_rank() * slice + i, v.table_stride - 1));
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank(), G = a.group;
  const Group whole{&cluster, size, rank}, single{nullptr, 1, 0};
  const uint64_t item = blockIdx.x / size;
  const uint32_t s = (uint32_t)(item / v.kv_heads), h = (uint32_t)(item % v.kv_heads);
  const float* q = a.q + s * a.q_stride + (size_t)h * G * D;
  const uint32_t length = v.lengths[s];
  // q: each head's size and scale.
  if (warp < GP) {
    float sum = 0.f, top = 0.f;
    for (int i = lane; i < D / 4 && warp < (int)G; i += 32) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(q + warp * D) + i);
      sum += fabsf(x.x) + fabsf(x.y) + fabsf(x.z) + fabsf(x.w);
      top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
    }
    sum = warp_sum(sum), top = warp_max(top);
    if (lane == 0) norm[warp] = 88.f * sum + top * (D / 2), scale[warp] = top == INFINITY ? NAN : __uint_as_float(query_exponent<T>(top) << 23);
  }
  const uint32_t entries = min(length, v.table_stride * v.page_slots);
  if (t == 0 && rank == 0 && length > entries) note(v, FZ_PAGED_BAD_LENGTH);
  const uint32_t pages = (entries + v.page_slots - 1) / v.slots;
  const uint32_t per = (pages + size - 1) / size, first = min(pages, rank * per), n = min(pages, first + per) - first;
  const uint32_t* table = v.table + (size_t)s * v.table_stride;
  const bool alone = together && size > 1, one = alone || size == 1;   // one CTA chooses
  for (uint32_t i = t; one && i < (pages + 31) / 32; i += kThreads) chosen[i] = 0;
  if (t == 0) nears = 0;

  // The copies, kStages - 1 stages ahead of their use: rows g4 and g4 + 8 of the
  // tile, 16 bytes of every 64.
  auto look = [&](uint32_t tile) {
    const uint32_t i = tile * 16 + lane;
    return lane < 16 && i < n ? table[first + i] : FZ_PAGED_NONE;
  };
  uint32_t ahead = warp, word = look(warp);
  const uint4 *row0 = nullptr, *row1 = nullptr;
  bool ok0 = false, ok1 = false;
  uint32_t fetched = 0;
  auto fetch = [&]() {
    const uint32_t st = fetched % STAGES;
    if (st == 0) {
      const uint32_t p0 = __shfl_sync(0xffffffffu, word, g4), p1 = __shfl_sync(0xffffffffu, word, g4 + 8);
      ok0 = p0 < v.pages, ok1 = p1 < v.pages;
      const uint4* b = reinterpret_cast<const uint4*>(v.bounds);
      row0 = b + ((size_t)(ok0 ? p0 : 0u) * v.kv_heads + h) * (D / 4) + t4;
      row1 = b + ((size_t)(ok1 ? p1 : 0u) * v.kv_heads + h) * (D / 4) + t4;
      ahead += kThreads / 32;
      word = look(ahead);
    }
    const uint32_t slot = smem_u32(ring + (fetched % kStages) * 4 * 32);
    copy16(slot, row0 + 8 * st, ok0);
    copy16(slot + 512, row1 + 8 * st, ok1);
    copy16(slot + 1024, row0 + 8 * st + 4, ok0);
    copy16(slot + 1536, row1 + 8 * st + 4, ok1);
    copy_commit();
    fetched++;
  };
#pragma unroll
  for (uint32_t k = 0; k < kStages - 1; k++) fetch();

  uint32_t* out = a.blocks + item * a.top;
  float* scores = a.scores ? a.scores + item * a.top : nullptr;
  for (uint32_t i = min(pages, a.top) + rank * kThreads + t; i < a.top; i += size * kThreads) {
    out[i] = FZ_PAGED_NONE;
    if (scores) scores[i] = 0.f;
  }
  __syncthreads();
  // Its parts.
  {
    const uint32_t g = g4 % GP;
    const float down = __uint_as_float((254u << 23) - __float_as_uint(scale[g]));   // the reciprocal of a power of two
    for (int k = warp; k < STEPS; k += kThreads / 32) {
      const int at = ((k / 2) * 4 + t4) * 8 + (k & 1) * 4;              // of the row's 2 D: least keys, then greatest
      const float4 x = g < G ? __ldcg(reinterpret_cast<const float4*>(q + g * D + at % D)) : make_float4(0.f, 0.f, 0.f, 0.f);
      // (a NaN stays one in both)
      const bool least = at < D;
      const float y[4] = {(x.x < 0.f) == least ? x.x : x.x * 0.f, (x.y < 0.f) == least ? x.y : x.y * 0.f,
                          (x.z < 0.f) == least ? x.z : x.z * 0.f, (x.w < 0.f) == least ? x.w : x.w * 0.f};
      const Parts<T> p0 = parts<T>(y[0] * down, y[1] * down), p1 = parts<T>(y[2] * down, y[3] * down);
#pragma unroll
      for (int c = 0; c < NT; c++)
        qf[(k * NT + c) * 32 + lane] = GP == 8 ? make_uint2(p0.w[c], p1.w[c])
                                               : (g4 < 4 ? make_uint2(p0.w[2 * c], p1.w[2 * c])
                                                         : make_uint2(p0.w[2 * c + 1], p1.w[2 * c + 1]));
    }
  }
  __syncthreads();

  // Every page to f32 accuracy.
  uint32_t largest = 0, used = 0;
  const float c0 = scale[(2 * t4) % GP], c1 = scale[(2 * t4 + 1) % GP];
  const bool has0 = (2 * t4) % GP < G, has1 = (2 * t4 + 1) % GP < G;
  for (uint32_t tile = warp; tile * 16 < n; tile += kThreads / 32) {
    const uint32_t mine = look(tile);
    float sum[NT][4];
#pragma unroll
    for (int c = 0; c < NT; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) sum[c][i] = 0.f;
#pragma unroll 1
    for (uint32_t st = 0; st < STAGES; st++, used++) {
      copy_wait<kStages - 2>();
      const uint4* at = ring + (used % kStages) * 4 * 32;
      const uint4 r0 = at[0], r1 = at[32], r2 = at[64], r3 = at[96];
      fetch();
      const uint32_t words[16] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w, r2.x, r2.y, r2.z, r2.w, r3.x, r3.y, r3.z, r3.w};
#pragma unroll
      for (int i = 0; i < 16; i++) largest = greater_size<T>(largest, words[i]);
      const uint32_t a0[4] = {r0.x, r1.x, r0.y, r1.y}, a1[4] = {r0.z, r1.z, r0.w, r1.w};
      const uint32_t a2[4] = {r2.x, r3.x, r2.y, r3.y}, a3[4] = {r2.z, r3.z, r2.w, r3.w};
#pragma unroll
      for (int c = 0; c < NT; c++) {
        const uint2* b = qf + (st * 4 * NT + c) * 32 + lane;
        const uint2 b0 = b[0], b1 = b[NT * 32], b2 = b[2 * NT * 32], b3 = b[3 * NT * 32];
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
        mma<T>(x, a0, b0.x, b0.y);
        mma<T>(y, a2, b2.x, b2.y);
        mma<T>(x, a1, b1.x, b1.y);
        mma<T>(y, a3, b3.x, b3.y);
#pragma unroll
        for (int i = 0; i < 4; i++) sum[c][i] += x[i] + y[i];
      }
    }
    // Rows g4 and g4 + 8, columns 2 t4 and 2 t4 + 1: the heads' parts together, the largest of the heads.
    uint32_t best[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      float x = sum[0][2 * r], y = sum[0][2 * r + 1];
#pragma unroll
      for (int c = 1; c < NT; c++) x += sum[c][2 * r], y += sum[c][2 * r + 1];
      if (GP == 4) x += __shfl_xor_sync(0xffffffffu, x, 2), y += __shfl_xor_sync(0xffffffffu, y, 2);
      best[r] = max(has0 ? order(x * c0) : 0u, has1 ? order(y * c1) : 0u);
      best[r] = max(best[r], __shfl_xor_sync(0xffffffffu, best[r], 1));
      if (GP == 8) best[r] = max(best[r], __shfl_xor_sync(0xffffffffu, best[r], 2));
      const uint32_t i = tile * 16 + g4 + 8 * r, page = __shfl_sync(0xffffffffu, mine, g4 + 8 * r);
      if (t4 == 0 && i < n) {
        keys[i] = page < v.pages ? best[r] : 0u;
        if (page >= v.pages) note(v, FZ_PAGED_BAD_PAGE);
      }
    }
  }
  copy_wait<0>();
  const float2 sizes = T::unpack(largest);
  const float warp_largest = warp_max(fmaxf(sizes.x, sizes.y));
  if (lane == 0) bound[warp] = warp_largest;
  __syncthreads();
  cluster.barrier_wait();
  if (warp == 0) tell(whole, sh.bound, warp_max(lane < kThreads / 32 ? bound[lane] : 0.f));
  if (alone && rank) {
    uint32_t* all = cluster.map_shared_rank(keys, 0) + first;
    for (uint32_t i = t; i < n; i += kThreads) all[i] = keys[i];
  }
  if (alone) cluster.sync();
  else __syncthreads();

  // q again, for the listed pages' scores (asked for here, needed after the choice).
  constexpr int QN = (GP * D + kThreads - 1) / kThreads;
  float again[QN];
#pragma unroll
  for (int i = 0; i < QN; i++) {
    const uint32_t at = t + i * kThreads;
    again[i] = scores && at < G * D ? __ldcg(q + at) : 0.f;
  }

  // The threshold among them, by the first CTA alone or by all (their first
  // barrier makes the bounds seen).
  const uint32_t take = min(a.top, pages);
  const Forced forced = forced_of(pages, a.sink, a.recent);
  bool refine = false;                             // too many near T for the first CTA: all of them score theirs in f64
  Threshold<uint32_t> r{};
  Range<uint32_t> near_t{0, 0};                    // the keys near T
  if (!alone || rank == 0) {
    const Group group = one ? single : whole;
    const uint32_t from = one ? 0u : first, count = one ? pages : n;
    r = one ? find_alone(sh, keys, count, take, forced) : find(group, sh, keys, count, from, take, forced);
    bool by_bit = false;
    if (!r.every && !r.none) {
      float m = 0.f, norms = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; c++) m = c < (int)size ? fmaxf(m, sh.bound[c]) : m;
#pragma unroll
      for (int g = 0; g < GP; g++) norms = g < (int)G && (norm[g] > norms || norm[g] != norm[g]) ? norm[g] : norms;   // (NaN stays)
      const float e = 2.f * 5.9604645e-8f * (norms * fmaxf(m, 1e-26f)) + 1e-40f;
      // The ends' scores, as topk_key orders them.  (A NaN threshold: ties by the index, as in f64.)
      const float tl = __uint_as_float(topk_bits(r.prefix)), th = __uint_as_float(topk_bits(r.prefix | ~r.mask));
      const bool vague = !(e < INFINITY);          // every page is near (but those that are no pages, key 0)
      near_t.low = vague ? 1u : max(1u, order(tl - e)), near_t.high = vague ? ~0u : order(th == th ? th + e : INFINITY);
      uint32_t in = 0, near = 0;
      for (uint32_t i = t; i < count; i += kThreads) {
        const int z = forced(from + i) ? 0 : near_t.side(keys[i]);
        in += z == 2, near += z == 1;
        if (z == 1 && one) {
          const uint32_t at = atomicAdd(&nears, 1u);
          if (at < kNear) near_at[at] = i;
        }
      }
      in = __reduce_add_sync(0xffffffffu, in), near = __reduce_add_sync(0xffffffffu, near);
      __syncthreads();
      if (lane == 0) sh.warp[0][warp] = in, sh.warp[1][warp] = near;
      __syncthreads();
      if (!one && warp == 0) {
        in = lane < kThreads / 32 ? sh.warp[0][lane] : 0u, near = lane < kThreads / 32 ? sh.warp[1][lane] : 0u;
        in = __reduce_add_sync(0xffffffffu, in), near = __reduce_add_sync(0xffffffffu, near);
        tell(group, sh.zones, make_uint2(in, near));
      }
      if (!one) sync(group);
      in = near = 0;
      if (one)
        for (int w = 0; w < kThreads / 32; w++) in += sh.warp[0][w], near += sh.warp[1][w];
      else
        for (uint32_t c = 0; c < size; c++) in += sh.zones[c].x, near += sh.zones[c].y;
      // (Fewer: the threshold is among what are no pages, and ties there go by the index.)
      refine = (vague || tl == tl) && in + near > r.want;
      if (refine && one && near <= kNear) {
        // The near pages' f64 scores, and their order among one another.
        refine = false, by_bit = true;
        for (uint32_t i = warp; i < near; i += kThreads / 32) {
          const double d = page_score<T, D>(a, q, table[near_at[i]], h, lane);
          if (lane == 0) near_key[i] = order(d);
        }
        __syncthreads();
        if (t < (int)near) {
          uint32_t ahead_of = 0;
          for (uint32_t i = 0; i < near; i++)
            ahead_of += near_key[i] > near_key[t] || (near_key[i] == near_key[t] && near_at[i] < near_at[t]);
          if (ahead_of < r.want - in) atomicOr(&chosen[near_at[t] / 32], 1u << (near_at[t] % 32));
        }
        __syncthreads();
      }
    }
    const Range<uint32_t> cut = by_bit ? near_t : range_of(r);
    if (!refine)
      emit_taken(
          group, sh, count, r.ties,
          [&](uint32_t i) {
            const int z = forced(from + i) ? 2 : cut.side(keys[i]);
            return z == 1 && by_bit ? (int)(chosen[i / 32] >> (i % 32) & 1) * 2 : z;
          },
          [&](uint32_t i, uint32_t at) { out[at] = from + i; });
  }
  double* lifted = reinterpret_cast<double*>(qf);  // (q's operands, 32 D bytes or more a four heads, are done with)
#pragma unroll
  for (int i = 0; i < QN; i++) {
    const uint32_t at = t + i * kThreads;
    if (at < GP * D) lifted[lifted_place<D>(at / D, at % D)] = (double)again[i] * __hiloint2double((1023 + kLift) << 20, 0);
  }
  if (alone) {
    if (rank == 0 && warp == 0 && t < (int)size)
      *cluster.map_shared_rank(&sh.verdict, t) = make_uint4(refine, near_t.low, near_t.high, 0);
    cluster.sync();
    refine = sh.verdict.x != 0, near_t = Range<uint32_t>{sh.verdict.y, sh.verdict.z};
  }
  if (refine) {
    // The near pages in f64, a CTA its own; the rest of the choice is made.
    auto taken_first = [&](uint32_t i, uint64_t = 0) { return forced(i) || near_t.side(keys[i - first]) == 2; };
    for (uint32_t i = warp; i < n; i += kThreads / 32) {
      double d = 0.0;
      const bool near = !forced(first + i) && near_t.side(keys[i]) == 1;
      if (near) d = page_score<T, D>(a, q, table[first + i], h, lane);
      if (lane == 0) exact[i] = near ? order(d) : 0ull;
    }
    __syncthreads();
    const Threshold<uint64_t> r64 = find(whole, sh, exact, n, first, take, taken_first);
    const Range<uint64_t> cut = range_of(r64);
    emit_taken(
        whole, sh, n, r64.ties, [&](uint32_t i) { return taken_first(first + i) ? 2 : cut.side(exact[i]); },
        [&](uint32_t i, uint32_t at) { out[at] = first + i; });
  }
  if (!scores) return;
  // The listed pages' scores, in f64, by all warps.  (A barrier since the list was written; one is past where the
  // first CTA wrote it alone.)
  if (refine || !alone) sync(whole);
  listed_scores<T, D, GP>(a, q, lifted, h, table, out, scores, take, warp * size + rank, size * (kThreads / 32));
}

// ------------------------------------------------------------ eviction

struct EvictArgs {
  PagedView from, to;
  uint32_t budget, sink, recent;
  uint32_t* kept;
};

// The choice: 4 bytes an entry read, so bound by its barriers: 8 sequences of up
// to 32,640 entries and 2 KV heads 18 us (49 while CTAs read one another's counts
// instead of being told them), 1,500 entries 6 us.
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
  // (A barrier of the choice lies between these and the entries taken.)
  for (uint32_t i = rank * kThreads + threadIdx.x; i < a.budget; i += size * kThreads) out[i] = FZ_PAGED_NONE;
  const uint32_t per = (entries + size - 1) / size, first = min(entries, rank * per), n = min(entries, first + per) - first;
  const uint32_t* table = v.table + (size_t)s * v.table_stride;
  for (uint32_t i0 = threadIdx.x; i0 < n; i0 += BATCH * kThreads) {
    uint32_t page[BATCH], slot[BATCH];
    float w[BATCH];
#pragma unroll
    for (int c = 0; c < BATCH; c++) {
      const uint32_t i = i0 + c * kThreads, j = first + i;
      const uint32_t logical = j / v.slots;
      page[c] = i < n ? table[logical] : FZ_PAGED_NONE;
      slot[c] = j - logical * v.page_slots;
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
  // (Entries of pages that are none, key 0, are not forced, chosen last and never taken.)
  const Forced ends = forced_of(entries, a.sink, a.recent);
  auto forced = [&](uint32_t i, uint32_t key) { return ends(i) && key; };
  const Group group = size == 1 ? Group{nullptr, 1, 0} : Group{&cluster, size, rank};
  const Threshold<uint32_t> r = size == 1 ? find_alone(sh, keys, n, min(a.budget, entries), forced)
                                          : find(group, sh, keys, n, first, min(a.budget, entries), forced);
  const Range<uint32_t> cut = range_of(r);
  emit_taken(
      group, sh, n, r.ties, [&](uint32_t i) {
        const uint32_t k = keys[i];
        return !k ? 0 : ends(first + i) ? 2 : cut.side(k);
      },
      [&](uint32_t i, uint32_t at) { out[at] = first + i; });
}

// The kept entries' keys and values, D / 8 lanes an entry, 16 bytes a lane, four
// steps' loads at once; their weights; and the new length.  Memory bound: 4 x D
// bytes read and written an entry: 8 sequences, 2 KV heads, 4,080 entries, 134 MB,
// 21 us (6.4 TB/s; 4 bytes a lane and a warp an entry: 45).
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
    const uint32_t from = f.table[(size_t)s * f.table_stride + j / f.slots],
                   to = t.table[(size_t)s * t.table_stride + r / t.slots];
    ok = from < f.pages && to < t.pages;
    if (to >= t.pages) note(t, FZ_PAGED_BAD_PAGE);
    if (ok) {
      src = element(f, from, j % f.slots, h), dst = element(t, to, r % t.slots, h);
      if (t.weights)
        t.weights[((size_t)to * t.kv_heads + h) * t.page_slots + r % t.slots] =
            __ldcg(f.weights + ((size_t)from * f.kv_heads + h) * f.page_slots + j % f.slots);
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

// CTAs a cluster: as many as fill the GPU once while each has `worth` keys, and
// at least enough that the slices fit shared memory; 0 when even the widest
// cluster's do not.
uint32_t cluster_for(uint64_t items, uint64_t longest, uint32_t worth, size_t key_bytes, size_t room) {
  uint32_t c = 1;
  while (c < kMaxCluster && ((longest + c - 1) / c * key_bytes > room || (items * c * 2 <= 148 && longest / c > worth))) c *= 2;
  return (longest + c - 1) / c * key_bytes > room ? 0 : c;
}

constexpr size_t kRoom = 196 * 1024;
constexpr uint32_t kMostListed = 1u << 30; // as many as a table may have (counters of 32 bits run over lists in steps)
constexpr size_t kOperands = 24 * 1024;    // q's, at most
constexpr size_t kPagesRoom = 58 * 1024;   // beside the ring and those
template <class T, int D>
const void* select_of(bool many) {
  return many ? (const void*)select_kernel<T, D, 8> : (const void*)select_kernel<T, D, 4>;
}

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
  if (top > kMostListed) return paged_refuse(FZ_ERR_ARGUMENT, "top of more than 2^30");
  if (top == 0 || (uint64_t)sink + recent > top) return paged_refuse(FZ_ERR_ARGUMENT, "top must be nonzero and at least sink + recent");
  const uint64_t items = (uint64_t)kv->sequences * kv->kv_heads;
  const uint32_t c = cluster_for(items, kv->table_stride, 32, 13, kPagesRoom);
  if (!c) return paged_refuse(FZ_ERR_NOT_SUPPORTED, "more pages a sequence than a cluster's shared memory holds scores of (36,000)");
  if (items * c > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many sequences");
  if (items == 0) return FZ_OK;
  const void* p[] = {kv->page_table, kv->lengths, kv->bounds, kv->error, q, blocks, scores};
  if ((st = paged_on_device(p, 7, "fz_paged_select"))) return st;
  a.q = q, a.q_stride = q_stride, a.group = heads / kv->kv_heads;
  a.top = top, a.sink = sink, a.recent = recent, a.blocks = blocks, a.scores = scores;
  const uint32_t d = kv->head_dim;
  uint32_t slice = (kv->table_stride + c - 1) / c;
  slice += slice & 1;
  // The first CTA takes all scores where it has the room for them.
  uint32_t together = (kv->table_stride + 31) / 32 * 32;
  if (together * 4ull + slice * 8ull > kPagesRoom - 8192) together = 0;
  void* args[] = {&a, &slice, &together};
  const bool f16 = kv->type == FZ_KV_F16, many = a.group > 4;
  const uint32_t tiles = f16 ? (many ? 2 : 1) : (many ? 3 : 2), all = together ? together : slice;
  const void* fn = f16 ? (d == 64    ? select_of<F16, 64>(many)
                          : d == 128 ? select_of<F16, 128>(many)
                                     : select_of<F16, 256>(many))
                       : (d == 64    ? select_of<Bf16, 64>(many)
                          : d == 128 ? select_of<Bf16, 128>(many)
                                     : select_of<Bf16, 256>(many));
  return paged_launch(fn, dim3((uint32_t)(items * c)), dim3(kThreads),
                      kRing + d / 8 * tiles * 256 + slice * 8 + all * 4 + (all + 31) / 32 * 4, kRing + kOperands + kPagesRoom, c, args,
                      stream);
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
  if (budget > kMostListed) return paged_refuse(FZ_ERR_ARGUMENT, "budget of more than 2^30");
  const uint64_t longest = (uint64_t)from->table_stride * from->page_slots, room = (uint64_t)to->table_stride * to->page_slots;
  if (std::min<uint64_t>(budget, longest) > room) return paged_refuse(FZ_ERR_ARGUMENT, "budget past the destination's table");
  const uint64_t items = (uint64_t)from->sequences * from->kv_heads;
  if (items > 65535) return paged_refuse(FZ_ERR_ARGUMENT, "more than 65,535 sequences times KV heads");
  // (One CTA chooses among 4,096 entries sooner than a cluster agrees: 1,500 entries 12.5 us by eight, 7.9 by one.)
  const uint32_t c = cluster_for(items, longest, 4096, 4, kRoom);
  if (!c) return paged_refuse(FZ_ERR_NOT_SUPPORTED, "more entries a sequence than a cluster's shared memory holds weights of (401,000)");
  if (items == 0) return FZ_OK;
  const void* p[] = {from->keys, from->values, from->page_table, from->lengths, from->weights, from->error,
                     to->keys,   to->values,   to->page_table,   to->lengths,   to->weights,   to->error, kept};
  if ((st = paged_on_device(p, 13, "fz_paged_evict"))) return st;
  a.budget = budget, a.sink = sink, a.recent = recent, a.kept = kept;
  uint32_t slice = (uint32_t)((longest + c - 1) / c);
  void* args[] = {&a, &slice};
  if ((st = paged_launch((const void*)keep_kernel, dim3((uint32_t)(items * c)), dim3(kThreads), slice * 4, kRoom, c, args, stream)))
    return st;
  void* move[] = {&a};
  const uint32_t rows = 8 * 4 * (256 / from->head_dim);    // a CTA's entries
  const void* fn = from->head_dim == 64    ? (const void*)move_kernel<64>
                   : from->head_dim == 128 ? (const void*)move_kernel<128>
                                           : (const void*)move_kernel<256>;
  return paged_launch(fn, dim3((uint32_t)((std::min<uint64_t>(budget, longest) + rows - 1) / rows), (uint32_t)items), dim3(256), 0, 0, 1,
                      move, stream);
}

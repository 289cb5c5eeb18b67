// Choosing among what a paged cache holds: the pages a query attends to
// (fz_paged_select) and the entries an eviction keeps (fz_paged_evict).
//
// Both take the best `take` of a (sequence, KV head)'s n scores, ties to the
// lower index.  A cluster of CTAs takes one (sequence, KV head): each CTA holds
// the keys of a contiguous slice in shared memory, order-preserving unsigned
// integers of the scores, and the cluster finds the take-th largest digit by
// digit from the top: a histogram a CTA, read by all the others through
// distributed shared memory, the digit that the take-th falls into, and on
// with that digit's keys only.  One pass over the slice at the end writes the
// chosen indices in ascending order, each at its rank.
#include "paged.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace fz {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 2048;           // 11 bits a digit
constexpr int kMaxCluster = 8;

// Shared by the CTAs of a cluster.
struct Shared {
  uint32_t bins[kBins];
  uint32_t warp[2][kThreads / 32];
  uint32_t more, equal;               // this CTA's keys above the threshold, and equal to it
  uint32_t digit, above, at_digit;
};

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

// The best `take` of the cluster's keys (this CTA's: keys[0 .. n), of indices
// first ..; `forced(i)` ones come first and are part of `take`), ascending:
// emit(index, rank) for each.  kBits: the keys' width.
template <int kBits, class K, class Forced, class Emit>
FZ_DEV void choose(cg::cluster_group& cluster, Shared& sh, const K* keys, uint32_t n, uint32_t first, uint32_t take,
                   Forced forced, Emit emit) {
  const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
  const int t = threadIdx.x;
  // How many are not forced, and how many of those are wanted.
  uint32_t free_keys = 0, pinned = 0;
  for (uint32_t i = t; i < n; i += kThreads) {
    const bool f = forced(first + i);
    pinned += f, free_keys += !f;
  }
  block_scan(sh, make_uint2(free_keys, pinned));
  cluster.sync();
  uint32_t all = 0, all_pinned = 0;
  for (uint32_t c = 0; c < size; c++) {
    const Shared* o = cluster.map_shared_rank(&sh, c);
    all += o->more, all_pinned += o->equal;
  }
  uint32_t want = take > all_pinned ? take - all_pinned : 0u;
  K prefix = 0, mask = 0;
  uint32_t ties = 0;                     // keys with `prefix` under `mask` to take, lowest index first
  bool every = false;                    // all of those
  if (want >= all) {
    every = true, ties = all;            // (mask 0: every key has the prefix)
  } else if (want) {
    int high = kBits;
    while (high > 0) {
      const int bits = high < 11 ? high : 11, shift = high - bits;
      const uint32_t bins = 1u << bits;
      cluster.sync();                    // (the last digit's bins are read)
      for (uint32_t i = t; i < bins; i += kThreads) sh.bins[i] = 0;
      __syncthreads();
      for (uint32_t i = t; i < n; i += kThreads) {
        const K k = keys[i];
        if ((k & mask) == prefix && !forced(first + i)) atomicAdd(&sh.bins[(uint32_t)(k >> shift) & (bins - 1)], 1u);
      }
      cluster.sync();
      // Thread t: bins from the top, 4 (of 2048) a thread, summed over the cluster.
      const uint32_t per = (bins + kThreads - 1) / kThreads;
      uint32_t count[4] = {0, 0, 0, 0}, sum = 0;
      for (uint32_t i = 0; i < per; i++) {
        const uint32_t b = t * per + i;
        if (b < bins)
          for (uint32_t c = 0; c < size; c++) count[i] += cluster.map_shared_rank(sh.bins, c)[bins - 1 - b];
        sum += count[i];
      }
      uint32_t before = block_scan(sh, make_uint2(sum, 0u)).x;
      for (uint32_t i = 0; i < per; i++) {
        if (before < want && want <= before + count[i]) {
          sh.digit = bins - 1 - (t * per + i);
          sh.above = before;
          sh.at_digit = count[i];
        }
        before += count[i];
      }
      __syncthreads();
      want -= sh.above;
      prefix |= (K)sh.digit << shift;
      mask |= (K)(bins - 1) << shift;
      ties = want;
      high = shift;
      if (want == sh.at_digit) break;    // the digit's keys are all taken
    }
  }
  // Each thread a run of the slice: its keys above the threshold (or forced), and equal to it.
  const uint32_t run = (n + kThreads - 1) / kThreads, i0 = min(n, t * run), i1 = min(n, i0 + run);
  const bool none = want == 0 && !every;
  auto state = [&](uint32_t i) -> int {  // 2 taken, 1 equal, 0 not
    if (forced(first + i)) return 2;
    if (none) return 0;
    const K k = keys[i] & mask;
    return k > prefix ? 2 : k == prefix ? 1 : 0;
  };
  uint2 mine = make_uint2(0, 0);
  for (uint32_t i = i0; i < i1; i++) {
    const int s = state(i);
    mine.x += s == 2, mine.y += s == 1;
  }
  cluster.sync();                        // (more and equal of the last scan are read)
  uint2 at = block_scan(sh, mine);
  cluster.sync();
  for (uint32_t c = 0; c < rank; c++) {
    const Shared* o = cluster.map_shared_rank(&sh, c);
    at.x += o->more, at.y += o->equal;
  }
  for (uint32_t i = i0; i < i1; i++) {
    const int s = state(i);
    if (s == 2 || (s == 1 && at.y < ties)) emit(first + i, i, at.x + min(at.y, ties));
    at.x += s == 2, at.y += s == 1;
  }
  cluster.sync();                        // (no CTA leaves while another reads its shared memory)
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

template <class T, int D>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectArgs a, uint32_t slice) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint64_t* keys = reinterpret_cast<uint64_t*>(dyn);
  float* q = reinterpret_cast<float*>(keys + slice);
  cg::cluster_group cluster = cg::this_cluster();
  pdl_wait();
  const PagedView& v = a.kv;
  const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
  const uint64_t item = blockIdx.x / size;
  const uint32_t s = (uint32_t)(item / v.kv_heads), h = (uint32_t)(item % v.kv_heads);
  const uint32_t entries = held(v, s);
  if (threadIdx.x == 0 && rank == 0 && v.lengths[s] > entries) note(v, FZ_PAGED_BAD_LENGTH);
  const uint32_t pages = (entries + v.page_slots - 1) / v.page_slots;
  uint32_t* out = a.blocks + item * a.top;
  float* scores = a.scores ? a.scores + item * a.top : nullptr;
  for (uint32_t i = min(pages, a.top) + rank * kThreads + threadIdx.x; i < a.top; i += size * kThreads) {
    out[i] = FZ_PAGED_NONE;
    if (scores) scores[i] = 0.f;
  }
  const uint32_t per = (pages + size - 1) / size, first = min(pages, rank * per), n = min(pages, first + per) - first;
  for (uint32_t i = threadIdx.x; i < a.group * D; i += kThreads) q[i] = a.q[s * a.q_stride + (size_t)h * a.group * D + i];
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (uint32_t i = threadIdx.x >> 5; i < n; i += kThreads / 32) {
    const uint32_t page = v.table[(size_t)s * v.table_stride + first + i];
    const bool ok = page < v.pages;
    const double d = ok ? page_score<T, D>(a, q, page, h, lane) : 0.0;
    if (!ok && lane == 0) note(v, FZ_PAGED_BAD_PAGE);
    if (lane == 0) keys[i] = ok ? order(d) : 0ull;
  }
  __syncthreads();
  choose<64>(cluster, sh, keys, n, first, min(a.top, pages),
             [&](uint32_t i) { return i < a.sink || i + a.recent >= pages; },
             [&](uint32_t page, uint32_t i, uint32_t r) {
               out[r] = page;
               if (!scores) return;
               const uint64_t k = keys[i];
               scores[r] = (float)__longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
             });
}

// ------------------------------------------------------------ eviction

struct EvictArgs {
  PagedView from, to;
  uint32_t budget, sink, recent;
  uint32_t* kept;
};

__global__ void __launch_bounds__(kThreads) keep_kernel(const EvictArgs a, uint32_t slice) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint32_t* keys = reinterpret_cast<uint32_t*>(dyn);
  cg::cluster_group cluster = cg::this_cluster();
  pdl_wait();
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
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t j = first + i, page = v.table[(size_t)s * v.table_stride + j / v.page_slots];
    const bool ok = page < v.pages;
    if (!ok) note(v, FZ_PAGED_BAD_PAGE);
    keys[i] = ok ? order(v.weights[((size_t)page * v.kv_heads + h) * v.page_slots + j % v.page_slots]) : 0u;
  }
  __syncthreads();
  choose<32>(cluster, sh, keys, n, first, min(a.budget, entries),
             [&](uint32_t i) { return i < a.sink || i + a.recent >= entries; },
             [&](uint32_t j, uint32_t, uint32_t r) { out[r] = j; });
}

// A warp a kept entry: its key and value rows, its weight, and the new length.
template <int D>
__global__ void __launch_bounds__(256) move_kernel(const EvictArgs a) {
  pdl_wait();
  const PagedView &f = a.from, &t = a.to;
  const int lane = threadIdx.x & 31;
  const uint32_t h = blockIdx.y % f.kv_heads, s = blockIdx.y / f.kv_heads;
  const uint32_t r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= a.budget) return;
  const uint32_t* kept = a.kept + (size_t)blockIdx.y * a.budget;
  const uint32_t j = kept[r];
  if (lane == 0 && h == 0) {
    if (j == FZ_PAGED_NONE) {
      if (r == 0) t.lengths[s] = 0;
    } else if (r + 1 == a.budget || kept[r + 1] == FZ_PAGED_NONE) {
      t.lengths[s] = r + 1;
    }
  }
  if (j == FZ_PAGED_NONE) return;
  const uint32_t from = f.table[(size_t)s * f.table_stride + j / f.page_slots], to =
      r / t.page_slots < t.table_stride ? t.table[(size_t)s * t.table_stride + r / t.page_slots] : FZ_PAGED_NONE;
  if (from >= f.pages || to >= t.pages) {
    if (lane == 0 && to >= t.pages) note(t, FZ_PAGED_BAD_PAGE);
    return;
  }
  const uint32_t *ks = reinterpret_cast<const uint32_t*>(f.keys + element(f, from, j % f.page_slots, h)),
                 *vs = reinterpret_cast<const uint32_t*>(f.values + element(f, from, j % f.page_slots, h));
  uint32_t *kd = reinterpret_cast<uint32_t*>(t.keys + element(t, to, r % t.page_slots, h)),
           *vd = reinterpret_cast<uint32_t*>(t.values + element(t, to, r % t.page_slots, h));
#pragma unroll
  for (int c = 0; c < D / 64; c++) kd[lane + 32 * c] = ks[lane + 32 * c], vd[lane + 32 * c] = vs[lane + 32 * c];
  if (lane == 0 && t.weights)
    t.weights[((size_t)to * t.kv_heads + h) * t.page_slots + r % t.page_slots] =
        f.weights[((size_t)from * f.kv_heads + h) * f.page_slots + j % f.page_slots];
}

// CTAs a cluster: as many as fill the GPU once, at least enough that the
// slices fit shared memory; 0 when even the widest cluster's do not.
uint32_t cluster_for(uint64_t items, uint64_t longest, size_t key_bytes, size_t room) {
  uint32_t c = 1;
  while (c < kMaxCluster && ((longest + c - 1) / c * key_bytes > room || (items * c < 148 && longest / c > 256))) c *= 2;
  return (longest + c - 1) / c * key_bytes > room ? 0 : c;
}

constexpr size_t kRoom = 200 * 1024;

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
  const uint32_t c = cluster_for(items, kv->table_stride, 8, kRoom);
  if (!c) return paged_refuse(FZ_ERR_NOT_SUPPORTED, "more pages a sequence than a cluster's shared memory holds scores of (204,800)");
  if (items * c > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many sequences");
  if (items == 0) return FZ_OK;
  const void* p[] = {kv->page_table, kv->lengths, kv->bounds, kv->error, q, blocks, scores};
  if ((st = paged_on_device(p, 7, "fz_paged_select"))) return st;
  a.q = q, a.q_stride = q_stride, a.group = heads / kv->kv_heads;
  a.top = top, a.sink = sink, a.recent = recent, a.blocks = blocks, a.scores = scores;
  uint32_t slice = (kv->table_stride + c - 1) / c;
  slice += slice & 1;
  void* args[] = {&a, &slice};
  const bool f16 = kv->type == FZ_KV_F16;
  const uint32_t d = kv->head_dim;
  const void* fn = f16 ? (d == 64    ? (const void*)select_kernel<F16, 64>
                          : d == 128 ? (const void*)select_kernel<F16, 128>
                                     : (const void*)select_kernel<F16, 256>)
                       : (d == 64    ? (const void*)select_kernel<Bf16, 64>
                          : d == 128 ? (const void*)select_kernel<Bf16, 128>
                                     : (const void*)select_kernel<Bf16, 256>);
  return paged_launch(fn, dim3((uint32_t)(items * c)), dim3(kThreads), slice * 8 + a.group * d * 4, c, args, stream);
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
  if (!c) return paged_refuse(FZ_ERR_NOT_SUPPORTED, "more entries a sequence than a cluster's shared memory holds weights of (409,600)");
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
  const void* fn = from->head_dim == 64    ? (const void*)move_kernel<64>
                   : from->head_dim == 128 ? (const void*)move_kernel<128>
                                           : (const void*)move_kernel<256>;
  return paged_launch(fn, dim3((uint32_t)((std::min<uint64_t>(budget, longest) + 7) / 8), (uint32_t)items), dim3(256), 0, 1,
                      move, stream);
}

// The paged cache's host checks, the append (QK-norm, rotation and store in
// one pass) and the pages' key bounds.
#include "paged.cuh"

#include <algorithm>
#include <cmath>
#include <cstdio>

#include "last_error.h"

namespace fz {

fz_status paged_refuse(fz_status s, const char* why) {
  set_last_error(why);
  return s;
}

fz_status paged_on_device(const void* const* pointers, int count, const char* what) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  for (int i = 0; e == cudaSuccess && i < count; i++) {
    if (!pointers[i]) continue;
    cudaPointerAttributes a{};
    e = cudaPointerGetAttributes(&a, pointers[i]);
    if (e != cudaSuccess) break;
    if (a.type == cudaMemoryTypeUnregistered || (a.type == cudaMemoryTypeDevice && a.device != device)) {
      char why[96];
      std::snprintf(why, sizeof(why), "%s: a pointer that is not memory of the current device", what);
      return paged_refuse(FZ_ERR_ARGUMENT, why);
    }
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return paged_refuse(FZ_ERR_CUDA, cudaGetErrorString(e));
  }
  return FZ_OK;
}

fz_status paged_view(const fz_paged_kv* kv, uint32_t need, PagedView* out) {
  if (!kv) return paged_refuse(FZ_ERR_ARGUMENT, "null cache description");
  if (kv->type > FZ_KV_BF16) return paged_refuse(FZ_ERR_ARGUMENT, "cache type other than f16 or bf16");
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
    return paged_refuse(FZ_ERR_NOT_SUPPORTED, "head dimension other than 64, 128 or 256");
  if (!kv->kv_heads || !kv->page_slots || !kv->pages || !kv->table_stride)
    return paged_refuse(FZ_ERR_ARGUMENT, "kv_heads, page_slots, pages and table_stride must be nonzero");
  if (kv->kv_heads > 65535) return paged_refuse(FZ_ERR_ARGUMENT, "more than 65,535 KV heads");
  // (Counters of 32 bits run over them in steps.)
  if ((uint64_t)kv->sequences * kv->kv_heads > 0x7FFFFFFFull)
    return paged_refuse(FZ_ERR_ARGUMENT, "more than 2^31 - 1 sequences times KV heads");
  if ((uint64_t)kv->table_stride * kv->page_slots > (1u << 30))
    return paged_refuse(FZ_ERR_ARGUMENT, "a table of more than 2^30 entries a sequence");
  if (!kv->page_table || !kv->lengths) return paged_refuse(FZ_ERR_ARGUMENT, "null page table or lengths");
  if (need & kNeedKeys) {
    if (!kv->keys || !kv->values) return paged_refuse(FZ_ERR_ARGUMENT, "null keys or values");
    if ((reinterpret_cast<uintptr_t>(kv->keys) | reinterpret_cast<uintptr_t>(kv->values)) & 15u)
      return paged_refuse(FZ_ERR_ARGUMENT, "keys or values not 16-byte aligned");
    if ((kv->page_stride | kv->slot_stride | kv->head_stride) & 7u)
      return paged_refuse(FZ_ERR_ARGUMENT, "cache strides must be multiples of 8 elements");
    if ((kv->pages > 1 && kv->page_stride < kv->head_dim) || (kv->page_slots > 1 && kv->slot_stride < kv->head_dim) ||
        (kv->kv_heads > 1 && kv->head_stride < kv->head_dim))
      return paged_refuse(FZ_ERR_ARGUMENT, "a cache stride shorter than the head dimension");
  }
  if (need & kNeedBounds) {
    if (!kv->bounds) return paged_refuse(FZ_ERR_ARGUMENT, "null bounds");
    if (reinterpret_cast<uintptr_t>(kv->bounds) & 15u) return paged_refuse(FZ_ERR_ARGUMENT, "bounds not 16-byte aligned");
  }
  if ((need & kNeedWeights) && !kv->weights) return paged_refuse(FZ_ERR_ARGUMENT, "null weights");
  if ((reinterpret_cast<uintptr_t>(kv->page_table) | reinterpret_cast<uintptr_t>(kv->lengths) |
       reinterpret_cast<uintptr_t>(kv->weights) | reinterpret_cast<uintptr_t>(kv->error)) & 3u)
    return paged_refuse(FZ_ERR_ARGUMENT, "table, lengths, weights or error not 4-byte aligned");
  *out = PagedView{static_cast<uint16_t*>(kv->keys), static_cast<uint16_t*>(kv->values), kv->page_table, kv->lengths,
                   kv->weights, static_cast<uint16_t*>(kv->bounds), kv->error, kv->page_stride, kv->slot_stride,
                   kv->head_stride, kv->sequences, kv->table_stride, kv->pages, kv->page_slots, kv->kv_heads,
                   divisor(kv->page_slots)};
  return FZ_OK;
}

fz_status paged_launch(const void* kernel, dim3 grid, dim3 block, size_t smem, size_t most, uint32_t cluster, void** args,
                       void* stream) {
  cudaError_t e = cudaSuccess;
  // (The limit is the function's, for all host threads: always the same one, so that a call with a short table never
  // lowers it between another's setting and launch.)
  if (smem > 16 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    e = cudaLaunchKernelExC(&cfg, kernel, args);
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return paged_refuse(FZ_ERR_CUDA, cudaGetErrorString(e));
  }
  return FZ_OK;
}

namespace {

// ------------------------------------------------------------ append

struct AppendArgs {
  PagedView kv;
  fz_paged_rows r;
};

// Norm, rotation and store in one pass over a row's heads: memory bound, 4 bytes
// read a value and 2 or 4 written.  A head is D / 8 lanes, four values of each
// half a lane (the rotation's pairs in one lane, 16-byte accesses); a warp takes
// PASSES times 256 / D heads of one row, all their loads first, so the row's
// sines and cosines are made once for them.  The sum of squares and the norm in
// f32; the angle's turns in f64 (position x turns loses its fraction in f32 past
// a few thousand positions), its fraction's sine and cosine in f32.  4,095 rows
// of 8 + 2 + 2 heads of 256, 92 MB: 20.7 us, 4.5 TB/s (a warp a head, with its
// own sines: 28 us; two heads a warp 21.7, six 25.9); 16,000 rows 5.5 TB/s; 16
// rows 2.5 us, a launch and four dependent reads.
template <class T, int D, int PASSES>
__global__ void __launch_bounds__(128) append_kernel(const AppendArgs a, uint32_t warps_a_row) {
  constexpr int LANES = D / 8, HEADS = 32 / LANES;
  pdl_wait();
  pdl_launch_dependents();
  const fz_paged_rows& r = a.r;
  const PagedView& v = a.kv;
  const int lane = threadIdx.x & 31, part = lane % LANES;
  const uint32_t heads = r.heads + 2 * v.kv_heads;
  const uint64_t warp = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint64_t row = (warp >> 32) ? warp / warps_a_row : (uint32_t)warp / warps_a_row;
  if (row >= r.rows) return;
  const uint32_t head0 = (uint32_t)(warp - row * warps_a_row) * (PASSES * HEADS) + lane / LANES;
  float4 x[PASSES], y[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; p++) {
    const uint32_t head = head0 + p * HEADS;
    if (head < heads) {
      const bool query = head < r.heads, value = head >= r.heads + v.kv_heads;
      const float* src = query   ? r.q + row * r.q_stride + (size_t)head * D
                         : value ? r.v + row * r.v_stride + (size_t)(head - r.heads - v.kv_heads) * D
                                 : r.k + row * r.k_stride + (size_t)(head - r.heads) * D;
      x[p] = __ldcs(reinterpret_cast<const float4*>(src) + part);
      y[p] = __ldcs(reinterpret_cast<const float4*>(src + D / 2) + part);
    } else {
      x[p] = y[p] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  const uint32_t seq = r.sequence ? r.sequence[row] : (uint32_t)row;
  const uint32_t index = r.index[row];
  if (seq == FZ_PAGED_NONE) return;
  const bool in_table = seq < v.sequences && index < v.table_stride * v.page_slots;
  const uint32_t page = in_table ? v.table[(size_t)seq * v.table_stride + index / v.slots] : 0u;
  const uint32_t slot = in_table ? index % v.slots : 0u;
  float sn[4], cs[4];
  if (r.turns) {
    const double pos = (double)(r.position ? r.position[row] : index);
    const double2 t0 = reinterpret_cast<const double2*>(r.turns)[2 * part], t1 = reinterpret_cast<const double2*>(r.turns)[2 * part + 1];
    const double turns[4] = {pos * t0.x, pos * t0.y, pos * t1.x, pos * t1.y};
#pragma unroll
    for (int i = 0; i < 4; i++) sincospif(2.0f * (float)(turns[i] - rint(turns[i])), &sn[i], &cs[i]);
  }
#pragma unroll
  for (int p = 0; p < PASSES; p++) {
    const uint32_t head = head0 + p * HEADS;
    const bool query = head < r.heads, value = head >= r.heads + v.kv_heads, any = head < heads;
    const float* gain = query ? r.q_gain : r.k_gain;
    const bool normed = any && !value && gain;
    float xs[4] = {x[p].x, x[p].y, x[p].z, x[p].w}, ys[4] = {y[p].x, y[p].y, y[p].z, y[p].w};
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) sum = fmaf(xs[i], xs[i], fmaf(ys[i], ys[i], sum));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!any) continue;
    if (normed) {
      const float inv = rsqrtf(fmaf(sum, 1.0f / D, r.eps));
      const float4 gx = reinterpret_cast<const float4*>(gain)[part], gy = reinterpret_cast<const float4*>(gain + D / 2)[part];
      const float g0[4] = {gx.x, gx.y, gx.z, gx.w}, g1[4] = {gy.x, gy.y, gy.z, gy.w};
#pragma unroll
      for (int i = 0; i < 4; i++) xs[i] = xs[i] * inv * g0[i], ys[i] = ys[i] * inv * g1[i];
    }
    if (!value && r.turns) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float u = xs[i], w = ys[i];
        xs[i] = u * cs[i] - w * sn[i];
        ys[i] = u * sn[i] + w * cs[i];
      }
    }
    if (query) {
      float* out = r.q_out + row * r.q_out_stride + (size_t)head * D;
      reinterpret_cast<float4*>(out)[part] = make_float4(xs[0], xs[1], xs[2], xs[3]);
      reinterpret_cast<float4*>(out + D / 2)[part] = make_float4(ys[0], ys[1], ys[2], ys[3]);
      continue;
    }
    const uint32_t h = value ? head - r.heads - v.kv_heads : head - r.heads;
    if (!in_table || page >= v.pages) {
      if (part == 0) note(v, in_table ? FZ_PAGED_BAD_PAGE : FZ_PAGED_BAD_ROW);
      continue;
    }
    uint16_t* dst = (value ? v.values : v.keys) + element(v, page, slot, h);
    reinterpret_cast<uint2*>(dst)[part] = make_uint2(T::pack(xs[0], xs[1]), T::pack(xs[2], xs[3]));
    reinterpret_cast<uint2*>(dst + D / 2)[part] = make_uint2(T::pack(ys[0], ys[1]), T::pack(ys[2], ys[3]));
    if (part == 0 && !value) {
      if (v.weights) v.weights[((size_t)page * v.kv_heads + h) * v.page_slots + slot] = 0.f;
      if (h == 0) atomicMax(v.lengths + seq, index + 1);
    }
  }
}

// ------------------------------------------------------------ bounds

constexpr uint32_t kWide = 128 * 256;        // a page's values of a head, from which a CTA takes it

struct BoundsArgs {
  PagedView kv;
  const uint32_t* first;
};

template <class T>
FZ_DEV uint32_t least2(uint32_t a, uint32_t b);
template <>
FZ_DEV uint32_t least2<F16>(uint32_t a, uint32_t b) {
  const __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
FZ_DEV uint32_t least2<Bf16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <class T>
FZ_DEV uint32_t most2(uint32_t a, uint32_t b);
template <>
FZ_DEV uint32_t most2<F16>(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
FZ_DEV uint32_t most2<Bf16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The least and greatest of a page's slots, D / 8 lanes a key and 16 bytes a
// lane, the other lanes of a warp (256 / D of them) every other slot, AHEAD
// loads in flight a lane; a page by one warp, or (WIDE) by the CTA's eight, which
// join in shared memory.
template <class T, int D, bool WIDE>
FZ_DEV void page_bounds(const PagedView& v, uint32_t page, uint32_t h, uint32_t slots, uint4 (*joined)[2][D / 8]) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES, AHEAD = WIDE ? 8 : 16, WARPS = WIDE ? 8 : 1;
  const int lane = threadIdx.x & 31, part = lane % LANES, warp = threadIdx.x >> 5;
  const uint16_t* k = v.keys + element(v, page, 0, h) + part * 8;
  // (Slots past the page's held ones repeat its first.)
  uint4 lo = *reinterpret_cast<const uint4*>(k), hi = lo;
  for (uint32_t i = (WIDE ? warp * ROWS : 0) + lane / LANES; i < slots; i += ROWS * AHEAD * WARPS) {
    uint4 x[AHEAD];
#pragma unroll
    for (int c = 0; c < AHEAD; c++) {
      const uint32_t j = i + c * ROWS * WARPS;
      x[c] = __ldcs(reinterpret_cast<const uint4*>(k + (j < slots ? j : 0u) * v.slot_stride));
    }
#pragma unroll
    for (int c = 0; c < AHEAD; c++) {
      lo = make_uint4(least2<T>(lo.x, x[c].x), least2<T>(lo.y, x[c].y), least2<T>(lo.z, x[c].z), least2<T>(lo.w, x[c].w));
      hi = make_uint4(most2<T>(hi.x, x[c].x), most2<T>(hi.y, x[c].y), most2<T>(hi.z, x[c].z), most2<T>(hi.w, x[c].w));
    }
  }
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1) {
    const uint4 l = make_uint4(__shfl_xor_sync(0xffffffffu, lo.x, o), __shfl_xor_sync(0xffffffffu, lo.y, o),
                               __shfl_xor_sync(0xffffffffu, lo.z, o), __shfl_xor_sync(0xffffffffu, lo.w, o));
    const uint4 m = make_uint4(__shfl_xor_sync(0xffffffffu, hi.x, o), __shfl_xor_sync(0xffffffffu, hi.y, o),
                               __shfl_xor_sync(0xffffffffu, hi.z, o), __shfl_xor_sync(0xffffffffu, hi.w, o));
    lo = make_uint4(least2<T>(lo.x, l.x), least2<T>(lo.y, l.y), least2<T>(lo.z, l.z), least2<T>(lo.w, l.w));
    hi = make_uint4(most2<T>(hi.x, m.x), most2<T>(hi.y, m.y), most2<T>(hi.z, m.z), most2<T>(hi.w, m.w));
  }
  uint4* b = reinterpret_cast<uint4*>(v.bounds + ((size_t)page * v.kv_heads + h) * 2 * D);
  if (!WIDE) {
    if (lane < LANES) b[part] = lo, b[LANES + part] = hi;
    return;
  }
  if (lane < LANES) joined[warp][0][part] = lo, joined[warp][1][part] = hi;
  __syncthreads();
  if (threadIdx.x < 2 * LANES) {
    const int side = threadIdx.x / LANES, at = threadIdx.x % LANES;
    uint4 x = joined[0][side][at];
#pragma unroll
    for (int w = 1; w < 8; w++) {
      const uint4 y = joined[w][side][at];
      x = side ? make_uint4(most2<T>(x.x, y.x), most2<T>(x.y, y.y), most2<T>(x.z, y.z), most2<T>(x.w, y.w))
               : make_uint4(least2<T>(x.x, y.x), least2<T>(x.y, y.y), least2<T>(x.z, y.z), least2<T>(x.w, y.w));
    }
    b[threadIdx.x] = x;
  }
  __syncthreads();
}

// The pages of first .. length - 1 of all sequences, counted 32 sequences at a
// time by one look at their lengths and spread over the CTAs in order, so the
// work is even whatever the lengths.  Memory bound: every key is read once, 2 /
// page_slots of that written.  By CTAs where those have at most two pages (times
// heads) each or pages are long (64 KiB of keys and more), else by warps: one
// page of 64 slots of each of 16 sequences 2.9 us, by warps 4.2; 508 pages 5.8
// and 8.0; 4 x 32,512 entries of 2 x 256 (at 40 to 100 %), 93 MB, in pages of 32
// slots 15.7 us by warps (6.0 TB/s), by CTAs 26.4; of 128 slots 19.0 and 17.6, of
// 512 42 and 15.8.  (4-byte loads: 24 us; 8 slots in flight and 4 CTAs an SM:
// 18.5.)
template <class T, int D>
__global__ void __launch_bounds__(256, 3) bounds_kernel(const BoundsArgs a) {
  __shared__ uint4 joined[8][2][D / 8];
  pdl_wait();
  pdl_launch_dependents();
  const PagedView& v = a.kv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t turn = blockIdx.x;                                          // this CTA's place in the order, from where the last ones ended
  for (uint32_t s0 = 0; s0 < v.sequences; s0 += 32) {
    // Lane s: sequence s0 + s's entries, first touched page and number of pages times heads.
    const uint32_t s = s0 + lane;
    uint32_t n = 0, page0 = 0;
    uint64_t count = 0;
    if (s < v.sequences) {
      n = held(v, s);
      if (v.lengths[s] > n) note(v, FZ_PAGED_BAD_LENGTH);
      const uint32_t first = a.first ? a.first[s] : 0u;
      if (first < n) {
        page0 = first / v.slots;
        count = (uint64_t)((n + v.page_slots - 1) / v.slots - page0) * v.kv_heads;
      }
    }
    uint64_t upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const uint64_t all = __shfl_sync(0xffffffffu, upto, 31);
    const bool wide = all <= 2 * gridDim.x || (uint64_t)v.page_slots * D >= kWide;
    const uint32_t step = wide ? gridDim.x : gridDim.x * 8;
    for (uint64_t at = wide ? turn : turn * 8 + warp; at < all; at += step) {
      const int of = __popc(__ballot_sync(0xffffffffu, upto <= at));    // the sequence that holds it
      const uint64_t in = at - (__shfl_sync(0xffffffffu, upto, of) - __shfl_sync(0xffffffffu, count, of));
      const uint32_t entries = __shfl_sync(0xffffffffu, n, of);
      const uint32_t logical = __shfl_sync(0xffffffffu, page0, of) + (uint32_t)(in / v.kv_heads), h = (uint32_t)(in % v.kv_heads);
      const uint32_t page = v.table[(size_t)(s0 + of) * v.table_stride + logical];
      const uint32_t slots = min(v.page_slots, entries - logical * v.page_slots);
      if (page >= v.pages) {
        if (lane == 0) note(v, FZ_PAGED_BAD_PAGE);
      } else if (wide) {
        page_bounds<T, D, true>(v, page, h, slots, joined);
      } else {
        page_bounds<T, D, false>(v, page, h, slots, joined);
      }
    }
    const uint32_t used = (uint32_t)((wide ? all : (all + 7) / 8) % gridDim.x);
    turn = turn >= used ? turn - used : turn + gridDim.x - used;
  }
}

template <template <class, int> class Of>
const void* pick(uint32_t type, uint32_t d) {
  if (type == FZ_KV_F16) return d == 64 ? Of<F16, 64>::fn() : d == 128 ? Of<F16, 128>::fn() : Of<F16, 256>::fn();
  return d == 64 ? Of<Bf16, 64>::fn() : d == 128 ? Of<Bf16, 128>::fn() : Of<Bf16, 256>::fn();
}
template <class T, int D>
struct AppendOf {
  static const void* fn() { return (const void*)append_kernel<T, D, 1>; }
};
template <class T, int D>
struct AppendManyOf {
  static const void* fn() { return (const void*)append_kernel<T, D, 4>; }
};
template <class T, int D>
struct BoundsOf {
  static const void* fn() { return (const void*)bounds_kernel<T, D>; }
};

}  // namespace
}  // namespace fz

extern "C" fz_status fz_paged_append(const fz_paged_kv* kv, const fz_paged_rows* rows, void* stream) {
  using namespace fz;
  AppendArgs a{};
  fz_status st = paged_view(kv, kNeedKeys, &a.kv);
  if (st) return st;
  if (!rows) return paged_refuse(FZ_ERR_ARGUMENT, "null rows");
  if (rows->rows == 0) return FZ_OK;
  if (!rows->k || !rows->v || !rows->index || (rows->heads && (!rows->q || !rows->q_out)))
    return paged_refuse(FZ_ERR_ARGUMENT, "null rows, index or q_out");
  if (rows->heads > (1u << 16)) return paged_refuse(FZ_ERR_ARGUMENT, "more than 65,536 query heads");
  if ((reinterpret_cast<uintptr_t>(rows->q) | reinterpret_cast<uintptr_t>(rows->k) | reinterpret_cast<uintptr_t>(rows->v) |
       reinterpret_cast<uintptr_t>(rows->q_out) | reinterpret_cast<uintptr_t>(rows->q_gain) |
       reinterpret_cast<uintptr_t>(rows->k_gain) | reinterpret_cast<uintptr_t>(rows->turns)) & 15u)
    return paged_refuse(FZ_ERR_ARGUMENT, "rows, gains or turns not 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(rows->sequence) | reinterpret_cast<uintptr_t>(rows->index) |
       reinterpret_cast<uintptr_t>(rows->position)) & 3u)
    return paged_refuse(FZ_ERR_ARGUMENT, "sequence, index or position not 4-byte aligned");
  if ((rows->q_stride | rows->k_stride | rows->v_stride | rows->q_out_stride) & 3u)
    return paged_refuse(FZ_ERR_ARGUMENT, "row strides must be multiples of 4 floats");
  const uint64_t kvw = (uint64_t)kv->kv_heads * kv->head_dim, qw = (uint64_t)rows->heads * kv->head_dim;
  if (rows->rows > 1 && (rows->k_stride < kvw || rows->v_stride < kvw || rows->q_stride < qw || rows->q_out_stride < qw))
    return paged_refuse(FZ_ERR_ARGUMENT, "a row stride shorter than its heads");
  if (!(rows->eps >= 0.0f) || std::isinf(rows->eps)) return paged_refuse(FZ_ERR_ARGUMENT, "eps must be finite and not negative");
  const void* p[] = {kv->keys, kv->values, kv->page_table, kv->lengths, kv->weights, kv->error, rows->q, rows->k, rows->v,
                     rows->q_out, rows->q_gain, rows->k_gain, rows->turns, rows->sequence, rows->index, rows->position};
  if ((st = paged_on_device(p, 16, "fz_paged_append"))) return st;
  a.r = *rows;
  // Steps of a row, 256 / head_dim heads a warp: one a warp while they do not
  // fill the GPU twice (32 warps an SM), else four.
  const uint32_t a_step = 256 / kv->head_dim, steps = (rows->heads + 2 * kv->kv_heads + a_step - 1) / a_step;
  const bool many = (uint64_t)rows->rows * steps > 2 * 148 * 32;
  uint32_t warps = many ? (steps + 3) / 4 : steps;
  const uint64_t blocks = ((uint64_t)rows->rows * warps + 3) / 4;
  if (blocks > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many rows");
  void* args[] = {&a, &warps};
  return paged_launch(many ? pick<AppendManyOf>(kv->type, kv->head_dim) : pick<AppendOf>(kv->type, kv->head_dim),
                      dim3((uint32_t)blocks), dim3(128), 0, 0, 1, args, stream);
}

extern "C" fz_status fz_paged_bounds(const fz_paged_kv* kv, const uint32_t* first, void* stream) {
  using namespace fz;
  BoundsArgs a{};
  fz_status st = paged_view(kv, kNeedKeys | kNeedBounds, &a.kv);
  if (st) return st;
  if (reinterpret_cast<uintptr_t>(first) & 3u) return paged_refuse(FZ_ERR_ARGUMENT, "first not 4-byte aligned");
  if (kv->sequences == 0) return FZ_OK;
  const void* p[] = {kv->keys, kv->page_table, kv->lengths, kv->bounds, kv->error, first};
  if ((st = paged_on_device(p, 6, "fz_paged_bounds"))) return st;
  a.first = first;
  const uint64_t items = (uint64_t)kv->table_stride * kv->kv_heads * kv->sequences;
  void* args[] = {&a};
  return paged_launch(pick<BoundsOf>(kv->type, kv->head_dim), dim3((uint32_t)std::min<uint64_t>(items, 3 * 148)), dim3(256), 0, 0,
                      1, args, stream);
}

// The paged cache's host checks, the append (QK-norm, rotation and store in
// one pass) and the pages' key bounds.
#include "paged.cuh"

#include <cmath>
#include <string>

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
    if (a.type == cudaMemoryTypeUnregistered || (a.type == cudaMemoryTypeDevice && a.device != device))
      return paged_refuse(FZ_ERR_ARGUMENT, (std::string(what) + ": a pointer that is not memory of the current device").c_str());
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
                   kv->head_stride, kv->sequences, kv->table_stride, kv->pages, kv->page_slots, kv->kv_heads};
  return FZ_OK;
}

fz_status paged_launch(const void* kernel, dim3 grid, dim3 block, size_t smem, uint32_t cluster, void** args,
                       void* stream) {
  cudaError_t e = cudaSuccess;
  if (smem > 16 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
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

// One warp a (row, head): D / 64 ... a lane holds D / 64 pairs (i, i + D / 2).
// The sum of squares and the norm in f32, the angle's turns in f64 (position
// x turns loses its fraction in f32 past a few thousand positions), its
// fraction's sine and cosine in f32.
template <class T, int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  constexpr int P = D / 64;                    // pairs a lane
  pdl_wait();
  const fz_paged_rows& r = a.r;
  const PagedView& v = a.kv;
  const int lane = threadIdx.x & 31;
  const uint32_t heads = r.heads + 2 * v.kv_heads;
  const uint64_t item = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint64_t row = item / heads;
  if (row >= r.rows) return;
  const uint32_t head = (uint32_t)(item % heads);
  const uint32_t seq = r.sequence ? r.sequence[row] : (uint32_t)row;
  if (seq == FZ_PAGED_NONE) return;
  const uint32_t index = r.index[row];
  const bool query = head < r.heads, value = head >= r.heads + v.kv_heads;
  const uint32_t h = query ? head : value ? head - r.heads - v.kv_heads : head - r.heads;
  const float* src = (query ? r.q + row * r.q_stride : value ? r.v + row * r.v_stride : r.k + row * r.k_stride) + (size_t)h * D;
  float x[P], y[P];
#pragma unroll
  for (int i = 0; i < P; i++) x[i] = src[lane * P + i], y[i] = src[D / 2 + lane * P + i];
  if (!value) {
    const float* gain = query ? r.q_gain : r.k_gain;
    if (gain) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < P; i++) s = fmaf(x[i], x[i], fmaf(y[i], y[i], s));
      s = warp_sum(s);
      const float inv = rsqrtf(fmaf(s, 1.0f / D, r.eps));
#pragma unroll
      for (int i = 0; i < P; i++) x[i] = x[i] * inv * gain[lane * P + i], y[i] = y[i] * inv * gain[D / 2 + lane * P + i];
    }
    if (r.turns) {
      const double pos = (double)(r.position ? r.position[row] : index);
#pragma unroll
      for (int i = 0; i < P; i++) {
        const double t = pos * r.turns[lane * P + i];
        float sn, cs;
        sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
        const float u = x[i], w = y[i];
        x[i] = u * cs - w * sn;
        y[i] = u * sn + w * cs;
      }
    }
  }
  if (query) {
    float* out = r.q_out + row * r.q_out_stride + (size_t)h * D;
#pragma unroll
    for (int i = 0; i < P; i++) out[lane * P + i] = x[i], out[D / 2 + lane * P + i] = y[i];
    return;
  }
  if (seq >= v.sequences || index >= v.table_stride * v.page_slots) {
    if (lane == 0) note(v, FZ_PAGED_BAD_ROW);
    return;
  }
  const uint32_t page = v.table[(size_t)seq * v.table_stride + index / v.page_slots], slot = index % v.page_slots;
  if (page >= v.pages) {
    if (lane == 0) note(v, FZ_PAGED_BAD_PAGE);
    return;
  }
  uint16_t* dst = (value ? v.values : v.keys) + element(v, page, slot, h);
#pragma unroll
  for (int i = 0; i < P; i++) {
    dst[lane * P + i] = (uint16_t)T::pack(x[i], 0.f);
    dst[D / 2 + lane * P + i] = (uint16_t)T::pack(y[i], 0.f);
  }
  if (lane == 0) {
    if (!value && v.weights) v.weights[((size_t)page * v.kv_heads + h) * v.page_slots + slot] = 0.f;
    if (!value && h == 0) atomicMax(v.lengths + seq, index + 1);
  }
}

// ------------------------------------------------------------ bounds

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

// One warp a (sequence, logical page, KV head), a lane D / 64 pairs of dimensions.
template <class T, int D>
__global__ void __launch_bounds__(256) bounds_kernel(const BoundsArgs a) {
  constexpr int P = D / 64;
  pdl_wait();
  const PagedView& v = a.kv;
  const int lane = threadIdx.x & 31;
  const uint64_t items = (uint64_t)v.table_stride * v.kv_heads;
  const uint64_t item = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= items) return;
  const uint32_t logical = (uint32_t)(item / v.kv_heads), h = (uint32_t)(item % v.kv_heads);
  for (uint32_t s = blockIdx.y; s < v.sequences; s += gridDim.y) {
    const uint32_t n = held(v, s), j0 = logical * v.page_slots;
    if (lane == 0 && item == 0 && v.lengths[s] > n) note(v, FZ_PAGED_BAD_LENGTH);
    if (j0 >= n || (a.first && a.first[s] >= n) || (a.first && a.first[s] >= j0 + v.page_slots)) continue;
    const uint32_t page = v.table[(size_t)s * v.table_stride + logical];
    if (page >= v.pages) {
      if (lane == 0) note(v, FZ_PAGED_BAD_PAGE);
      continue;
    }
    uint32_t lo[P], hi[P];
    const uint32_t slots = min(v.page_slots, n - j0);
    for (uint32_t i = 0; i < slots; i++) {
      const uint32_t* k = reinterpret_cast<const uint32_t*>(v.keys + element(v, page, i, h));
#pragma unroll
      for (int c = 0; c < P; c++) {
        const uint32_t w = k[lane + 32 * c];
        lo[c] = i ? least2<T>(lo[c], w) : w;
        hi[c] = i ? most2<T>(hi[c], w) : w;
      }
    }
    uint32_t* b = reinterpret_cast<uint32_t*>(v.bounds + ((size_t)page * v.kv_heads + h) * 2 * D);
#pragma unroll
    for (int c = 0; c < P; c++) b[lane + 32 * c] = lo[c], b[D / 2 + lane + 32 * c] = hi[c];
  }
}

template <template <class, int> class Of>
const void* pick(uint32_t type, uint32_t d) {
  if (type == FZ_KV_F16) return d == 64 ? Of<F16, 64>::fn() : d == 128 ? Of<F16, 128>::fn() : Of<F16, 256>::fn();
  return d == 64 ? Of<Bf16, 64>::fn() : d == 128 ? Of<Bf16, 128>::fn() : Of<Bf16, 256>::fn();
}
template <class T, int D>
struct AppendOf {
  static const void* fn() { return (const void*)append_kernel<T, D>; }
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
  const uint64_t blocks = ((uint64_t)rows->rows * (rows->heads + 2ull * kv->kv_heads) + 7) / 8;
  if (blocks > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many rows");
  void* args[] = {&a};
  return paged_launch(pick<AppendOf>(kv->type, kv->head_dim), dim3((uint32_t)blocks), dim3(256), 0, 1, args, stream);
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
  const uint64_t blocks = ((uint64_t)kv->table_stride * kv->kv_heads + 7) / 8;
  if (blocks > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many pages");
  void* args[] = {&a};
  return paged_launch(pick<BoundsOf>(kv->type, kv->head_dim), dim3((uint32_t)blocks, kv->sequences < 65535 ? kv->sequences : 65535),
                      dim3(256), 0, 1, args, stream);
}

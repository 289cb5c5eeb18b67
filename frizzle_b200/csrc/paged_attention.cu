// Attention of one new token a sequence over a paged cache (fz_paged_attention).
#include "paged.cuh"

#include <cmath>

namespace fz {
namespace {

constexpr int kWarps = 8;

struct AttendArgs {
  PagedView kv;
  const float* q;
  float* out;
  uint64_t q_stride, out_stride;
  const uint32_t* blocks;
  uint32_t group, top, window;
  float scale_log2e, decay;
};

// Entry `i` of an item's list: its logical index, or FZ_PAGED_NONE.  Without
// selected pages the list is the entries from `first` on.
FZ_DEV uint32_t listed(const AttendArgs& a, const uint32_t* blocks, uint32_t i, uint32_t first, uint32_t n, bool say) {
  const uint32_t slots = a.kv.page_slots;
  if (!blocks) return first + i < n ? first + i : FZ_PAGED_NONE;
  const uint32_t at = i / slots, b = __ldcg(blocks + at);
  if (b == FZ_PAGED_NONE) return FZ_PAGED_NONE;
  if (b >= (n + slots - 1) / slots || (at && __ldcg(blocks + at - 1) >= b)) {
    if (say) note(a.kv, FZ_PAGED_BAD_BLOCK);
    return FZ_PAGED_NONE;
  }
  const uint32_t j = b * slots + i % slots;
  return j < n && j >= first ? j : FZ_PAGED_NONE;
}

// One CTA a (sequence, KV head), a warp an entry at a time with its own
// running maximum and sum in log2 units, the warps joined at the end.
template <class T, int D>
__global__ void __launch_bounds__(32 * kWarps) attend_kernel(const AttendArgs a) {
  constexpr int P = D / 64;
  __shared__ float q[8 * D], o[8 * D], wm[kWarps][8], wl[kWarps][8];
  pdl_wait();
  const PagedView& v = a.kv;
  const int G = a.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t h = blockIdx.x % v.kv_heads, s = blockIdx.x / v.kv_heads;
  const uint32_t n = held(v, s);
  if (threadIdx.x == 0 && h == 0 && __ldcg(v.lengths + s) > n) note(v, FZ_PAGED_BAD_LENGTH);
  const uint32_t first = a.window && n > a.window ? n - a.window : 0;
  const uint32_t* blocks = a.blocks ? a.blocks + (size_t)blockIdx.x * a.top : nullptr;
  const uint32_t count = blocks ? min(a.top, (n + v.page_slots - 1) / v.page_slots) * v.page_slots : n - first;
  for (int i = threadIdx.x; i < G * D; i += 32 * kWarps) {
    q[i] = a.q[s * a.q_stride + (size_t)h * G * D + i] * a.scale_log2e;
    o[i] = 0.f;
  }
  __syncthreads();
  float m[8], l[8], acc[8][2 * P];
  for (int g = 0; g < 8; g++) {
    m[g] = -INFINITY, l[g] = 0.f;
    for (int c = 0; c < 2 * P; c++) acc[g][c] = 0.f;
  }
  auto score = [&](uint64_t at, int g) {
    const uint32_t* k = reinterpret_cast<const uint32_t*>(v.keys + at);
    float d = 0.f;
#pragma unroll
    for (int c = 0; c < P; c++) {
      const float2 x = T::unpack(k[lane + 32 * c]), y = reinterpret_cast<const float2*>(q + g * D)[lane + 32 * c];
      d = fmaf(x.x, y.x, fmaf(x.y, y.y, d));
    }
    return warp_sum(d);
  };
  auto place = [&](uint32_t i, uint32_t& page, uint32_t& slot) {
    const uint32_t j = listed(a, blocks, i, first, n, lane == 0);
    if (j == FZ_PAGED_NONE) return false;
    page = __ldcg(v.table + (size_t)s * v.table_stride + j / v.page_slots), slot = j % v.page_slots;
    if (page < v.pages) return true;
    if (lane == 0) note(v, FZ_PAGED_BAD_PAGE);
    return false;
  };
  for (uint32_t i = warp; i < count; i += kWarps) {
    uint32_t page, slot;
    if (!place(i, page, slot)) continue;
    const uint64_t at = element(v, page, slot, h);
    const uint32_t* val = reinterpret_cast<const uint32_t*>(v.values + at);
#pragma unroll
    for (int g = 0; g < 8; g++) {
      if (g >= G) break;
      const float d = score(at, g), mm = fmaxf(m[g], d), base = mm == -INFINITY ? 0.f : mm;
      const float f = exp2f(m[g] - base), p = exp2f(d - base);
      l[g] = fmaf(l[g], f, p);
#pragma unroll
      for (int c = 0; c < P; c++) {
        const float2 x = T::unpack(val[lane + 32 * c]);
        acc[g][2 * c] = fmaf(acc[g][2 * c], f, p * x.x);
        acc[g][2 * c + 1] = fmaf(acc[g][2 * c + 1], f, p * x.y);
      }
      m[g] = mm;
    }
  }
#pragma unroll
  for (int g = 0; g < 8; g++)
    if (lane == 0) wm[warp][g] = m[g], wl[warp][g] = l[g];
  __syncthreads();
  float top[8], sum[8];
#pragma unroll
  for (int g = 0; g < 8; g++) {
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, wm[w][g]);
    top[g] = mm == -INFINITY ? 0.f : mm;
    for (int w = 0; w < kWarps; w++) ll = fmaf(wl[w][g], exp2f(wm[w][g] - top[g]), ll);
    sum[g] = ll;
  }
  for (int w = 0; w < kWarps; w++) {
    if (w == warp) {
#pragma unroll
      for (int g = 0; g < 8; g++) {
        if (g >= G) break;
        const float f = exp2f(m[g] - top[g]);
#pragma unroll
        for (int c = 0; c < P; c++) {
          o[g * D + 2 * (lane + 32 * c)] += acc[g][2 * c] * f;
          o[g * D + 2 * (lane + 32 * c) + 1] += acc[g][2 * c + 1] * f;
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < G * D; i += 32 * kWarps) {
    float l1 = 0.f;
#pragma unroll
    for (int g = 0; g < 8; g++) l1 = i / D == g ? sum[g] : l1;
    a.out[s * a.out_stride + (size_t)h * G * D + i] = l1 == 0.f ? 0.f : o[i] / l1;
  }
  if (!v.weights) return;
  for (uint32_t i = warp; i < count; i += kWarps) {
    uint32_t page, slot;
    if (!place(i, page, slot)) continue;
    const uint64_t at = element(v, page, slot, h);
    float w = 0.f;
#pragma unroll
    for (int g = 0; g < 8; g++) {
      if (g >= G) break;
      const float p = exp2f(score(at, g) - top[g]);
      w += sum[g] == 0.f ? 0.f : p / sum[g];
    }
    float* to = v.weights + ((size_t)page * v.kv_heads + h) * v.page_slots + slot;
    if (lane == 0) *to = a.decay == 0.f ? w : fmaf(a.decay, *to, w);
  }
}

}  // namespace
}  // namespace fz

extern "C" size_t fz_paged_attention_workspace(const fz_paged_kv* kv, uint32_t heads) {
  (void)kv;
  (void)heads;
  return 256;
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
  if (!query->workspace || (reinterpret_cast<uintptr_t>(query->workspace) & 255u) || query->workspace_bytes < need)
    return paged_refuse(FZ_ERR_ARGUMENT, "workspace null, not 256-byte aligned, or shorter than fz_paged_attention_workspace");
  const uint64_t items = (uint64_t)kv->sequences * kv->kv_heads;
  if (items > 0x7FFFFFFFull) return paged_refuse(FZ_ERR_ARGUMENT, "too many sequences");
  if (items == 0) return FZ_OK;
  const void* p[] = {kv->keys, kv->values, kv->page_table, kv->lengths, kv->weights, kv->error,
                     query->q, query->out, query->blocks,  query->workspace};
  if ((st = paged_on_device(p, 10, "fz_paged_attention"))) return st;
  a.q = query->q, a.out = query->out, a.q_stride = query->q_stride, a.out_stride = query->out_stride;
  a.blocks = query->blocks, a.group = heads / kv->kv_heads, a.top = query->top, a.window = query->window;
  a.scale_log2e = (float)((double)query->scale * 1.4426950408889634);
  a.decay = query->decay;
  void* args[] = {&a};
  const bool f16 = kv->type == FZ_KV_F16;
  const uint32_t d = kv->head_dim;
  const void* fn = f16 ? (d == 64    ? (const void*)attend_kernel<F16, 64>
                          : d == 128 ? (const void*)attend_kernel<F16, 128>
                                     : (const void*)attend_kernel<F16, 256>)
                       : (d == 64    ? (const void*)attend_kernel<Bf16, 64>
                          : d == 128 ? (const void*)attend_kernel<Bf16, 128>
                                     : (const void*)attend_kernel<Bf16, 256>);
  return paged_launch(fn, dim3((uint32_t)items), dim3(32 * kWarps), 0, 1, args, stream);
}

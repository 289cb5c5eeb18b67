// The paged key/value cache as its kernels see it (fz_paged_* of
// frizzle_b200.h), and what their host entry points share.
#pragma once

#include <cuda_bf16.h>

#include "fz_common.cuh"
#include "frizzle_b200.h"

namespace fz {

struct PagedView {
  uint16_t* keys;
  uint16_t* values;
  const uint32_t* table;
  uint32_t* lengths;
  float* weights;
  uint16_t* bounds;
  uint32_t* error;
  uint64_t page_stride, slot_stride, head_stride;
  uint32_t sequences, table_stride, pages, page_slots, kv_heads;
};

// A cache element's type: f16 or bf16, its conversions to and from f32.
struct F16 {
  static constexpr uint32_t kType = FZ_KV_F16;
  FZ_DEV static float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  // Saturating at +-65,504, NaN kept (f16_pack keeps a NaN's sign only).
  FZ_DEV static uint32_t pack(float a, float b) {
    a = fabsf(a) > 65504.0f ? copysignf(65504.0f, a) : a;
    b = fabsf(b) > 65504.0f ? copysignf(65504.0f, b) : b;
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
struct Bf16 {
  static constexpr uint32_t kType = FZ_KV_BF16;
  FZ_DEV static float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  FZ_DEV static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

FZ_DEV void note(const PagedView& v, uint32_t bit) {
  if (v.error) atomicOr(v.error, bit);
}

// Entries sequence s holds, cut to its table.
FZ_DEV uint32_t held(const PagedView& v, uint32_t s) {
  const uint32_t n = v.lengths[s];
  return min(n, v.table_stride * v.page_slots);
}

// Where slot i of page p holds KV head h, in elements.
FZ_DEV uint64_t element(const PagedView& v, uint32_t page, uint32_t slot, uint32_t head) {
  return page * v.page_stride + slot * v.slot_stride + head * v.head_stride;
}

// ------------------------------------------------------------ host side

// FZ_OK, or the refusal (its message set) of a cache description; `need` are
// the parts the caller reads or writes.
enum : uint32_t { kNeedKeys = 1, kNeedBounds = 2, kNeedWeights = 4 };
fz_status paged_view(const fz_paged_kv* kv, uint32_t need, PagedView* out);
fz_status paged_refuse(fz_status s, const char* why);
// FZ_OK when every pointer (NULL ones left out) is memory the current device
// reaches as its own; a refusal naming `what` otherwise.
fz_status paged_on_device(const void* const* pointers, int count, const char* what);
fz_status paged_launch(const void* kernel, dim3 grid, dim3 block, size_t smem, uint32_t cluster, void** args,
                       void* stream);

}  // namespace fz

// The paged key/value cache as its kernels see it (fz_paged_* of
// frizzle_b200.h), and what their host entry points share.
#pragma once

#include <cuda_bf16.h>

#include "fz_common.cuh"
#include "frizzle_b200.h"

namespace fz {

// Division of numbers below 2^31 by a divisor known beforehand (Granlund and
// Montgomery 1994, theorem 4.2: multiplier floor(2^(31 + l) / d) + 1 with 2^l the
// least power of two not below d): a product and a shift where a division by a
// variable is some twenty instructions, at every look at a page table.
struct Divisor {
  uint32_t d, multiplier, shift;
};
inline Divisor divisor(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) l++;
  return Divisor{d, (uint32_t)((1ull << (31 + l)) / d + 1), 31 + l};
}
FZ_DEV uint32_t operator/(uint32_t n, const Divisor& d) { return (uint32_t)(((uint64_t)n * d.multiplier) >> d.shift); }
FZ_DEV uint32_t operator%(uint32_t n, const Divisor& d) { return n - n / d * d.d; }

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
  Divisor slots;                       // page_slots
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

// Into L2, before it is asked for (what it reads may still be written).
FZ_DEV void hint(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// 16-byte copies into shared memory (zeros where not valid), by groups.
FZ_DEV uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
FZ_DEV void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
FZ_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
FZ_DEV void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <class T>
FZ_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (T::kType == FZ_KV_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A pair of f32 as pairs of the cache's type that sum to it: f16 part and
// remainder (22 bits), the remainder times `lift`; bf16 three parts (24 bits).
template <class T>
struct Parts {
  static constexpr int N = T::kType == FZ_KV_F16 ? 2 : 3;
  uint32_t w[4];
};
template <class T>
FZ_DEV Parts<T> parts(float x, float y, float lift = 1.f) {
  Parts<T> p;
#pragma unroll
  for (int i = 0; i < Parts<T>::N; i++) {
    p.w[i] = T::pack(x, y);
    const float2 u = T::unpack(p.w[i]);
    x = (x - u.x) * lift, y = (y - u.y) * lift;
  }
#pragma unroll
  for (int i = Parts<T>::N; i < 4; i++) p.w[i] = 0;
  return p;
}
// A query is divided by 2^(e - 127), of its largest value `top`: to [1, 2) for
// f16 keys (2^14 times that in attend_kernel), to 2^-10 of that for bf16 ones,
// which may be as large as an f32, so that no sum of up to 256 products overflows
// by the way (2^8 x 2^-9 x the largest key).  2^(e - 127) and its reciprocal are
// normal.
template <class T>
FZ_DEV uint32_t query_exponent(float top) {
  return min(max(__float_as_uint(top) >> 23, 1u) + (T::kType == FZ_KV_F16 ? 0u : 10u), 253u);
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
// `most`: the most dynamic shared memory that any call gives this kernel.
fz_status paged_launch(const void* kernel, dim3 grid, dim3 block, size_t smem, size_t most, uint32_t cluster, void** args,
                       void* stream);

}  // namespace fz

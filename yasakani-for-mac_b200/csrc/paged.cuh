// Shared pieces of the batch operators over a paged 16-bit K/V cache (batchplan.cu,
// pagedprep.cu, prefixattn.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace yskn {

// Element (block b, place t, KV head h, channel d) of a cache at
// b * block_stride + t * token_stride + h * head_stride + d (in elements).
struct CacheStrides {
  int64_t block, token, head;
};

template <int DT>
struct Elem;
template <>
struct Elem<YSKN_DT_BF16> {
  __device__ static __forceinline__ float to_float(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
  __device__ static __forceinline__ uint16_t from_float(float x) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  }
  // Two values rounded to nearest, lo in the low half.
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
template <>
struct Elem<YSKN_DT_F16> {
  __device__ static __forceinline__ float to_float(uint16_t b) { return __half2float(__ushort_as_half(b)); }
  __device__ static __forceinline__ uint16_t from_float(float x) { return __half_as_ushort(__float2half_rn(x)); }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool is_16bit(int dt) { return dt == YSKN_DT_F16 || dt == YSKN_DT_BF16; }

}  // namespace yskn

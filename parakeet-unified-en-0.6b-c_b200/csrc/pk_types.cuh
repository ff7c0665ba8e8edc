// pk_types.cuh -- the element types of the 8-bit operators (PKCU_DTYPE_*):
// sizes and alignment for the argument checks, conversions for the kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "pkcuda_internal.h"

namespace pk {

// Bytes of a floating row type, 0 for any other type.
inline int dtype_size(int dtype) {
  return dtype == PKCU_DTYPE_F32 ? 4 : (dtype == PKCU_DTYPE_BF16 || dtype == PKCU_DTYPE_F16 ? 2 : 0);
}
inline bool misaligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) != 0; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);   // rounded to nearest even
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// max and min that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace pk

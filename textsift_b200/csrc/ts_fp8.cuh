// ts_fp8.cuh — device helpers of the 8-bit floating point operators.
#pragma once

#include "textsift_cuda.h"
#include "ts_common.cuh"
#include "ts_fp8.h"

#include <cuda_bf16.h>

namespace ts {

constexpr float kFp8SmallestScale = 7.888609052210118e-31f;  // 2^-100: the scale of a block of zeros

template <int DT>
struct Fp8Type;
template <>
struct Fp8Type<TS_DTYPE_F16> {
  using T = __half;
  static __device__ __forceinline__ float up(T v) { return __half2float(v); }
  static __device__ __forceinline__ T down(float v) { return __float2half_rn(v); }
};
template <>
struct Fp8Type<TS_DTYPE_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float up(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T down(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Fp8Type<TS_DTYPE_F32> {
  using T = float;
  static __device__ __forceinline__ float up(T v) { return v; }
  static __device__ __forceinline__ T down(float v) { return v; }
};

// |x| where x is finite, 0 where it is not: a block's scale comes from its
// finite values alone.
__device__ __forceinline__ float fp8_mag(float x) {
  const float a = fabsf(x);
  return a < __int_as_float(0x7f800000) ? a : 0.0f;
}
// The format's scale of a block whose largest finite magnitude is a, and its
// reciprocal r: both roundings to f32 are part of the format.
__device__ __forceinline__ float fp8_scale(float a) {
  return fmaxf(__fmul_rn(a, 1.0f / 448.0f), kFp8SmallestScale);
}
__device__ __forceinline__ float fp8_inverse(float s) { return __frcp_rn(s); }

// Codes of x0 r (low byte) and x1 r: nearest even, beyond +-448 clamped, NaN 0x7F.
__device__ __forceinline__ uint32_t fp8_codes2(float x0, float x1, float r) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(__fmul_rn(x1, r)), "f"(__fmul_rn(x0, r)));
  return c;
}
// The two values of a pair of codes, exact in fp16.
__device__ __forceinline__ __half2 fp8_pair(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return *reinterpret_cast<__half2*>(&h);
}
__device__ __forceinline__ float fp8_value(uint8_t c) { return __low2float(fp8_pair(c)); }

}  // namespace ts

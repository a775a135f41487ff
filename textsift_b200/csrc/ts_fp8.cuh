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
// The larger magnitude of each half of a pair of 16-bit values (a NaN gives
// way), and the halves as f32.
template <int DT>
__device__ __forceinline__ uint32_t fp8_mag_max2(uint32_t a, uint32_t b) {
  if constexpr (DT == TS_DTYPE_F16) {
    const __half2 m = __hmax2(__habs2(*reinterpret_cast<__half2*>(&a)), __habs2(*reinterpret_cast<__half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m =
        __hmax2(__habs2(*reinterpret_cast<__nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<__nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}

// 16 values of a row (or column) of type DT: eight lanes hold one block of 128.
template <int DT>
struct Fp8Piece {
  float v[16];

  // Largest magnitude over the block's eight lanes.  fmaxf passes over a NaN;
  // only an infinity needs the second look that leaves it out.
  __device__ __forceinline__ float block_max() const {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++) m = fmaxf(m, fabsf(v[j]));
    m = lanes_max(m);
    if (!(m < __int_as_float(0x7f800000))) {  // the same for all eight lanes
      m = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j++) m = fmaxf(m, fp8_mag(v[j]));
      m = lanes_max(m);
    }
    return m;
  }
  static __device__ __forceinline__ float lanes_max(float m) {
    const uint32_t mask = 0xffu << (threadIdx.x & 24u);
#pragma unroll
    for (int d = 4; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, d));
    return m;
  }
  __device__ __forceinline__ uint4 codes(float r) const {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      w[j] = fp8_codes2(v[4 * j], v[4 * j + 1], r) | fp8_codes2(v[4 * j + 2], v[4 * j + 3], r) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // values i .. i + 15 of a row of n, zeros past its end
  __device__ __forceinline__ void load(const typename Fp8Type<DT>::T* x, uint32_t i, uint32_t n, bool vec) {
    using T = typename Fp8Type<DT>::T;
    if (vec && fp8_whole(i, n)) {
      constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
      for (int j = 0; j < 16 / PER; j++) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + i) + j);
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int l = 0; l < PER; l++) v[j * PER + l] = Fp8Type<DT>::up(t[l]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++) v[j] = i + j < n ? Fp8Type<DT>::up(x[i + j]) : 0.0f;
    }
  }
};

}  // namespace ts

// k_fp8_gemm.cu — products of 8-bit operands with a scale for each block of
// 128: out[m, n] = sum_b as[b, m] ws[., b] (sum_{k in b} a[m, k] w[n, k]).
#include "ts_fp8.cuh"

#include <algorithm>

namespace ts {

static __device__ int g_fp8_err;

int* fp8_err_flag() {
  void* p = nullptr;
  return cudaGetSymbolAddress(&p, g_fp8_err) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

template <int DT>
__device__ __forceinline__ void fp8_store(const Fp8MmArgs& a, uint32_t m, uint32_t n, float v) {
  using D = Fp8Type<DT>;
  auto* o = reinterpret_cast<typename D::T*>(a.out) + m * a.ldo + n;
  if (DT == TS_DTYPE_F32 && a.accumulate) v += D::up(*o);
  *o = D::down(v);
}

// 64 x 64 outputs of rows [row0, row_end) by one weight; 16 x 16 threads with
// 4 x 4 outputs each, one block of 128 k at a time through shared memory.
template <int DT>
__global__ void __launch_bounds__(256) fp8_matmul_simt_kernel(const Fp8MmArgs a) {
  __shared__ float sa[64][33], sw[64][33];
  const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n0 = blockIdx.x * 64, e = blockIdx.z;
  const uint32_t nb = fp8_blocks(a.N), kb = fp8_blocks(a.K);
  uint32_t lo = 0, hi = a.M;
  if (a.seg) {
    lo = (uint32_t)min(max(a.seg[e], 0), (int)a.M);
    hi = max(lo, (uint32_t)min(max(a.seg[e + 1], 0), (int)a.M));
  }
  const uint8_t* w = a.w + (uint64_t)e * a.N * a.ldw;
  for (uint32_t m0 = lo + blockIdx.y * 64; m0 < hi; m0 += gridDim.y * 64) {
    float acc[4][4] = {};
    for (uint32_t b = 0; b < kb; b++) {
      float part[4][4] = {};
      for (uint32_t k0 = b * kFp8Block; k0 < min(a.K, (b + 1) * kFp8Block); k0 += 32) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 64 * 32; i += 256) {
          const uint32_t r = i / 32, k = k0 + i % 32;
          sa[r][i % 32] = m0 + r < hi && k < a.K ? fp8_value(a.a[(m0 + r) * a.lda + k]) : 0.0f;
          sw[r][i % 32] = n0 + r < a.N && k < a.K ? fp8_value(w[(n0 + r) * a.ldw + k]) : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 32; k++)
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) part[i][j] = fmaf(sa[ty * 4 + i][k], sw[tx * 4 + j][k], part[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t m = m0 + ty * 4 + i;
        const float s = m < hi ? a.as[b * a.ldas + m] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t n = n0 + tx * 4 + j;
          const float t = n >= a.N ? 0.0f
                          : a.w_block == 1 ? a.ws[b * a.ldws + n]
                                           : a.ws[((uint64_t)e * nb + n / kFp8Block) * kb + b];
          acc[i][j] = fmaf(part[i][j], s * t, acc[i][j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
        if (m >= hi || n >= a.N) continue;
        const float bias =
            a.bias ? __half2float(reinterpret_cast<const __half*>(a.bias)[(uint64_t)e * a.N + n]) : 0.0f;
        fp8_store<DT>(a, m, n, acc[i][j] + bias);
      }
  }
}

cudaError_t launch_fp8_matmul(const Fp8MmArgs& a, cudaStream_t st) {
  const dim3 grid((a.N + 63) / 64, std::min((a.M + 63) / 64, 65535u), a.E);
  if (a.out_dtype == TS_DTYPE_F16) fp8_matmul_simt_kernel<TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  else if (a.out_dtype == TS_DTYPE_BF16) fp8_matmul_simt_kernel<TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else fp8_matmul_simt_kernel<TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

// One warp for each output row n of the weight and row m of x: lane l takes
// the values l, l + 32, ... of a block, quantises them and multiplies.
template <int XT, int OT>
__global__ void __launch_bounds__(256) fp8_matvec_simt_kernel(const Fp8MvArgs a) {
  using X = Fp8Type<XT>;
  using O = Fp8Type<OT>;
  const uint32_t n = blockIdx.x * 8 + (threadIdx.x >> 5), m = blockIdx.y, lane = threadIdx.x & 31;
  if (n >= a.N) return;
  const uint32_t kb = fp8_blocks(a.K);
  const auto* x = reinterpret_cast<const typename X::T*>(a.x) + m * a.ldx;
  float acc = 0.0f;
  for (uint32_t b = 0; b < kb; b++) {
    float v[4], mx = 0.0f, part = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t k = b * kFp8Block + j * 32 + lane;
      v[j] = k < a.K ? X::up(x[k]) : 0.0f;
      mx = fmaxf(mx, fp8_mag(v[j]));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float s = fp8_scale(mx), r = fp8_inverse(s);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t k = b * kFp8Block + j * 32 + lane;
      if (k < a.K) part = fmaf(fp8_value((uint8_t)fp8_codes2(v[j], 0.0f, r)), fp8_value(a.w[n * a.ldw + k]), part);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
    acc = fmaf(part, s * a.ws[(uint64_t)(n / kFp8Block) * kb + b], acc);
  }
  if (lane == 0) {
    if (a.bias) acc += __half2float(reinterpret_cast<const __half*>(a.bias)[n]);
    (reinterpret_cast<typename O::T*>(a.out) + m * a.ldo)[n] = O::down(acc);
  }
}

template <int XT>
static void launch_mv(const Fp8MvArgs& a, cudaStream_t st) {
  const dim3 grid((a.N + 7) / 8, a.M);
  if (a.out_dtype == TS_DTYPE_F16) fp8_matvec_simt_kernel<XT, TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  else if (a.out_dtype == TS_DTYPE_BF16) fp8_matvec_simt_kernel<XT, TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else fp8_matvec_simt_kernel<XT, TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
}

cudaError_t launch_fp8_matvec(const Fp8MvArgs& a, cudaStream_t st) {
  if (a.x_dtype == TS_DTYPE_F16) launch_mv<TS_DTYPE_F16>(a, st);
  else if (a.x_dtype == TS_DTYPE_BF16) launch_mv<TS_DTYPE_BF16>(a, st);
  else launch_mv<TS_DTYPE_F32>(a, st);
  return cudaGetLastError();
}

}  // namespace ts

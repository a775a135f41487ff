// k_fp8_quant.cu — quantising to e4m3 with a scale for each block of 128, by
// rows or by columns, and the relayout of a quantised weight by its columns.
//
// With a = max |x| over the finite values of a block: s = max(a * (1/448),
// 2^-100), r = 1/s, code = e4m3(x * r), every f32 step rounded to nearest.
#include "ts_fp8.cuh"

#include <algorithm>

namespace ts {

// One warp for each (row, block of 128 columns).
template <int DT>
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const Fp8QuantArgs a) {
  using D = Fp8Type<DT>;
  const uint32_t nb = fp8_blocks(a.cols), lane = threadIdx.x & 31;
  const uint64_t total = (uint64_t)a.rows * nb;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += (uint64_t)gridDim.x * 8) {
    const uint32_t row = (uint32_t)(i / nb), b = (uint32_t)(i % nb);
    const auto* x = reinterpret_cast<const typename D::T*>(a.x) + row * a.ldx;
    float v[4], m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t c = b * kFp8Block + lane * 4 + j;
      v[j] = c < a.cols ? D::up(x[c]) : 0.0f;
      m = fmaxf(m, fp8_mag(v[j]));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float s = fp8_scale(m), r = fp8_inverse(s);
    if (lane == 0) a.scales[b * a.lds + row] = s;
    const uint32_t c4 = fp8_codes2(v[0], v[1], r) | fp8_codes2(v[2], v[3], r) << 16;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t c = b * kFp8Block + lane * 4 + j;
      if (c < a.cols) a.codes[row * a.ldc + c] = (uint8_t)(c4 >> 8 * j);
    }
  }
}

// One block for 128 rows x 32 columns: thread (column, part) takes 16 rows.
template <int DT>
__global__ void __launch_bounds__(256) fp8_quant_cols_kernel(const Fp8QuantArgs a) {
  using D = Fp8Type<DT>;
  __shared__ float part[8][32];
  const uint32_t tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const uint32_t col = blockIdx.x * 32 + tx;
  for (uint32_t b = blockIdx.y; b < fp8_blocks(a.rows); b += gridDim.y) {
    const auto* x = reinterpret_cast<const typename D::T*>(a.x);
    float v[16], m = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const uint32_t row = b * kFp8Block + ty * 16 + j;
      v[j] = row < a.rows && col < a.cols ? D::up(x[row * a.ldx + col]) : 0.0f;
      m = fmaxf(m, fp8_mag(v[j]));
    }
    __syncthreads();
    part[ty][tx] = m;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) m = fmaxf(m, part[j][tx]);
    const float s = fp8_scale(m), r = fp8_inverse(s);
    if (col < a.cols) {
      if (ty == 0) a.scales[b * a.lds + col] = s;
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const uint32_t row = b * kFp8Block + ty * 16 + j, c2 = fp8_codes2(v[j], v[j + 1], r);
        if (row < a.rows) a.codes[col * a.ldc + row] = (uint8_t)c2;
        if (row + 1 < a.rows) a.codes[col * a.ldc + row + 1] = (uint8_t)(c2 >> 8);
      }
    }
  }
}

// 64 x 64 codes of one expert through shared memory; the first thread of a
// block that starts a 128 x 128 block moves its scale.
__global__ void __launch_bounds__(256)
    fp8_transpose_kernel(const uint8_t* __restrict__ codes, uint64_t ldw, const float* __restrict__ scales, uint32_t N,
                         uint32_t K, uint8_t* __restrict__ codes_t, uint64_t ldt, float* __restrict__ scales_t,
                         uint32_t k_tiles) {
  __shared__ uint8_t tile[64][65];
  const uint32_t e = blockIdx.y, n0 = blockIdx.x / k_tiles * 64, k0 = blockIdx.x % k_tiles * 64;
  const uint8_t* src = codes + (uint64_t)e * N * ldw;
  uint8_t* dst = codes_t + (uint64_t)e * K * ldt;
  for (uint32_t i = threadIdx.x; i < 64 * 64; i += 256) {
    const uint32_t n = n0 + i / 64, k = k0 + i % 64;
    if (n < N && k < K) tile[i / 64][i % 64] = src[n * ldw + k];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 64 * 64; i += 256) {
    const uint32_t k = k0 + i / 64, n = n0 + i % 64;
    if (n < N && k < K) dst[k * ldt + n] = tile[i % 64][i / 64];
  }
  if (threadIdx.x == 0 && n0 % kFp8Block == 0 && k0 % kFp8Block == 0) {
    const uint32_t nb = fp8_blocks(N), kb = fp8_blocks(K), n = n0 / kFp8Block, k = k0 / kFp8Block;
    scales_t[((uint64_t)e * kb + k) * nb + n] = scales[((uint64_t)e * nb + n) * kb + k];
  }
}

cudaError_t launch_fp8_quant_rows(const Fp8QuantArgs& a, cudaStream_t st) {
  const uint64_t warps = (uint64_t)a.rows * fp8_blocks(a.cols);
  const uint32_t grid = (uint32_t)std::min<uint64_t>((warps + 7) / 8, 1u << 20);
  if (a.dtype == TS_DTYPE_F16) fp8_quant_rows_kernel<TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  else if (a.dtype == TS_DTYPE_BF16) fp8_quant_rows_kernel<TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else fp8_quant_rows_kernel<TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_fp8_quant_cols(const Fp8QuantArgs& a, cudaStream_t st) {
  const dim3 grid((a.cols + 31) / 32, std::min(fp8_blocks(a.rows), 65535u));
  if (a.dtype == TS_DTYPE_F16) fp8_quant_cols_kernel<TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  else if (a.dtype == TS_DTYPE_BF16) fp8_quant_cols_kernel<TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else fp8_quant_cols_kernel<TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_fp8_transpose(const uint8_t* codes, uint64_t ldw, const float* scales, uint32_t E, uint32_t N,
                                 uint32_t K, uint8_t* codes_t, uint64_t ldt, float* scales_t, cudaStream_t st) {
  const uint32_t k_tiles = (K + 63) / 64;
  const dim3 grid((N + 63) / 64 * k_tiles, E);
  fp8_transpose_kernel<<<grid, 256, 0, st>>>(codes, ldw, scales, N, K, codes_t, ldt, scales_t, k_tiles);
  return cudaGetLastError();
}

}  // namespace ts

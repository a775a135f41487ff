// k_fp8_quant.cu — quantising to e4m3 with a scale for each block of 128, by
// rows or by columns, and the relayout of a quantised weight by its columns.
//
// With a = max |x| over the finite values of a block: s = max(a * (1/448),
// 2^-100), r = 1/s, code = e4m3(x * r), every f32 step rounded to nearest.
#include "ts_fp8.cuh"

namespace ts {

// Eight lanes for each (row, block of 128 columns), 16 values a lane: the row
// is read and its codes are written in 16-byte pieces.  A warp takes the same
// block of four rows, so the scales it writes lie together; consecutive warps
// take the row's next blocks.
template <int DT>
__global__ void __launch_bounds__(256, 8) fp8_quant_rows_kernel(const Fp8QuantArgs a, uint32_t vec) {
  pdl_trigger();
  pdl_wait();
  const uint32_t nb = fp8_blocks(a.cols), lane = threadIdx.x & 31;
  const uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint64_t row = i / nb * 4 + (lane >> 3);
  const uint32_t b = (uint32_t)(i % nb), c = b * kFp8Block + (lane & 7) * 16;
  if (row >= a.rows) return;
  Fp8Piece<DT> p;
  p.load(reinterpret_cast<const typename Fp8Type<DT>::T*>(a.x) + row * a.ldx, c, a.cols, vec);
  const float s = fp8_scale(p.block_max());
  if ((lane & 7) == 0) a.scales[b * a.lds + row] = s;
  if (c < a.cols) *reinterpret_cast<uint4*>(a.codes + row * a.ldc + c) = p.codes(fp8_inverse(s));
}

// A tile of 128 rows x 128 bytes (64 or 32 columns) through shared memory:
// rows come in as they lie, and eight lanes then take one column (or, of
// 16-bit types, two neighbours), 16 rows a lane, so that a column's 128 codes
// leave as one line.  Four words after every 16 rows put the eight lanes'
// rows into different banks.
template <int DT>
__global__ void __launch_bounds__(256, 6) fp8_quant_cols_kernel(const Fp8QuantArgs a, uint32_t vec, uint32_t col_tiles) {
  using D = Fp8Type<DT>;
  using T = typename D::T;
  constexpr uint32_t COLS = 128 / sizeof(T), W = sizeof(T) == 2 ? 2 : 1;  // columns a lane takes
  constexpr uint32_t GROUP = 16 * 128 + 16;                               // bytes of 16 rows
  __shared__ __align__(16) uint8_t tile[8 * GROUP];
  pdl_trigger();
  pdl_wait();
  const uint32_t b = blockIdx.x / col_tiles, c0 = blockIdx.x % col_tiles * COLS;
  const T* x = reinterpret_cast<const T*>(a.x);
#pragma unroll
  for (uint32_t j = 0; j < 4; j++) {
    const uint32_t r = j * 32 + (threadIdx.x >> 3), o = (threadIdx.x & 7) * 16;
    const uint32_t c = c0 + o / sizeof(T);
    const uint64_t row = (uint64_t)b * kFp8Block + r;
    uint8_t* dst = tile + (r >> 4) * GROUP + (r & 15) * 128 + o;
    constexpr uint32_t PER = 16 / sizeof(T);
    if (vec && row < a.rows && c + PER <= a.cols) {
      *reinterpret_cast<uint4*>(dst) = __ldg(reinterpret_cast<const uint4*>(x + row * a.ldx + c));
    } else {
#pragma unroll
      for (uint32_t l = 0; l < PER; l++)
        reinterpret_cast<T*>(dst)[l] = row < a.rows && c + l < a.cols ? x[row * a.ldx + c + l] : D::down(0.0f);
    }
  }
  __syncthreads();
  const uint32_t col = threadIdx.x / 8 * W, g = threadIdx.x & 7;
  const uint8_t* src = tile + g * GROUP + col * sizeof(T);
  uint32_t raw[16];  // of both columns
#pragma unroll
  for (uint32_t j = 0; j < 16; j++) raw[j] = *reinterpret_cast<const uint32_t*>(src + j * 128);
  const uint32_t row0 = b * kFp8Block + g * 16;
#pragma unroll
  for (uint32_t w = 0; w < W; w++) {
    Fp8Piece<DT> p;
#pragma unroll
    for (uint32_t j = 0; j < 16; j++) p.v[j] = D::up(reinterpret_cast<const T*>(&raw[j])[w]);
    const float s = fp8_scale(p.block_max());
    const uint64_t c = c0 + col + w;
    if (c >= a.cols) continue;
    if (g == 0) a.scales[b * a.lds + c] = s;
    if (row0 < a.rows) *reinterpret_cast<uint4*>(a.codes + c * a.ldc + row0) = p.codes(fp8_inverse(s));
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

// Rows of x can be read in 16-byte pieces.
static uint32_t fp8_vec(const Fp8QuantArgs& a) {
  const uint64_t bytes = a.dtype == TS_DTYPE_F32 ? 4 : 2;
  return !(reinterpret_cast<uintptr_t>(a.x) & 15u) && a.ldx * bytes % 16 == 0;
}

cudaError_t launch_fp8_quant_rows(const Fp8QuantArgs& a, cudaStream_t st) {
  const uint64_t warps = ((uint64_t)a.rows + 3) / 4 * fp8_blocks(a.cols), grid = (warps + 7) / 8;
  if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
  const dim3 g((uint32_t)grid), t(256);
  if (a.dtype == TS_DTYPE_F16) return launch_pdl(fp8_quant_rows_kernel<TS_DTYPE_F16>, g, t, 0, st, a, fp8_vec(a));
  if (a.dtype == TS_DTYPE_BF16) return launch_pdl(fp8_quant_rows_kernel<TS_DTYPE_BF16>, g, t, 0, st, a, fp8_vec(a));
  return launch_pdl(fp8_quant_rows_kernel<TS_DTYPE_F32>, g, t, 0, st, a, fp8_vec(a));
}

cudaError_t launch_fp8_quant_cols(const Fp8QuantArgs& a, cudaStream_t st) {
  const uint32_t cols = a.dtype == TS_DTYPE_F32 ? 32 : 64, col_tiles = a.cols / cols + (a.cols % cols != 0);
  const uint64_t grid = (uint64_t)col_tiles * fp8_blocks(a.rows);
  if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
  const dim3 g((uint32_t)grid), t(256);
  if (a.dtype == TS_DTYPE_F16)
    return launch_pdl(fp8_quant_cols_kernel<TS_DTYPE_F16>, g, t, 0, st, a, fp8_vec(a), col_tiles);
  if (a.dtype == TS_DTYPE_BF16)
    return launch_pdl(fp8_quant_cols_kernel<TS_DTYPE_BF16>, g, t, 0, st, a, fp8_vec(a), col_tiles);
  return launch_pdl(fp8_quant_cols_kernel<TS_DTYPE_F32>, g, t, 0, st, a, fp8_vec(a), col_tiles);
}

cudaError_t launch_fp8_transpose(const uint8_t* codes, uint64_t ldw, const float* scales, uint32_t E, uint32_t N,
                                 uint32_t K, uint8_t* codes_t, uint64_t ldt, float* scales_t, cudaStream_t st) {
  const uint32_t k_tiles = (K + 63) / 64;
  const dim3 grid((N + 63) / 64 * k_tiles, E);
  fp8_transpose_kernel<<<grid, 256, 0, st>>>(codes, ldw, scales, N, K, codes_t, ldt, scales_t, k_tiles);
  return cudaGetLastError();
}

}  // namespace ts

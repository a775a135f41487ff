// k_fp8_quant.cu — quantising to e4m3 with a scale for each block of 128, by
// rows or by columns, and the relayout of a quantised weight by its columns.
//
// With a = max |x| over the finite values of a block: s = max(a * (1/448),
// 2^-100), r = 1/s, code = e4m3(x * r), every f32 step rounded to nearest.
//
// Every value is read once and every code written once.  By rows 65,536 x 640
// fp16 takes 22.5 us (5.7 of the 6.55 TB/s that a copy reaches; a warp issues
// in 68% of the cycles), by columns 16,391 x 1280 bf16 13.9 us (4.6 TB/s):
// there instructions bound it, 74% of the issue slots, with DRAM at 31% and
// nothing read but the input.  (Times of calls whose input changes from one to
// the next.)
#include "ts_fp8.cuh"
#include "ts_kernels.h"

#include <algorithm>

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
  const uint32_t i = blockIdx.x * 8 + (threadIdx.x >> 5), quad = i / nb;  // below 2^32 (launcher)
  const uint64_t row = (uint64_t)quad * 4 + (lane >> 3);
  const uint32_t b = i - quad * nb, c = b * kFp8Block + (lane & 7) * 16;
  if (row >= a.rows) return;
  Fp8Piece<DT> p;
  p.load(reinterpret_cast<const typename Fp8Type<DT>::T*>(a.x) + row * a.ldx, c, a.cols, vec);
  const float s = fp8_scale(p.block_max());
  if ((lane & 7) == 0) a.scales[b * a.lds + row] = s;
  if (c < a.cols) *reinterpret_cast<uint4*>(a.codes + row * a.ldc + c) = p.codes(fp8_inverse(s));
}

// Tiles of 128 rows x 128 bytes (64 or 32 columns) through shared memory: rows
// come in as they lie, by cp.async, and eight lanes then take one column (or,
// of 16-bit types, two neighbours), 16 rows a lane, so that a column's 128
// codes leave as one line.  Four words after every 16 rows put the eight
// lanes' rows into different banks.  The next tile is on its way while one is
// quantised: with each block waiting for its own loads alone, DRAM was a
// third as busy as it can be.
namespace qc {
constexpr uint32_t GROUP = 16 * 128 + 16;  // bytes of 16 rows
constexpr uint32_t TILE = 8 * GROUP;
constexpr uint32_t BLOCKS = 4;  // per SM (6 and 5 spill registers: 16.9 and 15.4 against 14.0 us, 16,391 x 1280 bf16)
}  // namespace qc

template <int DT>
__device__ __forceinline__ void fp8_cols_load(const Fp8QuantArgs& a, uint32_t vec, uint32_t b, uint32_t c0, uint8_t* tile) {
  using D = Fp8Type<DT>;
  using T = typename D::T;
  const T* x = reinterpret_cast<const T*>(a.x);
  if (vec) {
    constexpr uint32_t PER = 16 / sizeof(T);
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      const uint32_t r = j * 32 + (threadIdx.x >> 3), o = (threadIdx.x & 7) * 16, c = c0 + o / sizeof(T);
      const uint64_t row = (uint64_t)b * kFp8Block + r;
      const uint32_t n = row < a.rows && c < a.cols ? min(PER, a.cols - c) : 0u;  // the rest becomes zeros
      const T* src = n ? x + row * a.ldx + c : x;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       smem_u32(tile + (r >> 4) * qc::GROUP + (r & 15) * 128 + o)),
                   "l"(src), "r"(n * (uint32_t)sizeof(T))
                   : "memory");
    }
  } else {
    // value by value, a warp a row: 16 rows a warp, eight on their way together
    constexpr uint32_t STEPS = 128 / sizeof(T) / 32;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (uint32_t r0 = 0; r0 < 16; r0 += 8) {
      T v[8][STEPS];
#pragma unroll
      for (uint32_t j = 0; j < 8; j++)
#pragma unroll
        for (uint32_t l = 0; l < STEPS; l++) {
          const uint64_t row = (uint64_t)b * kFp8Block + warp * 16 + r0 + j;
          const uint32_t c = c0 + l * 32 + lane;
          v[j][l] = row < a.rows && c < a.cols ? x[row * a.ldx + c] : D::down(0.0f);
        }
#pragma unroll
      for (uint32_t j = 0; j < 8; j++)
#pragma unroll
        for (uint32_t l = 0; l < STEPS; l++)
          reinterpret_cast<T*>(tile + warp * qc::GROUP + (r0 + j) * 128)[l * 32 + lane] = v[j][l];
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <int DT>
__global__ void __launch_bounds__(256, qc::BLOCKS)
    fp8_quant_cols_kernel(const Fp8QuantArgs a, uint32_t vec, uint32_t col_tiles, uint32_t tiles) {
  using D = Fp8Type<DT>;
  using T = typename D::T;
  constexpr uint32_t COLS = 128 / sizeof(T), W = sizeof(T) == 2 ? 2 : 1;  // columns a lane takes
  __shared__ __align__(16) uint8_t tile[2][qc::TILE];
  pdl_trigger();
  pdl_wait();
  uint32_t turn = 0;
  // block of rows and tile of columns; a step over the grid is the same pair each time
  uint32_t next_b = blockIdx.x / col_tiles, next_c = blockIdx.x % col_tiles;
  const uint32_t step_b = gridDim.x / col_tiles, step_c = gridDim.x % col_tiles;
  if (blockIdx.x < tiles) fp8_cols_load<DT>(a, vec, next_b, next_c * COLS, tile[0]);
  for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x, turn ^= 1) {
    const uint32_t b = next_b, c0 = next_c * COLS;
    next_b += step_b;
    next_c += step_c;
    if (next_c >= col_tiles) {
      next_c -= col_tiles;
      next_b++;
    }
    if (t + gridDim.x < tiles) {
      fp8_cols_load<DT>(a, vec, next_b, next_c * COLS, tile[turn ^ 1]);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const uint32_t col = threadIdx.x / 8 * W, g = threadIdx.x & 7;
    const uint8_t* src = tile[turn] + g * qc::GROUP + col * sizeof(T);
    uint32_t raw[16];  // of both columns
#pragma unroll
    for (uint32_t j = 0; j < 16; j++) raw[j] = *reinterpret_cast<const uint32_t*>(src + j * 128);
    const uint32_t row0 = b * kFp8Block + g * 16;
    uint32_t both = 0;  // 16-bit types: the largest magnitudes of both columns at once
    if constexpr (W == 2) {
#pragma unroll
      for (uint32_t j = 0; j < 16; j++) both = fp8_mag_max2<DT>(both, raw[j]);
#pragma unroll
      for (int d = 4; d; d >>= 1) both = fp8_mag_max2<DT>(both, __shfl_xor_sync(0xffffffffu, both, d));
    }
#pragma unroll
    for (uint32_t w = 0; w < W; w++) {
      Fp8Piece<DT> p;
#pragma unroll
      for (uint32_t j = 0; j < 16; j++) p.v[j] = D::up(reinterpret_cast<const T*>(&raw[j])[w]);
      float m = W == 2 ? D::up(reinterpret_cast<const T*>(&both)[w]) : p.block_max();
      if (W == 2 && !(m < __int_as_float(0x7f800000))) m = p.block_max();  // an infinity, which is left out
      const float s = fp8_scale(m);
      const uint64_t c = c0 + col + w;
      if (c >= a.cols) continue;
      if (g == 0) a.scales[b * a.lds + c] = s;
      if (row0 < a.rows) *reinterpret_cast<uint4*>(a.codes + c * a.ldc + row0) = p.codes(fp8_inverse(s));
    }
    __syncthreads();  // the tile's place is free for the load after the next
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
  if (grid > 0x1fffffffu) return cudaErrorInvalidValue;
  const dim3 g((uint32_t)grid), t(256);
  if (a.dtype == TS_DTYPE_F16) return launch_pdl(fp8_quant_rows_kernel<TS_DTYPE_F16>, g, t, 0, st, a, fp8_vec(a));
  if (a.dtype == TS_DTYPE_BF16) return launch_pdl(fp8_quant_rows_kernel<TS_DTYPE_BF16>, g, t, 0, st, a, fp8_vec(a));
  return launch_pdl(fp8_quant_rows_kernel<TS_DTYPE_F32>, g, t, 0, st, a, fp8_vec(a));
}

cudaError_t launch_fp8_quant_cols(const Fp8QuantArgs& a, cudaStream_t st) {
  const uint32_t cols = a.dtype == TS_DTYPE_F32 ? 32 : 64, col_tiles = a.cols / cols + (a.cols % cols != 0);
  const uint64_t tiles = (uint64_t)col_tiles * fp8_blocks(a.rows);
  if (tiles > 0x7fffffffu) return cudaErrorInvalidValue;
  const dim3 g((uint32_t)std::min<uint64_t>(tiles, (uint64_t)num_sms() * qc::BLOCKS)), t(256);
  const uint32_t n = (uint32_t)tiles;
  if (a.dtype == TS_DTYPE_F16)
    return launch_pdl(fp8_quant_cols_kernel<TS_DTYPE_F16>, g, t, 0, st, a, fp8_vec(a), col_tiles, n);
  if (a.dtype == TS_DTYPE_BF16)
    return launch_pdl(fp8_quant_cols_kernel<TS_DTYPE_BF16>, g, t, 0, st, a, fp8_vec(a), col_tiles, n);
  return launch_pdl(fp8_quant_cols_kernel<TS_DTYPE_F32>, g, t, 0, st, a, fp8_vec(a), col_tiles, n);
}

cudaError_t launch_fp8_transpose(const uint8_t* codes, uint64_t ldw, const float* scales, uint32_t E, uint32_t N,
                                 uint32_t K, uint8_t* codes_t, uint64_t ldt, float* scales_t, cudaStream_t st) {
  const uint32_t k_tiles = K / 64 + (K % 64 != 0), n_tiles = N / 64 + (N % 64 != 0);
  if ((uint64_t)n_tiles * k_tiles > 0x7fffffffu) return cudaErrorInvalidValue;
  const dim3 grid(n_tiles * k_tiles, E);
  fp8_transpose_kernel<<<grid, 256, 0, st>>>(codes, ldw, scales, N, K, codes_t, ldt, scales_t, k_tiles);
  return cudaGetLastError();
}

}  // namespace ts

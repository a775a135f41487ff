// k_fp8_matvec.cu — the 8-bit product for up to 16 rows of x (single tokens):
// the weight is read once, and quantising x is part of the same launch.
//
// out[m, n] = sum_b xs[b, m] ws[n / 128, b] (sum_{k in b} x[m, k] w[n, k]).
// What bounds it is reading the weight, so its codes go from global memory
// straight into the registers of mma.sync (e4m3, 16 x 8 x 32: legacy tensor
// path, no shared memory and no barrier per step between a load and its use).
// The sum over k does not care for its order, so a lane's operand words are
// the 16-byte pieces c and c + 4 of a block (c = lane % 4) of the weight's
// rows, taken in the same order from x.  A block of 8 warps owns 16 rows of
// the weight; warp i takes the 128-blocks i, i + 8, ..., four of them loaded
// ahead, and the warps' sums are added in a fixed order.  1 x 4096 x 4096 takes
// 5.9 us a call in a row of calls, the host's time for one; the weight's 16.8 MB
// take 2.6 us from DRAM.
#include "ts_fp8.cuh"

namespace ts {

namespace mv {
constexpr uint32_t ROWS = 16, WARPS = 8, AHEAD = 4;
}

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 codes from byte i of a row of n; bytes past its end may hold anything
// (a NaN among them) and become zero.
__device__ __forceinline__ uint4 mv_codes(const uint8_t* row, uint32_t i, uint32_t n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (i < n) {
    v = __ldg(reinterpret_cast<const uint4*>(row + i));
    if (i + 16 > n) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const uint32_t left = n > i + 4 * j ? n - i - 4 * j : 0;  // bytes of word j inside the row
        if (left < 4) w[j] &= (1u << (8 * left)) - 1u;
      }
    }
  }
  return v;
}

__device__ __forceinline__ void mv_store(const Fp8MvArgs& a, uint32_t m, uint32_t n, float v) {
  if (a.bias) v += __half2float(reinterpret_cast<const __half*>(a.bias)[n]);
  const uint64_t i = m * a.ldo + n;
  if (a.out_dtype == TS_DTYPE_F16) {
    static_cast<__half*>(a.out)[i] = __float2half_rn(v);
  } else if (a.out_dtype == TS_DTYPE_BF16) {
    static_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(v);
  } else {
    float* o = static_cast<float*>(a.out) + i;
    *o = a.accumulate ? v + *o : v;
  }
}

// XT: type of x (TS_DTYPE_U8: codes); NT: 8-row tiles of x.
template <int XT, int NT>
__global__ void __launch_bounds__(256) fp8_matvec_kernel(const Fp8MvArgs a, uint32_t vec) {
  using namespace mv;
  // a row of x's 128 codes of one chunk, per warp; pieces 0-3 and 4-7 of odd
  // rows change places, which keeps the reads below free of bank conflicts
  __shared__ __align__(16) uint4 xc[WARPS][NT * 8][8];
  __shared__ float xs[WARPS][NT * 8];
  __shared__ float red[WARPS][ROWS][NT * 8 + 1];
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const uint32_t n0 = blockIdx.x * ROWS, kb = fp8_blocks(a.K);
  for (uint32_t i = lane; i < NT * 8 * 8; i += 32) (&xc[warp][0][0])[i] = make_uint4(0, 0, 0, 0);
  for (uint32_t i = lane; i < NT * 8; i += 32) xs[warp][i] = 0.0f;
  __syncwarp();
  const uint8_t* w0 = a.w + (uint64_t)min(n0 + g, a.N - 1) * a.ldw;
  const uint8_t* w1 = a.w + (uint64_t)min(n0 + g + 8, a.N - 1) * a.ldw;
  const float* ws = a.ws + (uint64_t)(n0 / kFp8Block) * kb;
  float acc[NT][4] = {};
  for (uint32_t b0 = warp; b0 < kb; b0 += WARPS * AHEAD) {
    uint4 wl[AHEAD][2], wh[AHEAD][2];
    float wsc[AHEAD];
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; u++) {
      const uint32_t b = b0 + u * WARPS, k = b * kFp8Block + c * 16;
      wl[u][0] = mv_codes(w0, k, a.K);
      wl[u][1] = mv_codes(w1, k, a.K);
      wh[u][0] = mv_codes(w0, k + 64, a.K);
      wh[u][1] = mv_codes(w1, k + 64, a.K);
      wsc[u] = b < kb ? ws[b] : 0.0f;
    }
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; u++) {
      const uint32_t b = b0 + u * WARPS;
      if (b >= kb) break;
#pragma unroll
      for (uint32_t r = 0; r < NT * 8; r += 4) {  // eight lanes a row, four rows at once
        const uint32_t m = r + (lane >> 3), j = lane & 7, k = b * kFp8Block + j * 16;
        if (m >= a.M) continue;
        uint4 codes;
        float s;
        if constexpr (XT == TS_DTYPE_U8) {
          codes = mv_codes(static_cast<const uint8_t*>(a.x) + m * a.ldx, k, a.K);
          s = a.xs[b * a.ldxs + m];
        } else {
          Fp8Piece<XT> p;
          p.load(static_cast<const typename Fp8Type<XT>::T*>(a.x) + m * a.ldx, k, a.K, vec);
          s = fp8_scale(p.block_max());
          codes = p.codes(fp8_inverse(s));
        }
        xc[warp][m][j ^ ((m & 1) << 2)] = codes;
        if (j == 0) xs[warp][m] = s;
      }
      __syncwarp();
#pragma unroll
      for (uint32_t t = 0; t < NT; t++) {
        const uint4 xl = xc[warp][t * 8 + g][c ^ ((g & 1) << 2)], xh = xc[warp][t * 8 + g][(c + 4) ^ ((g & 1) << 2)];
        float d[4] = {};
        mma_e4m3(d, wl[u][0].x, wl[u][1].x, wh[u][0].x, wh[u][1].x, xl.x, xh.x);
        mma_e4m3(d, wl[u][0].y, wl[u][1].y, wh[u][0].y, wh[u][1].y, xl.y, xh.y);
        mma_e4m3(d, wl[u][0].z, wl[u][1].z, wh[u][0].z, wh[u][1].z, xl.z, xh.z);
        mma_e4m3(d, wl[u][0].w, wl[u][1].w, wh[u][0].w, wh[u][1].w, xl.w, xh.w);
        const float s0 = xs[warp][t * 8 + 2 * c] * wsc[u], s1 = xs[warp][t * 8 + 2 * c + 1] * wsc[u];
        acc[t][0] = fmaf(d[0], s0, acc[t][0]);
        acc[t][1] = fmaf(d[1], s1, acc[t][1]);
        acc[t][2] = fmaf(d[2], s0, acc[t][2]);
        acc[t][3] = fmaf(d[3], s1, acc[t][3]);
      }
      __syncwarp();
    }
  }
#pragma unroll
  for (uint32_t t = 0; t < NT; t++)
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) red[warp][g + (i >> 1) * 8][t * 8 + 2 * c + (i & 1)] = acc[t][i];
  __syncthreads();
  const uint32_t m = threadIdx.x / ROWS, n = threadIdx.x % ROWS;
  if (m < a.M && n0 + n < a.N) {
    float v = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < WARPS; i++) v += red[i][n][m];
    mv_store(a, m, n0 + n, v);
  }
}

template <int XT>
static cudaError_t launch_mv(const Fp8MvArgs& a, uint32_t vec, cudaStream_t st) {
  const dim3 grid((a.N + mv::ROWS - 1) / mv::ROWS), block(32 * mv::WARPS);
  if (a.M <= 8) return launch_pdl(fp8_matvec_kernel<XT, 1>, grid, block, 0, st, a, vec);
  return launch_pdl(fp8_matvec_kernel<XT, 2>, grid, block, 0, st, a, vec);
}

cudaError_t launch_fp8_matvec(const Fp8MvArgs& a, cudaStream_t st) {
  const uint32_t vec = !(reinterpret_cast<uintptr_t>(a.x) & 15u) && a.ldx * (a.x_dtype == TS_DTYPE_F32 ? 4 : 2) % 16 == 0;
  if (a.x_dtype == TS_DTYPE_U8) return launch_mv<TS_DTYPE_U8>(a, vec, st);
  if (a.x_dtype == TS_DTYPE_F16) return launch_mv<TS_DTYPE_F16>(a, vec, st);
  if (a.x_dtype == TS_DTYPE_BF16) return launch_mv<TS_DTYPE_BF16>(a, vec, st);
  return launch_mv<TS_DTYPE_F32>(a, vec, st);
}

}  // namespace ts

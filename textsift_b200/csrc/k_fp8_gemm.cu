// k_fp8_gemm.cu — products of 8-bit operands with a scale for each block of
// 128: out[m, n] = sum_b as[b, m] ws[., b] (sum_{k in b} a[m, k] w[n, k]),
// on tcgen05.
//
// A block's scale multiplies the sum over its 128 k, so those 128 are one
// accumulation of the tensor core (four tcgen05.mma.kind::f8f6f4 of 32 k) and
// the sum over blocks is taken in registers: every chunk of 128 k has a TMEM
// buffer of its own, out of a ring, and 16 warps add it, times its scale, to
// accumulators that stay in registers for the whole tile (64 x f32 a thread
// at the widest).  Tiles are 128 rows of a by BN rows of w; thread = one row
// of a, so as is one value a thread and chunk, and ws one value a warp.
//
// Persistent, warp-specialized, one CTA per SM:
//   warp 0       TMA producer: per chunk a box of 128 rows x 128 bytes of a
//                and up to BN / 64 boxes of 64 rows of w (128-byte swizzle);
//                allocates TMEM
//   warp 1       MMA issuer
//   warps 2..17  scale and add: warp w owns TMEM lanes 32 (w % 4).. (rows) and
//                the columns of part (w - 2) / 4 of the tile; writes the tile
// The scales of the two chunks ahead are in registers before they are needed.
// All waits are bounded (ts_common.cuh) and set the device error flag.
#include "ts_fp8.cuh"
#include "ts_kernels.h"

#include <algorithm>

namespace ts {

static __device__ int g_fp8_err;

int* fp8_err_flag() {
  void* p = nullptr;
  return cudaGetSymbolAddress(&p, g_fp8_err) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

namespace f8 {
constexpr uint32_t BM = 128;                  // rows of a per tile = TMEM lanes
constexpr uint32_t A_BYTES = BM * kFp8Block;  // one chunk of a tile's rows
constexpr uint32_t W_BOX = 64;                // rows of w per TMA box
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t DRAIN_WARPS = 16;
constexpr uint32_t THREADS = 32 * (2 + DRAIN_WARPS);
constexpr uint32_t MAX_E = 1024;
constexpr uint32_t GROUP_M = 16;  // tiles of a that share their tiles of w in L2

template <int BN>
struct Cfg {
  static constexpr uint32_t W_BYTES = BN * kFp8Block;
  static constexpr uint32_t STAGE = A_BYTES + W_BYTES;
  static constexpr uint32_t S = BN == 256 ? 3 : BN == 128 ? 4 : 6;
  static constexpr uint32_t NB = TMEM_COLS / BN;      // TMEM buffers
  static constexpr uint32_t PART = BN / 4;            // columns a warp owns
  // a warp's rows on their way out: 32 of up to 128 bytes
  static constexpr uint32_t OUT_BYTES = 32 * (PART * 4 < 128 ? PART * 4 : 128);
  static constexpr uint32_t OFF_OUT = S * STAGE;
  static constexpr uint32_t OFF_BAR = OFF_OUT + DRAIN_WARPS * OUT_BYTES;
  static constexpr uint32_t NUM_BARS = 2 * S + 2 * NB + 1;
  static constexpr uint32_t OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr uint32_t OFF_SEG = OFF_MISC + 16;  // tile prefix of the segments, then their first rows
  // the scales of a warp's columns, three chunks deep (w_block 1)
  static constexpr uint32_t OFF_WS = (OFF_SEG + 16 + 15) / 16 * 16;
  static constexpr uint32_t SMEM_SEG = OFF_SEG + (2 * MAX_E + 2) * 4 + 1024;
  static constexpr uint32_t SMEM_ROW = OFF_WS + 3 * DRAIN_WARPS * PART * 4 + 1024;
  static_assert(STAGE % 1024 == 0, "swizzle atoms");
  static_assert(SMEM_SEG <= 227 * 1024 && SMEM_ROW <= 227 * 1024, "shared memory budget");
};
}  // namespace f8

struct Fp8Tile {
  uint32_t e, row0, row_end, n0;
};

// Tile t in an order that walks GROUP_M tiles of a for each tile of w.
__device__ __forceinline__ Fp8Tile fp8_tile(const Fp8MmArgs& a, uint32_t t, uint32_t m_tiles, uint32_t n_tiles, uint32_t bn,
                                            const uint32_t* pre, const int* first) {
  const uint32_t per = f8::GROUP_M * n_tiles, g = t / per, r = t - g * per;
  const uint32_t gm = min(f8::GROUP_M, m_tiles - g * f8::GROUP_M);
  const uint32_t m = g * f8::GROUP_M + r % gm;
  Fp8Tile ti;
  ti.n0 = r / gm * bn;
  if (a.seg) {
    uint32_t lo = 0, hi = a.E;  // pre[lo] <= m < pre[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (pre[mid] <= m) lo = mid;
      else hi = mid;
    }
    ti.e = lo;
    ti.row0 = (uint32_t)first[lo] + (m - pre[lo]) * f8::BM;
    ti.row_end = min(ti.row0 + f8::BM, (uint32_t)min(max(a.seg[lo + 1], 0), (int)a.M));
  } else {
    ti.e = 0;
    ti.row0 = m * f8::BM;
    ti.row_end = min(ti.row0 + f8::BM, a.M);
  }
  return ti;
}

__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x PART columns of f32 from TMEM.
template <int N>
__device__ __forceinline__ void fp8_tmem_ld(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_ld_32x32b_x32(addr, r);
  else tmem_ld_32x32b_x16(addr, r);
}

__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* smem_src, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(c0), "r"(c1), "r"(smem_u32(smem_src))
               : "memory");
}
// The same, added to what is there (f32).
__device__ __forceinline__ void tma_add_2d(const void* tmap, const void* smem_src, int32_t c0, int32_t c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(c0), "r"(c1), "r"(smem_u32(smem_src))
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// The thread's bulk stores have read their shared memory.
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int OT>
__device__ __forceinline__ uint32_t fp8_out2(float x0, float x1) {
  if constexpr (OT == TS_DTYPE_F16) {
    const __half2 h = __floats2half2_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 16 bytes of bias: the 8 columns from n.
__device__ __forceinline__ void fp8_bias8(const __half* bias, uint32_t n, uint32_t N, float (&b)[8]) {
  if (n + 8 <= N && !(reinterpret_cast<uintptr_t>(bias + n) & 15u)) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(bias + n));
    const __half* h = reinterpret_cast<const __half*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; i++) b[i] = __half2float(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) b[i] = n + i < N ? __half2float(bias[n + i]) : 0.0f;
  }
}

// Writes a warp's 32 rows (from row, those below row_end) x PART columns (from
// n), thread = row: acc + bias (+ what out holds).  The rows go through the
// warp's shared memory, 16-byte pieces swizzled as a tensor map of that row
// size has them, and leave by one TMA store where all 32 rows are this tile's
// (tma: out can be mapped), else row by row, consecutive lanes on consecutive
// columns.
template <int OT, int PART>
__device__ __forceinline__ void fp8_write(const Fp8MmArgs& a, const CUtensorMap* tmap_o, bool tma, uint8_t* stage,
                                          uint32_t e, uint32_t row, uint32_t row_end, uint32_t n,
                                          const uint64_t (&acc)[PART / 2]) {
  using D = Fp8Type<OT>;
  using T = typename D::T;
  constexpr uint32_t RB = PART * sizeof(T) < 128 ? PART * sizeof(T) : 128;  // bytes of a staged row
  constexpr uint32_t COLS = RB / sizeof(T), PER = 16 / sizeof(T);
  const uint32_t lane = threadIdx.x & 31;
  auto piece = [&](uint32_t r, uint32_t c) {  // piece c of staged row r
    return stage + r * RB + ((c ^ ((r * RB / 128) % (RB / 16))) * 16);
  };
  const bool whole = tma && row + 32 <= row_end;
#pragma unroll
  for (uint32_t c0 = 0; c0 < PART; c0 += COLS) {
    if (n + c0 >= a.N) break;
    if (lane == 0) bulk_wait_read();
    __syncwarp();
#pragma unroll
    for (uint32_t c = 0; c < COLS; c += 8) {
      float b[8] = {};
      if (a.bias) fp8_bias8(reinterpret_cast<const __half*>(a.bias) + (uint64_t)e * a.N, n + c0 + c, a.N, b);
      uint32_t w[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; i += 2) {
        float x0, x1;
        f2unpack(acc[(c0 + c + i) / 2], x0, x1);
        x0 += b[i];
        x1 += b[i + 1];
        if constexpr (OT == TS_DTYPE_F32) {
          w[i] = __float_as_uint(x0);
          w[i + 1] = __float_as_uint(x1);
        } else {
          w[i / 2] = fp8_out2<OT>(x0, x1);
        }
      }
      *reinterpret_cast<uint4*>(piece(lane, c / PER)) = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (OT == TS_DTYPE_F32) *reinterpret_cast<uint4*>(piece(lane, c / PER + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
    }
    if (whole) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (OT == TS_DTYPE_F32 && a.accumulate) tma_add_2d(tmap_o, stage, (int32_t)(n + c0), (int32_t)row);
        else tma_store_2d(tmap_o, stage, (int32_t)(n + c0), (int32_t)row);
        bulk_commit();
      }
    } else {
      __syncwarp();
      for (uint32_t r = 0; r < 32 && row + r < row_end; r++) {
        T* o = reinterpret_cast<T*>(a.out) + (uint64_t)(row + r) * a.ldo + n + c0;
        for (uint32_t c = lane; c < COLS && n + c0 + c < a.N; c += 32) {
          const T v = reinterpret_cast<const T*>(piece(r, c / PER))[c % PER];
          if (OT == TS_DTYPE_F32 && a.accumulate) o[c] = D::down(D::up(v) + D::up(o[c]));
          else o[c] = v;
        }
      }
      __syncwarp();
    }
  }
}

template <int BN, int WB, int OT>
__global__ void __launch_bounds__(f8::THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                    const __grid_constant__ CUtensorMap tmap_o, const Fp8MmArgs args, uint32_t n_tiles, uint32_t tma_out) {
  using namespace f8;
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_dyn[];
  pdl_trigger();
  pdl_wait();
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [S] a chunk of both operands landed
  uint64_t* empty = full + C::S;                                   // [S] its MMAs completed
  uint64_t* acc_full = empty + C::S;                               // [NB] a chunk's product is in TMEM
  uint64_t* acc_empty = acc_full + C::NB;                          // [NB] the 16 warps have read it
  uint64_t* drain = acc_empty + C::NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  uint32_t* pre = reinterpret_cast<uint32_t*>(smem + C::OFF_SEG);  // [E + 1] tiles before each segment
  int* first = reinterpret_cast<int*>(pre + MAX_E + 1);            // [E] first row of each segment
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < C::S; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < C::NB; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], DRAIN_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (args.seg && warp == 1) {
    // tiles before each segment: lane l sums the tiles of segments 32 l ..
    uint32_t sum = 0;
    for (uint32_t i = 0; i < MAX_E / 32; i++) {
      const uint32_t e = lane * (MAX_E / 32) + i;
      if (e >= args.E) break;
      const int lo = min(max(args.seg[e], 0), (int)args.M), hi = min(max(args.seg[e + 1], lo), (int)args.M);
      first[e] = lo;
      pre[e] = sum;
      sum += (uint32_t)(hi - lo + (int)BM - 1) / BM;
    }
    uint32_t incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    for (uint32_t i = 0; i < MAX_E / 32; i++) {
      const uint32_t e = lane * (MAX_E / 32) + i;
      if (e < args.E) pre[e] += incl - sum;
    }
    if (lane == 31) pre[args.E] = incl;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t n_kc = fp8_blocks(args.K);
  const uint32_t m_tiles = args.seg ? pre[args.E] : (args.M + BM - 1) / BM;
  const uint32_t total = m_tiles * n_tiles;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const Fp8Tile ti = fp8_tile(args, t, m_tiles, n_tiles, BN, pre, first);
        const uint32_t boxes = (min((uint32_t)BN, args.N - ti.n0) + W_BOX - 1) / W_BOX;
        const int32_t wrow = (int32_t)(ti.e * args.N + ti.n0);
        for (uint32_t kc = 0; kc < n_kc; kc++, it++) {
          const uint32_t s = it % C::S, u = it / C::S;
          if (!wait_or_abort(&empty[s], (u & 1u) ^ 1u, args.err, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::STAGE;
          mbar_arrive_expect_tx(&full[s], A_BYTES + boxes * W_BOX * kFp8Block);
          tma_load_2d(st, &tmap_a, (int32_t)(kc * kFp8Block), (int32_t)ti.row0, &full[s]);
          for (uint32_t b = 0; b < boxes; b++)
            tma_load_2d(st + A_BYTES + b * W_BOX * kFp8Block, &tmap_w, (int32_t)(kc * kFp8Block),
                        wrow + (int32_t)(b * W_BOX), &full[s]);
        }
      }
      if (!ok)  // the copies in flight land before this CTA's shared memory goes
        for (uint32_t j = it > C::S ? it - C::S : 0u; j < it; j++) mbar_wait(&full[j % C::S], (j / C::S) & 1u, args.err);
    }
  } else if (warp == 1) {
    const uint64_t adesc0 = umma_desc_sw128(smem_u32(smem)), wdesc0 = umma_desc_sw128(smem_u32(smem + A_BYTES));
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const Fp8Tile ti = fp8_tile(args, t, m_tiles, n_tiles, BN, pre, first);
      // as many columns as the tile has, in steps of 16
      const uint32_t idesc = umma_idesc_f16_f32(BM, (min((uint32_t)BN, args.N - ti.n0) + 15u) & ~15u);
      for (uint32_t kc = 0; kc < n_kc; kc++, it++) {
        const uint32_t s = it % C::S, b = it % C::NB;
        ok = __all_sync(0xffffffffu, wait_or_abort(&acc_empty[b], ((it / C::NB) & 1u) ^ 1u, args.err, abort_flag) &&
                                         wait_or_abort(&full[s], (it / C::S) & 1u, args.err, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t off = (uint64_t)(s * (C::STAGE >> 4));
#pragma unroll
          for (uint32_t k = 0; k < 4; k++)  // 32 k = 32 bytes = 2 descriptor units
            tc_mma_f8(tmem_base + b * BN, adesc0 + off + 2u * k, wdesc0 + off + 2u * k, idesc, k != 0);
          tc_commit(&empty[s]);
          tc_commit(&acc_full[b]);
        }
        __syncwarp();
      }
    }
    if (elect_one()) tc_commit(drain);
    __syncwarp();
    if (lane == 0) mbar_wait(drain, 0, args.err);
  } else {
    constexpr int PART = (int)C::PART, LD = PART == 32 ? 32 : 16;
    const uint32_t q = (uint32_t)(warp & 3), p = (uint32_t)(warp - 2) >> 2;
    const uint32_t taddr = tmem_base + ((q * 32u) << 16) + p * PART;
    const uint32_t nb = fp8_blocks(args.N);
    uint8_t* stage = smem + C::OFF_OUT + (warp - 2) * C::OUT_BYTES;
    // scales of row m and of column block (or columns) n, chunk c
    float* ring = reinterpret_cast<float*>(smem + C::OFF_WS) + (warp - 2) * PART;
    auto a_scale = [&](uint32_t m, uint32_t c) { return args.as[c * args.ldas + min(m, args.M - 1)]; };
    auto w_scale = [&](const Fp8Tile& ti, uint32_t c) {
      const uint32_t n = min(ti.n0 + p * PART, args.N - 1);
      return args.ws[((uint64_t)ti.e * nb + n / kFp8Block) * n_kc + c];
    };
    auto w_rows = [&](const Fp8Tile& ti, uint32_t c) {  // into slot c % 3 of this warp's ring
#pragma unroll
      for (int j = lane; j < PART; j += 32)
        ring[(c % 3) * DRAIN_WARPS * PART + j] = args.ws[c * args.ldws + min(ti.n0 + p * PART + j, args.N - 1)];
    };
    float a0 = 0, a1 = 0, w0 = 0, w1 = 0;
    auto ahead = [&](const Fp8Tile& ti) {  // the first two chunks of a tile
      const uint32_t m = ti.row0 + q * 32u + lane;
      a0 = a_scale(m, 0);
      a1 = n_kc > 1 ? a_scale(m, 1) : 0.0f;
      if constexpr (WB == 1) {
        __syncwarp();
        w_rows(ti, 0);
        if (n_kc > 1) w_rows(ti, 1);
      } else {
        w0 = w_scale(ti, 0);
        w1 = n_kc > 1 ? w_scale(ti, 1) : 0.0f;
      }
    };
    Fp8Tile ti{};
    if (blockIdx.x < total) {
      ti = fp8_tile(args, blockIdx.x, m_tiles, n_tiles, BN, pre, first);
      ahead(ti);
    }
    uint32_t it = 0;
    for (uint32_t t = blockIdx.x; t < total; t += gridDim.x) {
      const uint32_t m = ti.row0 + q * 32u + lane;
      uint64_t acc[PART / 2];
#pragma unroll
      for (int j = 0; j < PART / 2; j++) acc[j] = 0;
      bool ok = true;
      for (uint32_t kc = 0; kc < n_kc; kc++, it++) {
        const uint32_t b = it % C::NB;
        const float s = WB == 1 ? a0 : a0 * w0;
        const uint64_t s2 = f2pack(s, s);
        a0 = a1;
        w0 = w1;
        if (kc + 2 < n_kc) {
          a1 = a_scale(m, kc + 2);
          if constexpr (WB != 1) w1 = w_scale(ti, kc + 2);
        }
        if constexpr (WB == 1) {
          __syncwarp();  // slot kc % 3 is written, slot (kc + 2) % 3 has been read
          if (kc + 2 < n_kc) w_rows(ti, kc + 2);
        }
        if (!wait_or_abort(&acc_full[b], (it / C::NB) & 1u, args.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < PART; c += LD) {
          uint32_t r[LD];
          fp8_tmem_ld<LD>(taddr + b * BN + c, r);
          tmem_ld_wait();
          if (c + LD >= PART) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
          }
#pragma unroll
          for (int j = 0; j < LD; j += 2) {
            uint64_t v = f2pack(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
            if constexpr (WB == 1) {
              const float2 w = *reinterpret_cast<const float2*>(ring + (kc % 3) * DRAIN_WARPS * PART + c + j);
              v = mul_f32x2(v, f2pack(w.x, w.y));
            }
            acc[(c + j) / 2] = fma_f32x2(v, s2, acc[(c + j) / 2]);
          }
        }
      }
      if (!ok) break;
      const Fp8Tile done = ti;
      if (t + gridDim.x < total) {
        ti = fp8_tile(args, t + gridDim.x, m_tiles, n_tiles, BN, pre, first);
        ahead(ti);
      }
      fp8_write<OT, PART>(args, &tmap_o, tma_out, stage, done.e, done.row0 + q * 32u, done.row_end, done.n0 + p * PART, acc);
    }
    if (lane == 0) bulk_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int BN, int WB, int OT>
static cudaError_t launch_gemm(const CUtensorMap& ta, const CUtensorMap& tw, const Fp8MmArgs& a, uint64_t m_tiles,
                               cudaStream_t st) {
  using C = f8::Cfg<BN>;
  static std::atomic<uint64_t> attr_done{0};
  constexpr uint32_t smem = WB == 1 ? C::SMEM_ROW : C::SMEM_SEG;
  if (cudaError_t e = smem_attr_per_device(fp8_gemm_kernel<BN, WB, OT>, (int)smem, attr_done); e != cudaSuccess) return e;
  const uint32_t n_tiles = (a.N + BN - 1) / BN;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(m_tiles * n_tiles, (uint64_t)num_sms());
  // out as 16-byte pieces of rows that can be mapped: the tensor map's box is a
  // warp's 32 rows of up to 128 bytes
  constexpr uint32_t size = sizeof(typename Fp8Type<OT>::T), bytes = std::min<uint32_t>(C::PART * size, 128);
  CUtensorMap to = ta;
  const uint32_t tma_out = make_out_tmap(&to, a.out, OT, a.M, a.N, a.ldo, bytes / size, 32) ? 1 : 0;
  return launch_pdl(fp8_gemm_kernel<BN, WB, OT>, dim3(grid), dim3(f8::THREADS), smem, st, ta, tw, to, a, n_tiles, tma_out);
}

template <int BN, int WB>
static cudaError_t launch_gemm_out(const CUtensorMap& ta, const CUtensorMap& tw, const Fp8MmArgs& a, uint64_t m_tiles,
                                   cudaStream_t st) {
  if (a.out_dtype == TS_DTYPE_F16) return launch_gemm<BN, WB, TS_DTYPE_F16>(ta, tw, a, m_tiles, st);
  if (a.out_dtype == TS_DTYPE_BF16) return launch_gemm<BN, WB, TS_DTYPE_BF16>(ta, tw, a, m_tiles, st);
  return launch_gemm<BN, WB, TS_DTYPE_F32>(ta, tw, a, m_tiles, st);
}

// K = 0: bias or zero (+ what out holds) on the rows that a segment covers.
template <int OT>
__global__ void __launch_bounds__(256) fp8_empty_sum_kernel(const Fp8MmArgs a) {
  using D = Fp8Type<OT>;
  for (uint32_t e = 0; e < a.E; e++) {
    const int lo = a.seg ? min(max(a.seg[e], 0), (int)a.M) : 0;
    const int hi = a.seg ? min(max(a.seg[e + 1], 0), (int)a.M) : (int)a.M;
    for (int m = lo + (int)blockIdx.x; m < hi; m += gridDim.x)
      for (uint32_t n = threadIdx.x; n < a.N; n += 256) {
        auto* o = reinterpret_cast<typename D::T*>(a.out) + (uint64_t)m * a.ldo + n;
        float v = a.bias ? __half2float(reinterpret_cast<const __half*>(a.bias)[(uint64_t)e * a.N + n]) : 0.0f;
        if (a.accumulate) v += D::up(*o);
        *o = D::down(v);
      }
  }
}

cudaError_t launch_fp8_matmul(const Fp8MmArgs& a, cudaStream_t st) {
  if (a.K == 0) {
    const uint32_t grid = std::min(a.M, 4096u);
    if (a.out_dtype == TS_DTYPE_F16) fp8_empty_sum_kernel<TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
    else if (a.out_dtype == TS_DTYPE_BF16) fp8_empty_sum_kernel<TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
    else fp8_empty_sum_kernel<TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
  }
  if (a.M <= kFp8MatvecRows && a.w_block != 1 && !a.seg) {
    Fp8MvArgs v;
    v.x = a.a; v.x_dtype = TS_DTYPE_U8; v.ldx = a.lda; v.xs = a.as; v.ldxs = a.ldas; v.w = a.w; v.ldw = a.ldw;
    v.ws = a.ws; v.bias = a.bias; v.out = a.out; v.out_dtype = a.out_dtype; v.ldo = a.ldo; v.accumulate = a.accumulate;
    v.M = a.M; v.N = a.N; v.K = a.K;
    return launch_fp8_matvec(v, st);
  }
  CUtensorMap ta, tw;
  if (!make_codes_tmap(&ta, a.a, a.M, a.K, a.lda, f8::BM) ||
      !make_codes_tmap(&tw, a.w, (uint64_t)a.E * a.N, a.K, a.ldw, f8::W_BOX))
    return cudaErrorInvalidValue;
  // tiles of a: exact without segments; with them, an upper bound of what
  // M rows in E segments can make
  const uint64_t m_tiles = a.seg ? a.M / f8::BM + std::min(a.E, a.M) : (a.M + f8::BM - 1) / f8::BM;
  // the widest tile that still gives every SM one
  const uint64_t sms = (uint64_t)num_sms();
  auto fills = [&](uint32_t bn) { return m_tiles * ((a.N + bn - 1) / bn) >= sms; };
  if (a.w_block == 1) {
    if (fills(256)) return launch_gemm_out<256, 1>(ta, tw, a, m_tiles, st);
    if (fills(128)) return launch_gemm_out<128, 1>(ta, tw, a, m_tiles, st);
    return launch_gemm_out<64, 1>(ta, tw, a, m_tiles, st);
  }
  if (fills(256)) return launch_gemm_out<256, 128>(ta, tw, a, m_tiles, st);
  if (fills(128)) return launch_gemm_out<128, 128>(ta, tw, a, m_tiles, st);
  return launch_gemm_out<64, 128>(ta, tw, a, m_tiles, st);
}

}  // namespace ts

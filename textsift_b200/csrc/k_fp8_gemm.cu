// k_fp8_gemm.cu — products of 8-bit operands with a scale for each block of
// 128: out[m, n] = sum_b as[b, m] ws[., b] (sum_{k in b} a[m, k] w[n, k]),
// on tcgen05.
//
// A block's scale multiplies the sum over its 128 k, so those 128 are one
// accumulation of the tensor core (four tcgen05.mma.kind::f8f6f4 of 32 k) and
// the sum over blocks is taken in registers: every chunk of 128 k has a TMEM
// buffer of its own, out of a ring, and 8 warps add it, times its scale, to
// accumulators that stay in registers for the whole tile (128 x f32 a thread
// at the widest).  Thread = one row of a, so as is one value a thread and
// chunk, and ws one value a warp.  Where w has a scale for each row (w_block
// 1), that layout would read as many scales as it adds values, and reading one
// address by all lanes costs its bytes 32 times; TMEM is then read in the 16 x
// 8 fragments of an mma (FRAG): four rows and a quarter of the columns a
// thread, a quarter of the scales.
//
// Large products run on CTA pairs (cta_group::2, CG = 2): 256 rows of a by 256
// rows of w, each CTA holding its half of both in shared memory and 128 of the
// rows in its TMEM, so a chunk costs 32 KB of copies a CTA instead of 48; the
// others on single CTAs with 128 rows of a by 128 or 64 of w.
//
// Where the tiles are too few for the GPU and k is long, a cluster of 2, 4 or 8
// CTAs shares a tile (SPLIT): each sums a range of its chunks, the sums meet in
// distributed shared memory and are added in the order of the ranges.
//
// Persistent, warp-specialized, one CTA per SM:
//   warp 0       TMA producer: per chunk a box of 128 rows x 128 bytes of a
//                and boxes of 64 rows of w (128-byte swizzle)
//   warp 1       MMA issuer (the pair's first CTA)
//   warp 2       allocates TMEM
//   warp 3       loads the scales, four chunks at a time (4-byte cp.async:
//                a segment's first row has any alignment)
//   warps 4..11  scale and add: warp w owns TMEM lanes 32 (w % 4).. (rows) and
//                half (w - 4) / 4 of the tile's columns; writes the tile.
//                They take the registers that the others do not need.
// The waits on mbarriers are bounded (ts_common.cuh) and set the device error
// flag.  The cluster barriers and the TMEM allocation have no limit of their
// own and need none: every thread of a cluster comes to each barrier after its
// bounded waits, whether they succeeded or not, and a block takes 64,512 of the
// SM's 65,536 registers, so no kernel of this library that takes TMEM for
// longer than a bounded wait is on the SM beside it.
//
// What bounds it: the tensor core stands still while TMEM is read, 128 KB for
// each 128 x 256 x 128; at 8192^3 the MMAs with their copies alone take 373 us,
// with TMEM read beside them 485, all of it 539 to 545 (2.0 PFLOP/s; 2.95 and
// 2.27 for the others).  At k = 640 a tile's output is 2,500 of its 8,300
// cycles: 65,536 x 1152 x 640 takes 82 us, with a bias 100, 128 experts' 262,144
// x 1280 x 640 378 us (1.14 PFLOP/s).  These are times of one call repeated on
// the same inputs, on one B200; with inputs that change from call to call
// 8192^3 takes 622 us (power), 65,536 x 1152 x 640 with a bias 96, the experts
// 426.
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
constexpr uint32_t BM = 128;                  // rows of a per CTA = TMEM lanes
constexpr uint32_t A_BYTES = BM * kFp8Block;  // one chunk of them
constexpr uint32_t W_BOX = 64;                // rows of w per TMA box
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t FIRST_DRAIN = 4, DRAIN_WARPS = 8;
constexpr uint32_t THREADS = 32 * (FIRST_DRAIN + DRAIN_WARPS);
// registers a thread: 168 at launch, moved to the warps that add
constexpr uint32_t REGS_LAUNCH = 168, REGS_ROLES = 40, REGS_DRAIN = 232;
static_assert(REGS_ROLES * 32 * FIRST_DRAIN + REGS_DRAIN * 32 * DRAIN_WARPS <= REGS_LAUNCH * THREADS, "register split");
constexpr uint32_t MAX_E = 1024;
constexpr uint32_t GROUP_M = 16;  // tiles of a that share their tiles of w in L2
constexpr uint32_t BATCH = 4;     // chunks whose scales are loaded together
constexpr uint32_t SB = 2;        // such batches in flight

template <int CG, int BN, int WB>
struct Cfg {
  static constexpr uint32_t W_ROWS = BN / CG;  // rows of w that a CTA holds
  static constexpr uint32_t STAGE = A_BYTES + W_ROWS * kFp8Block;
  static constexpr uint32_t S = BN == 64 ? 6 : 4;
  static constexpr uint32_t NB = TMEM_COLS / BN;  // TMEM buffers
  static constexpr uint32_t PART = BN / 2;        // columns a warp owns
  // a warp's rows on their way out: twice 32 of up to 128 bytes
  static constexpr uint32_t OUT_BYTES = 2 * 32 * 128;
  static constexpr uint32_t OFF_OUT = S * STAGE;
  // scales of a chunk: of the CTA's rows of a, then of the tile's columns, one
  // for each (w_block 1) or for each 128
  static constexpr uint32_t W_SCALES = WB == 1 ? BN : (BN + 127) / 128, SCALES = BM + (W_SCALES + 3) / 4 * 4;
  static constexpr uint32_t OFF_SCALES = OFF_OUT + DRAIN_WARPS * OUT_BYTES;
  static constexpr uint32_t OFF_BIAS = OFF_SCALES + SB * BATCH * SCALES * 4;  // a warp's columns' bias
  static constexpr uint32_t OFF_BAR = OFF_BIAS + DRAIN_WARPS * PART * 2;
  static constexpr uint32_t NUM_BARS = 2 * S + 2 * NB + 2 * SB + 1;
  static constexpr uint32_t OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr uint32_t OFF_SEG = OFF_MISC + 16;  // tile prefix of the segments, then their first rows
  static constexpr uint32_t SMEM = OFF_SEG + (WB == 1 ? 0 : (2 * MAX_E + 2) * 4) + 1024;
  static_assert(STAGE % 1024 == 0, "swizzle atoms");
  static_assert(OFF_BAR % 8 == 0 && SMEM <= 227 * 1024, "shared memory budget");
};
}  // namespace f8

struct Fp8Tile {
  uint32_t e, row0, row_end, n0;
};

// Walks the tiles of bm x bn that are `first`, `first + step`, ... in an order
// that takes GROUP_M tiles of a for each tile of w.
struct Fp8Walk {
  uint32_t m_tiles, n_tiles, step, bm, bn;
  uint32_t g, r;  // group of tiles of a, place in it

  __device__ __forceinline__ Fp8Walk(uint32_t m_tiles_, uint32_t n_tiles_, uint32_t start, uint32_t step_, uint32_t bm_,
                                     uint32_t bn_)
      : m_tiles(m_tiles_), n_tiles(n_tiles_), step(step_), bm(bm_), bn(bn_), g(0), r(start) {
    settle();
  }
  __device__ __forceinline__ uint32_t tiles_of_a() const { return min(f8::GROUP_M, m_tiles - g * f8::GROUP_M); }
  __device__ __forceinline__ void settle() {
    while (more() && r >= tiles_of_a() * n_tiles) {
      r -= tiles_of_a() * n_tiles;
      g++;
    }
  }
  __device__ __forceinline__ bool more() const { return g * f8::GROUP_M < m_tiles; }
  __device__ __forceinline__ void next() {
    r += step;
    settle();
  }
  __device__ __forceinline__ Fp8Tile tile(const Fp8MmArgs& a, const uint32_t* pre, const int* first) const {
    const uint32_t gm = tiles_of_a(), n = gm == f8::GROUP_M ? r / f8::GROUP_M : r / gm, m = g * f8::GROUP_M + r - n * gm;
    Fp8Tile ti;
    ti.n0 = n * bn;
    if (a.seg) {
      uint32_t lo = 0, hi = a.E;  // pre[lo] <= m < pre[hi]
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (pre[mid] <= m) lo = mid;
        else hi = mid;
      }
      ti.e = lo;
      ti.row0 = (uint32_t)first[lo] + (m - pre[lo]) * bm;
      ti.row_end = min(ti.row0 + bm, (uint32_t)min(max(__ldg(&a.seg[lo + 1]), 0), (int)a.M));
    } else {
      ti.e = 0;
      ti.row0 = m * bm;
      ti.row_end = min(ti.row0 + bm, a.M);
    }
    return ti;
  }
};

// --- PTX of single CTAs and of pairs (cta_group::2) ---
template <uint32_t N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <uint32_t N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Shared-memory address of the same variable in the pair's first CTA.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
template <int CG>
__device__ __forceinline__ void fp8_tmem_alloc(uint32_t* slot, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void fp8_tmem_dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
template <int CG>
__device__ __forceinline__ void fp8_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on bar, in both CTAs of a pair, once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void fp8_commit(uint64_t* bar) {
  if constexpr (CG == 1) tc_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// The same for this CTA's barrier alone.
template <int CG>
__device__ __forceinline__ void fp8_commit_own(uint64_t* bar) {
  if constexpr (CG == 1) tc_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// A tile into this CTA's shared memory; its bytes count on the barrier at bar
// (of a pair: the first CTA's).
template <int CG>
__device__ __forceinline__ void fp8_load(void* dst, const void* tmap, int32_t c0, int32_t c1, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}

// A load that stays where it is written.
__device__ __forceinline__ uint16_t ld_u16(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
// 4 bytes to shared memory, asynchronously; the barrier gets this thread's
// arrival once all its copies so far have landed.
__device__ __forceinline__ void cp_async_4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// 32 lanes x N columns of f32 from TMEM, thread = lane.  The wait is part of
// the load, so nothing can use the values before.
template <int N>
__device__ __forceinline__ void fp8_ld(uint32_t addr, float (&r)[N]);
template <>
__device__ __forceinline__ void fp8_ld<64>(uint32_t addr, float (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
        "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]), "=f"(r[38]), "=f"(r[39]),
        "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]), "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]),
        "=f"(r[48]), "=f"(r[49]), "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
        "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]), "=f"(r[62]), "=f"(r[63])
      : "r"(addr)
      : "memory");
}
template <>
__device__ __forceinline__ void fp8_ld<32>(uint32_t addr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr)
      : "memory");
}
// 16 lanes x 2 N columns: thread t gets, of each 8 columns g, columns 2 (t % 4)
// and + 1 of lane t / 4 in r[4 g], r[4 g + 1] and of lane t / 4 + 8 in the
// next two.
template <int N>
__device__ __forceinline__ void fp8_ld_frag(uint32_t addr, float (&r)[N]);
template <>
__device__ __forceinline__ void fp8_ld_frag<64>(uint32_t addr, float (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x16.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
        "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]), "=f"(r[38]), "=f"(r[39]),
        "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]), "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]),
        "=f"(r[48]), "=f"(r[49]), "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
        "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]), "=f"(r[62]), "=f"(r[63])
      : "r"(addr)
      : "memory");
}
template <>
__device__ __forceinline__ void fp8_ld_frag<32>(uint32_t addr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void prefetch_tmap(const void* tmap) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tmap)) : "memory");
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
// All but the last LEFT groups of the thread's bulk stores have read their shared memory.
template <int LEFT>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}
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

// Writes a warp's 32 rows (from row, those below row_end) x PART columns (from
// n), thread = row (or fragments): acc (+ what out holds).  The rows go through
// the warp's shared memory, two turns of 32 x 128 bytes so that one is filled
// while the other leaves, their 16-byte pieces swizzled as a tensor map of that
// row size has them, and leave by one TMA store where all 32 rows are this
// tile's (tma: out can be mapped), else row by row, consecutive lanes on
// consecutive columns.  (Measured at 65,536 x 1152 x 640 without bias, one call
// repeated: 80 us; the four warps
// of a column half behind one store of 128 rows 88 us; the stores issued by a
// warp of their own 83 us; whole lines by ordinary stores from shared memory
// 98 us.)
template <int OT, int PART, bool FRAG>
__device__ __forceinline__ void fp8_write(const Fp8MmArgs& a, const CUtensorMap* tmap_o, bool tma, uint8_t* stages,
                                          uint32_t& turn, uint32_t row, uint32_t row_end, uint32_t n,
                                          const float (&acc)[PART]) {
  using D = Fp8Type<OT>;
  using T = typename D::T;
  constexpr uint32_t RB = PART * sizeof(T) < 128 ? PART * sizeof(T) : 128;  // bytes of a staged row
  constexpr uint32_t COLS = RB / sizeof(T), PER = 16 / sizeof(T);
  const uint32_t lane = threadIdx.x & 31;
  uint8_t* stage = stages;
  auto piece = [&](uint32_t r, uint32_t c) {  // piece c of staged row r
    return stage + r * RB + ((c ^ ((r * RB / 128) % (RB / 16))) * 16);
  };
  const bool whole = tma && row + 32 <= row_end;
#pragma unroll
  for (uint32_t c0 = 0; c0 < PART; c0 += COLS) {
    if (n + c0 < a.N) {
      stage = stages + (turn++ & 1u) * (32 * 128);
      if (lane == 0) bulk_wait_read<1>();  // the store before the last has left this turn's place
      __syncwarp();
      if constexpr (FRAG) {
#pragma unroll
        for (uint32_t c = 0; c < COLS; c += 8) {
          const uint32_t col = c + (lane & 3) * 2;
#pragma unroll
          for (uint32_t i = 0; i < 4; i++) {  // rows lane / 4, + 8, + 16, + 24
            const float* v = &acc[((i >> 1) * (PART / 8) + (c0 + c) / 8) * 4 + (i & 1) * 2];
            uint8_t* dst = piece(i * 8 + (lane >> 2), col / PER) + col % PER * sizeof(T);
            if constexpr (OT == TS_DTYPE_F32) *reinterpret_cast<float2*>(dst) = make_float2(v[0], v[1]);
            else *reinterpret_cast<uint32_t*>(dst) = fp8_out2<OT>(v[0], v[1]);
          }
        }
      } else {
#pragma unroll
        for (uint32_t c = 0; c < COLS; c += PER) {
          const float* v = &acc[c0 + c];
          uint4 w;
          if constexpr (OT == TS_DTYPE_F32)
            w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
          else
            w = make_uint4(fp8_out2<OT>(v[0], v[1]), fp8_out2<OT>(v[2], v[3]), fp8_out2<OT>(v[4], v[5]),
                           fp8_out2<OT>(v[6], v[7]));
          *reinterpret_cast<uint4*>(piece(lane, c / PER)) = w;
        }
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
        if (lane == 0) bulk_commit();  // an empty group keeps the count
        __syncwarp();
        constexpr uint32_t AT_ONCE = 8, STEPS = (COLS + 31) / 32;  // rows on their way together
        for (uint32_t r0 = 0; r0 < 32 && row + r0 < row_end; r0 += AT_ONCE) {
          T v[AT_ONCE][STEPS];
          T* o = reinterpret_cast<T*>(a.out) + (uint64_t)(row + r0) * a.ldo + n + c0;
          auto each = [&](auto f) {
#pragma unroll
            for (uint32_t r = 0; r < AT_ONCE; r++)
#pragma unroll
              for (uint32_t j = 0; j < STEPS; j++) {
                const uint32_t c = j * 32 + lane;
                if (c < COLS && n + c0 + c < a.N && row + r0 + r < row_end) f(r, c, v[r][j]);
              }
          };
          each([&](uint32_t r, uint32_t c, T& x) { x = reinterpret_cast<const T*>(piece(r0 + r, c / PER))[c % PER]; });
          if (OT == TS_DTYPE_F32 && a.accumulate)
            each([&](uint32_t r, uint32_t c, T& x) { x = D::down(D::up(x) + D::up(o[r * a.ldo + c])); });
          each([&](uint32_t r, uint32_t c, T& x) { o[r * a.ldo + c] = x; });
        }
        __syncwarp();
      }
    }
  }
}

// Place of 16-byte piece c of a row of BN floats: the rows of eight lanes that
// write the same piece lie in different banks.
template <int BN>
__device__ __forceinline__ uint32_t fp8_swizzle(uint32_t c, uint32_t row) {
  return c ^ (row & 7u);
}

// Adds the cluster's sums of a tile (f32 [128][BN] at the start of each CTA's
// shared memory) in the order of the CTAs; the adding warps of CTA `part` of
// `parts` write 128 / parts of the rows.
template <int BN, int OT>
__device__ __forceinline__ void fp8_join(const Fp8MmArgs& a, const Fp8Tile& ti, const uint8_t* smem, uint32_t part,
                                         uint32_t parts) {
  using D = Fp8Type<OT>;
  using T = typename D::T;
  const uint32_t rows = f8::BM / parts, base = smem_u32(smem);
  for (uint32_t i = threadIdx.x - 32 * f8::FIRST_DRAIN; i < rows * (BN / 4); i += 32 * f8::DRAIN_WARPS) {
    const uint32_t r = part * rows + i / (BN / 4), c = i % (BN / 4), m = ti.row0 + r, n = ti.n0 + c * 4;
    if (m >= ti.row_end || n >= a.N) continue;
    float4 v[8];  // all on their way before the first is added
#pragma unroll
    for (uint32_t s = 0; s < 8; s++)
      if (s < parts)
        asm volatile(
            "{\n\t.reg .b32 a;\n\t"
            "mapa.shared::cluster.u32 a, %4, %5;\n\t"
            "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
            : "=f"(v[s].x), "=f"(v[s].y), "=f"(v[s].z), "=f"(v[s].w)
            : "r"(base + (r * (BN / 4) + fp8_swizzle<BN>(c, r)) * 16), "r"(s)
            : "memory");
    float x[4] = {};
#pragma unroll
    for (uint32_t s = 0; s < 8; s++)
      if (s < parts) {
        x[0] += v[s].x;
        x[1] += v[s].y;
        x[2] += v[s].z;
        x[3] += v[s].w;
      }
    T* o = reinterpret_cast<T*>(a.out) + (uint64_t)m * a.ldo + n;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      if (n + j >= a.N) break;
      float v = x[j];
      if (a.bias) v += __half2float(__ushort_as_half(__ldg(&a.bias[(uint64_t)ti.e * a.N + n + j])));
      if (OT == TS_DTYPE_F32 && a.accumulate) v += D::up(o[j]);
      o[j] = D::down(v);
    }
  }
}

template <int CG, int BN, int WB, int OT, bool SPLIT>
__global__ void __launch_bounds__(f8::THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                    const __grid_constant__ CUtensorMap tmap_o, const Fp8MmArgs args, uint32_t n_tiles, uint32_t tma_out, uint32_t split) {
  using namespace f8;
  using C = Cfg<CG, BN, WB>;
  constexpr uint32_t TILE_M = CG * BM;
  static_assert(CG == 1 || !SPLIT, "a cluster is a pair or a split");
  extern __shared__ uint8_t smem_dyn[];
  pdl_trigger();
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [S] a chunk of both operands landed (all CTAs')
  uint64_t* empty = full + C::S;                                   // [S] its MMAs completed
  uint64_t* acc_full = empty + C::S;                               // [NB] a chunk's product is in TMEM
  uint64_t* acc_empty = acc_full + C::NB;                          // [NB] the adding warps (all CTAs') have read it
  uint64_t* sc_full = acc_empty + C::NB;                           // [SB] a batch of scales landed
  uint64_t* sc_empty = sc_full + SB;                               // [SB] the adding warps have read it
  uint64_t* drain = sc_empty + SB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  uint32_t* pre = reinterpret_cast<uint32_t*>(smem + C::OFF_SEG);  // [E + 1] tiles before each segment
  int* first = reinterpret_cast<int*>(pre + MAX_E + 1);            // [E] first row of each segment
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < C::S; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < C::NB; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], CG * DRAIN_WARPS);
    }
    for (uint32_t i = 0; i < SB; i++) {
      mbar_init(&sc_full[i], 32);
      mbar_init(&sc_empty[i], DRAIN_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) fp8_tmem_alloc<CG>(tmem_slot, TMEM_COLS);
  if (warp == 3 && lane == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_w);
    if (tma_out) prefetch_tmap(&tmap_o);
  }
  pdl_wait();  // global memory from here on
  if (args.seg && warp == 1) {
    // tiles before each segment: lane l sums the tiles of segments 32 l ..
    uint32_t sum = 0;
    for (uint32_t i = 0; i < MAX_E / 32; i++) {
      const uint32_t e = lane * (MAX_E / 32) + i;
      if (e >= args.E) break;
      const int lo = min(max(args.seg[e], 0), (int)args.M), hi = min(max(args.seg[e + 1], lo), (int)args.M);
      first[e] = lo;
      pre[e] = sum;
      sum += (uint32_t)(hi - lo + (int)TILE_M - 1) / TILE_M;
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
  if constexpr (CG == 2) cluster_sync();  // both CTAs' barriers are there
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t n_kc = fp8_blocks(args.K);
  // this CTA's chunks
  const uint32_t part = SPLIT ? cluster_rank() : 0, parts = SPLIT ? split : 1;
  const uint32_t k_lo = SPLIT ? n_kc * part / parts : 0, k_hi = SPLIT ? n_kc * (part + 1) / parts : n_kc;
  const uint32_t m_tiles = args.seg ? pre[args.E] : (args.M + TILE_M - 1) / TILE_M;
  Fp8Walk walk(m_tiles, n_tiles, blockIdx.x / (CG * parts), gridDim.x / (CG * parts), TILE_M, BN);
  const bool busy = walk.more();  // the same for all CTAs of a cluster
  // the MMA's columns: those that the tile has, in steps of 16; a CTA of a pair holds half
  auto columns = [&](uint32_t n0) { return (min((uint32_t)BN, args.N - n0) + 15u) & ~15u; };

  if (warp < (int)FIRST_DRAIN) {  // a warpgroup changes its registers as one
    regs_dec<REGS_ROLES>();
    if (warp == 0) {
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (; walk.more() && ok; walk.next()) {
          const Fp8Tile ti = walk.tile(args, pre, first);
          const uint32_t held = columns(ti.n0) / CG, boxes = (held + W_BOX - 1) / W_BOX;
          const int32_t wrow = (int32_t)(ti.e * args.N + ti.n0 + rank * held), arow = (int32_t)(ti.row0 + rank * BM);
          for (uint32_t kc = k_lo; kc < k_hi; kc++, it++) {
            const uint32_t s = it % C::S, u = it / C::S;
            if (!wait_or_abort(&empty[s], (u & 1u) ^ 1u, args.err, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* st = smem + s * C::STAGE;
            const uint32_t bar = CG == 2 ? leader_addr(&full[s]) : smem_u32(&full[s]);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], CG * (A_BYTES + boxes * W_BOX * kFp8Block));
            fp8_load<CG>(st, &tmap_a, (int32_t)(kc * kFp8Block), arow, bar);
            for (uint32_t b = 0; b < boxes; b++)
              fp8_load<CG>(st + A_BYTES + b * W_BOX * kFp8Block, &tmap_w, (int32_t)(kc * kFp8Block),
                           wrow + (int32_t)(b * W_BOX), bar);
          }
        }
        if (!ok && rank == 0)  // the copies in flight land before this CTA's shared memory goes
          for (uint32_t j = it > C::S ? it - C::S : 0u; j < it; j++) mbar_wait(&full[j % C::S], (j / C::S) & 1u, args.err);
        // every signal that the pair's first CTA sends to these barriers has come
        if (ok && CG == 2)
          for (uint32_t j = it > C::S ? it - C::S : 0u; j < it; j++)
            if (!wait_or_abort(&empty[j % C::S], (j / C::S) & 1u, args.err, abort_flag)) break;
      }
    } else if (warp == 1 && rank == 0) {
      const uint64_t adesc0 = umma_desc_sw128(smem_u32(smem)), wdesc0 = umma_desc_sw128(smem_u32(smem + A_BYTES));
      uint32_t it = 0;
      bool ok = true;
      for (; walk.more() && ok; walk.next()) {
        const Fp8Tile ti = walk.tile(args, pre, first);
        const uint32_t idesc = umma_idesc_f16_f32(TILE_M, columns(ti.n0));
        for (uint32_t kc = k_lo; kc < k_hi; kc++, it++) {
          const uint32_t s = it % C::S, b = it % C::NB;
          ok = __all_sync(0xffffffffu, wait_or_abort(&acc_empty[b], ((it / C::NB) & 1u) ^ 1u, args.err, abort_flag) &&
                                           wait_or_abort(&full[s], (it / C::S) & 1u, args.err, abort_flag));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t off = (uint64_t)(s * (C::STAGE >> 4));
#pragma unroll
            for (uint32_t k = 0; k < 4; k++)  // 32 k = 32 bytes = 2 descriptor units
              fp8_mma<CG>(tmem_base + b * BN, adesc0 + off + 2u * k, wdesc0 + off + 2u * k, idesc, k != 0);
            fp8_commit<CG>(&empty[s]);
            fp8_commit<CG>(&acc_full[b]);
          }
          __syncwarp();
        }
      }
      if (elect_one()) fp8_commit_own<CG>(drain);
      __syncwarp();
      if (lane == 0) mbar_wait(drain, 0, args.err);
    } else if (warp == 3) {
      const uint32_t nb = fp8_blocks(args.N);
      uint32_t batch = 0;
      bool ok = true;
      for (; walk.more() && ok; walk.next()) {
        const Fp8Tile ti = walk.tile(args, pre, first);
        const uint32_t row = ti.row0 + rank * BM;
        for (uint32_t k0 = k_lo; k0 < k_hi; k0 += BATCH, batch++) {
          const uint32_t sl = batch % SB;
          ok = __all_sync(0xffffffffu, wait_or_abort(&sc_empty[sl], ((batch / SB) & 1u) ^ 1u, args.err, abort_flag));
          if (!ok) break;
          float* dst = reinterpret_cast<float*>(smem + C::OFF_SCALES) + sl * BATCH * C::SCALES;
          for (uint32_t kc = k0; kc < min(k_hi, k0 + BATCH); kc++, dst += C::SCALES) {
            const float* as = args.as + (uint64_t)kc * args.ldas;
            for (uint32_t j = lane; j < BM; j += 32) cp_async_4(dst + j, as + min(row + j, args.M - 1));
            if constexpr (WB == 1) {
              const float* ws = args.ws + (uint64_t)kc * args.ldws;
              for (uint32_t j = lane; j < BN; j += 32) cp_async_4(dst + BM + j, ws + min(ti.n0 + j, args.N - 1));
            } else if (lane < C::W_SCALES) {
              const uint32_t n = min(ti.n0 / kFp8Block + lane, nb - 1);
              cp_async_4(dst + BM + lane, args.ws + ((uint64_t)ti.e * nb + n) * n_kc + kc);
            }
          }
          cp_async_arrive(&sc_full[sl]);
        }
      }
      cp_async_wait_all();
    }
    __syncwarp();
    if (SPLIT && busy) cluster_sync();  // where the adding warps join the sums
  } else {
    regs_inc<REGS_DRAIN>();
    constexpr int PART = (int)C::PART;
    constexpr bool FRAG = WB == 1;
    static_assert(!FRAG || PART >= 64, "fragments of 64 columns");
    const uint32_t q = (uint32_t)(warp & 3), p = (uint32_t)(warp - (int)FIRST_DRAIN) >> 2;
    const uint32_t taddr = tmem_base + ((q * 32u) << 16) + p * PART, mine = rank * BM + q * 32u;
    uint8_t* stages = smem + C::OFF_OUT + (warp - (int)FIRST_DRAIN) * C::OUT_BYTES;
    uint32_t turn = 0;
    const uint32_t empty_addr = CG == 2 ? leader_addr(acc_empty) : smem_u32(acc_empty);
    const float* const scales = reinterpret_cast<const float*>(smem + C::OFF_SCALES);
    __half* const bias = reinterpret_cast<__half*>(smem + C::OFF_BIAS) + (warp - (int)FIRST_DRAIN) * PART;
    uint32_t it = 0, batch = 0;
    bool ok = true;  // after a wait that ran out: no more waits and no output
    for (; walk.more() && ok; walk.next()) {
      const Fp8Tile ti = walk.tile(args, pre, first);
      const uint32_t n = ti.n0 + p * PART;
      uint16_t b16[PART / 32];  // fp16 bias of columns lane, lane + 32, ..: on its way while the tile is summed
      if (args.bias)
#pragma unroll
        for (int j = 0; j < PART / 32; j++)
          b16[j] = ld_u16(&args.bias[(uint64_t)ti.e * args.N + min(n + j * 32 + lane, args.N - 1)]);
      float acc[PART];
#pragma unroll
      for (int j = 0; j < PART; j++) acc[j] = 0.0f;
#pragma unroll 1
      for (uint32_t kc = k_lo; kc < k_hi; kc++, it++) {
        const uint32_t b = it % C::NB, sl = batch % SB, in_batch = (kc - k_lo) % BATCH;
        if (in_batch == 0 && ok) ok = wait_or_abort(&sc_full[sl], (batch / SB) & 1u, args.err, abort_flag);
        const float* sc = scales + (sl * BATCH + in_batch) * C::SCALES;
        float s[4];  // of the thread's row, or its fragments' four
        if constexpr (FRAG) {
#pragma unroll
          for (int j = 0; j < 4; j++) s[j] = sc[q * 32u + j * 8 + (lane >> 2)];
        } else {
          s[0] = sc[q * 32u + lane] * sc[BM + p * PART / 128];
        }
        if (ok) ok = wait_or_abort(&acc_full[b], (it / C::NB) & 1u, args.err, abort_flag);
        __syncwarp();
        tc_fence_after();
        const uint32_t src = taddr + b * BN;
        auto release = [&]() {  // the buffer has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(empty_addr + b * 8);
            else mbar_arrive(&acc_empty[b]);
          }
        };
        // as many columns a load as the registers hold beside the sums: the
        // tensor core stands still while TMEM is read, the longer the more
        // loads there are (32 columns each, one ahead of the adding: 451
        // against 402 us for 128 experts)
        if constexpr (FRAG) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
            float r[PART / 2];
            fp8_ld_frag<PART / 2>(src + ((uint32_t)half << 20), r);
            if (half == 1) release();
            float* to = &acc[half * (PART / 2)];
#pragma unroll
            for (int g = 0; g < PART / 8; g++) {
              const float2 w = *reinterpret_cast<const float2*>(sc + BM + p * PART + g * 8 + (lane & 3) * 2);
              to[4 * g] = fmaf(r[4 * g], w.x * s[2 * half], to[4 * g]);
              to[4 * g + 1] = fmaf(r[4 * g + 1], w.y * s[2 * half], to[4 * g + 1]);
              to[4 * g + 2] = fmaf(r[4 * g + 2], w.x * s[2 * half + 1], to[4 * g + 2]);
              to[4 * g + 3] = fmaf(r[4 * g + 3], w.y * s[2 * half + 1], to[4 * g + 3]);
            }
          }
        } else {
          constexpr int LD = PART < 64 ? PART : 64;
#pragma unroll
          for (int c = 0; c < PART; c += LD) {
            float r[LD];
            fp8_ld<LD>(src + c, r);
            if (c + LD == PART) release();
#pragma unroll
            for (int j = 0; j < LD; j++) acc[c + j] = fmaf(r[j], s[0], acc[c + j]);
          }
        }
        if (in_batch == BATCH - 1 || kc + 1 == k_hi) {  // the batch's scales have been read
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_empty[sl]);
          batch++;
        }
      }
      if constexpr (SPLIT) {
        // the only tile of this CTA: its operands' shared memory is free now
        if constexpr (FRAG) {
#pragma unroll
          for (int i = 0; i < PART / 2; i++) {  // pairs: half, 8 columns, upper or lower 8 rows
            const uint32_t r = q * 32u + i / (PART / 4) * 16 + (i & 1) * 8 + (lane >> 2);
            const uint32_t col = p * PART + i / 2 % (PART / 8) * 8 + (lane & 3) * 2;
            float* dst = reinterpret_cast<float*>(smem) + (r * (BN / 4) + fp8_swizzle<BN>(col / 4, r)) * 4 + col % 4;
            *reinterpret_cast<float2*>(dst) = make_float2(acc[2 * i], acc[2 * i + 1]);
          }
        } else {
          float4* row = reinterpret_cast<float4*>(smem) + (q * 32u + lane) * (BN / 4);
#pragma unroll
          for (int j = 0; j < PART / 4; j++)
            row[fp8_swizzle<BN>(p * (PART / 4) + j, lane)] =
                make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
        }
        cluster_sync();
        if (ok) fp8_join<BN, OT>(args, ti, smem, part, parts);
        break;
      }
      if (args.bias) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < PART / 32; j++) bias[j * 32 + lane] = __ushort_as_half(b16[j]);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < PART; j += 2) {
          // columns j, j + 1 of the row; of fragments, pair j / 2: half, 8 columns, upper or lower 8 rows
          const int col = FRAG ? j / 4 % (PART / 8) * 8 + (lane & 3) * 2 : j;
          const float2 b = __half22float2(*reinterpret_cast<const __half2*>(bias + col));
          acc[j] += b.x;
          acc[j + 1] += b.y;
        }
      }
      if (__all_sync(0xffffffffu, ok))
        fp8_write<OT, PART, FRAG>(args, &tmap_o, tma_out, stages, turn, ti.row0 + mine, ti.row_end, n, acc);
    }
    if (lane == 0) bulk_wait();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2 || SPLIT) cluster_sync();  // no CTA leaves while the other may signal it or read its operands
  if (warp == 2) {
    tc_fence_after();
    fp8_tmem_dealloc<CG>(tmem_base, TMEM_COLS);
  }
}

template <int CG, int BN, int WB, int OT, bool SPLIT>
static cudaError_t launch_gemm(const CUtensorMap& ta, const CUtensorMap& tw, const Fp8MmArgs& a, uint64_t m_tiles,
                               uint32_t split, cudaStream_t st) {
  using C = f8::Cfg<CG, BN, WB>;
  auto* kernel = fp8_gemm_kernel<CG, BN, WB, OT, SPLIT>;
  static std::atomic<uint64_t> attr_done{0};
  constexpr uint32_t smem = C::SMEM;
  if (cudaError_t e = smem_attr_per_device(kernel, (int)smem, attr_done); e != cudaSuccess) return e;
  const uint32_t n_tiles = (a.N + BN - 1) / BN, cluster = CG * split;
  const uint64_t tiles = m_tiles * n_tiles;
  const uint32_t grid = cluster * (uint32_t)(SPLIT ? tiles : std::min<uint64_t>(tiles, (uint64_t)num_sms() / CG));
  // out as 16-byte pieces of rows that can be mapped: the tensor map's box is a
  // warp's 32 rows of up to 128 bytes
  constexpr uint32_t size = sizeof(typename Fp8Type<OT>::T), bytes = std::min<uint32_t>(C::PART * size, 128);
  CUtensorMap to = ta;
  const uint32_t tma_out = !SPLIT && make_out_tmap(&to, a.out, OT, a.M, a.N, a.ldo, bytes / size, 32) ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(f8::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, ta, tw, to, a, n_tiles, tma_out, split);
}

template <int CG, int BN, bool SPLIT>
static cudaError_t launch_gemm_out(const CUtensorMap& ta, const CUtensorMap& tw, const Fp8MmArgs& a, uint64_t m_tiles,
                                   uint32_t split, cudaStream_t st) {
  if constexpr (BN >= 128) {
    if (a.w_block == 1) {
      if (a.out_dtype == TS_DTYPE_F16) return launch_gemm<CG, BN, 1, TS_DTYPE_F16, SPLIT>(ta, tw, a, m_tiles, split, st);
      if (a.out_dtype == TS_DTYPE_BF16) return launch_gemm<CG, BN, 1, TS_DTYPE_BF16, SPLIT>(ta, tw, a, m_tiles, split, st);
      return launch_gemm<CG, BN, 1, TS_DTYPE_F32, SPLIT>(ta, tw, a, m_tiles, split, st);
    }
  }
  if (a.out_dtype == TS_DTYPE_F16) return launch_gemm<CG, BN, 128, TS_DTYPE_F16, SPLIT>(ta, tw, a, m_tiles, split, st);
  if (a.out_dtype == TS_DTYPE_BF16) return launch_gemm<CG, BN, 128, TS_DTYPE_BF16, SPLIT>(ta, tw, a, m_tiles, split, st);
  return launch_gemm<CG, BN, 128, TS_DTYPE_F32, SPLIT>(ta, tw, a, m_tiles, split, st);
}

// K = 0: bias or zero (+ what out holds) on the rows that a segment covers.
constexpr uint32_t kFp8EmptyBlocks = 4096;
// a block's step past the last row stays in 32 bits
static_assert(kFp8MaxSize <= 0xffffffffu - kFp8EmptyBlocks, "rows of an empty sum");
template <int OT>
__global__ void __launch_bounds__(256) fp8_empty_sum_kernel(const Fp8MmArgs a) {
  using D = Fp8Type<OT>;
  for (uint32_t e = 0; e < a.E; e++) {
    const uint32_t lo = a.seg ? (uint32_t)min(max(a.seg[e], 0), (int)a.M) : 0;
    const uint32_t hi = a.seg ? (uint32_t)min(max(a.seg[e + 1], 0), (int)a.M) : a.M;
    for (uint32_t m = lo + blockIdx.x; m < hi; m += gridDim.x)
      for (uint32_t n = threadIdx.x; n < a.N; n += 256) {
        auto* o = reinterpret_cast<typename D::T*>(a.out) + (uint64_t)m * a.ldo + n;
        float v = a.bias ? __half2float(reinterpret_cast<const __half*>(a.bias)[(uint64_t)e * a.N + n]) : 0.0f;
        if (a.accumulate) v += D::up(*o);
        *o = D::down(v);
      }
  }
}

// Tiles of bm rows: exact without segments; with them, an upper bound of what
// M rows in E segments can make.
static uint64_t fp8_m_tiles(const Fp8MmArgs& a, uint32_t bm) {
  return a.seg ? a.M / bm + std::min(a.E, a.M) : ((uint64_t)a.M + bm - 1) / bm;
}

// The form with the shortest estimate: rounds of tiles over the SMs, each
// `chunk` us for 128 of k (w_block 128, 1) and `tile` for the rest; the CTAs
// of a split do not outlive their tile, so a second round costs them a start.
// Measured, us a call repeated on the same inputs, [pairs, 128, 64, 128 / 2,
// 128 / 4] at w_block 128:
//   8192 x 8192 x 8192   [546, 726, 1228, -, -]   1024 x 1024 x 8192  [40, 29, 27, 21, 27]
//   2048 x 2048 x 2048   [16, 19, 28, -, -]       128 x 4096 x 4096   [22, 16, 15, 14, 10]
//   512 x 640 x 640      [8.7, 6.8, 5.8, -, -]
// and 1280 x 640 x 16384 at w_block 1 [117, 80, -, 47, 53].
struct Fp8Tiling {
  Fp8Form form;
  uint32_t cg, bn, split;
  double chunk[2], tile;
};
static constexpr Fp8Tiling kFp8Tilings[] = {
    {Fp8Form::pairs, 2, 256, 1, {0.60, 0.92}, 1.1},   {Fp8Form::wide, 1, 128, 1, {0.40, 0.60}, 1.0},
    {Fp8Form::narrow, 1, 64, 1, {0.35, 0}, 0.6},      {Fp8Form::split2, 1, 128, 2, {0.40, 0.60}, 3.5},
    {Fp8Form::split4, 1, 128, 4, {0.40, 0.60}, 3.5},  {Fp8Form::split8, 1, 128, 8, {0.40, 0.60}, 3.5}};

static const Fp8Tiling* fp8_tiling(const Fp8MmArgs& a, uint64_t sms) {
  const uint64_t n_kc = fp8_blocks(a.K);
  const Fp8Tiling* best = nullptr;
  double least = 0.0;
  for (const Fp8Tiling& f : kFp8Tilings) {
    if (f.split > n_kc || (f.bn < 128 && a.w_block == 1)) continue;
    const uint64_t tiles = fp8_m_tiles(a, f.cg * f8::BM) * ((a.N + f.bn - 1) / f.bn), at_once = sms / (f.cg * f.split);
    const uint64_t rounds = (tiles + at_once - 1) / at_once, chunks = (n_kc + f.split - 1) / f.split;
    const double us = (double)rounds * ((double)chunks * f.chunk[a.w_block == 1] + f.tile) +
                      (f.split > 1 ? (double)(rounds - 1) * 3.5 : 0.0);
    if (!best || us < least) best = &f, least = us;
  }
  return best;
}

Fp8Form fp8_matmul_form(const Fp8MmArgs& a, uint32_t sms) {
  if (a.K == 0) return Fp8Form::empty;
  if (a.M <= kFp8MatvecRows && a.w_block != 1 && !a.seg) return Fp8Form::matvec;
  return fp8_tiling(a, sms)->form;
}

cudaError_t launch_fp8_matmul(const Fp8MmArgs& a, cudaStream_t st) {
  const Fp8Form form = fp8_matmul_form(a, (uint32_t)num_sms());
  if (form == Fp8Form::empty) {
    const uint32_t grid = std::min(a.M, kFp8EmptyBlocks);
    if (a.out_dtype == TS_DTYPE_F16) fp8_empty_sum_kernel<TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
    else if (a.out_dtype == TS_DTYPE_BF16) fp8_empty_sum_kernel<TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
    else fp8_empty_sum_kernel<TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
  }
  if (form == Fp8Form::matvec) {
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
  switch (form) {
    case Fp8Form::pairs: return launch_gemm_out<2, 256, false>(ta, tw, a, fp8_m_tiles(a, 2 * f8::BM), 1, st);
    case Fp8Form::wide: return launch_gemm_out<1, 128, false>(ta, tw, a, fp8_m_tiles(a, f8::BM), 1, st);
    case Fp8Form::narrow: return launch_gemm_out<1, 64, false>(ta, tw, a, fp8_m_tiles(a, f8::BM), 1, st);
    case Fp8Form::split2: return launch_gemm_out<1, 128, true>(ta, tw, a, fp8_m_tiles(a, f8::BM), 2, st);
    case Fp8Form::split4: return launch_gemm_out<1, 128, true>(ta, tw, a, fp8_m_tiles(a, f8::BM), 4, st);
    default: return launch_gemm_out<1, 128, true>(ta, tw, a, fp8_m_tiles(a, f8::BM), 8, st);
  }
}

}  // namespace ts

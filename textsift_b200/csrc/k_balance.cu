// k_balance.cu — the router's balance loss, per-expert counts and gradient
// over packed documents (formulas: ts_cuda_op_router_balance in the header).
//
// The gradient needs every count of its document but no probability of other
// tokens, so counts are taken first (they read T k indices only) and one pass
// over the logits then gives the probabilities' sums and the gradient: each
// logit is read once and each gradient written once, which is what bounds it.
//
// Probabilities are summed across blocks as integers, which do not depend on
// the order of the atomics: whole units of 2^-40 in one 64-bit word and the
// rest in units of 2^-80 in another, so that 2^23 tokens (the most that a call
// takes) add up to 2^63 in either, and a term's rounding error is 2^-81, that
// of an f32 as small as 2^-57.  An f32 of 2^-16 or more has no such rest, and
// words that would get nothing are not touched.  Inside a block they are f32
// sums of at most MAX_RUN tokens a lane in a fixed order.
//
// Large calls run as four launches (clear, count, tokens, loss), small ones
// as one block that keeps counts and sums in shared memory: there the chain
// of launches and of global round trips is all that costs.  65,536 x 128 f32
// over 44 documents takes 28.2 us (clear 2, count 6, tokens 19, loss 6, partly
// at once; 10.4 us at the copy's rate), 80 x 128 7.0 to 7.5 us a call, the host's
// time for one (17 us as five launches).
#include "ts_fp8.cuh"
#include "ts_kernels.h"

#include <algorithm>

namespace ts {

namespace bal {
constexpr uint32_t THREADS = 256, WARPS = 8;
constexpr uint32_t COUNT_TOKENS = 256;  // tokens of a counting tile
constexpr uint32_t COUNT_AHEAD = 4;     // of its routes, those a thread loads at once
constexpr uint32_t MAX_RUN = 16;        // most tokens a lane group takes in a row
constexpr uint32_t SEQ_SMEM = 1024;     // document offsets that a block keeps in shared memory
constexpr uint32_t MAX_LOSS_BLOCKS = 256;
constexpr float UNIT = 1099511627776.0f;  // 2^40
constexpr float DIGIT = 1048576.0f;       // 2^20
// the one-block form
constexpr uint32_t ONE_THREADS = 1024, ONE_TABLE = 4096, ONE_TOKENS = 1024;
}  // namespace bal

static uint32_t balance_loss_blocks(uint32_t S, uint32_t E) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(bal::MAX_LOSS_BLOCKS, (uint64_t)S * E / bal::THREADS));
}

// Work area: sums u64 [2][S][E] (units of 2^-40, of 2^-80), partial losses f64
// [blocks], tokens i32 [S], poisoned i32 [S], then a ticket.
struct BalanceWork {
  unsigned long long *sum, *rest;
  double* part;
  int* tokens;
  int* bad;
  unsigned* ticket;
};
__device__ __forceinline__ BalanceWork balance_work(const BalanceArgs& a) {
  BalanceWork w;
  w.sum = static_cast<unsigned long long*>(a.work);
  w.rest = w.sum + (uint64_t)a.S * a.E;
  w.part = reinterpret_cast<double*>(w.rest + (uint64_t)a.S * a.E);
  w.tokens = reinterpret_cast<int*>(w.part + a.loss_blocks);
  w.bad = w.tokens + a.S;
  w.ticket = reinterpret_cast<unsigned*>(w.bad + a.S);
  return w;
}
size_t balance_work_bytes(uint32_t S, uint32_t E) {
  return (size_t)S * E * 16 + balance_loss_blocks(S, E) * 8 + (size_t)S * 8 + 4;
}

// Adds v >= 0.  Every step but the last rounding is exact: from 2^24 units of
// 2^-40 on v is a whole number of them, below that its whole units fit 32 bits
// and an f32.
__device__ __forceinline__ void balance_add(const BalanceWork& w, uint64_t i, float v) {
  const float u = v * bal::UNIT;
  if (u >= 16777216.0f) {
    atomicAdd(&w.sum[i], __float2ull_rn(u));
  } else if (u > 0.0f) {
    const uint32_t whole = __float2uint_rd(u);
    const unsigned long long rest = __float2ull_rn((u - (float)whole) * bal::UNIT);
    if (whole) atomicAdd(&w.sum[i], (unsigned long long)whole);
    if (rest) atomicAdd(&w.rest[i], rest);
  }
}

__device__ __forceinline__ bool balance_token(const BalanceArgs& a, uint32_t t) { return !a.mask || __ldg(&a.mask[t]); }

// Document offsets as a block sees them: in shared memory when there are few.
struct BalanceSeq {
  const int* at;  // null: one document of all tokens
  uint32_t S;
  // The document of token t, or -1 outside [seq[0], seq[S]).
  __device__ __forceinline__ int doc(uint32_t t) const {
    if (!at) return 0;
    if ((int)t < at[0] || (int)t >= at[S]) return -1;
    uint32_t lo = 0, hi = S;  // at[lo] <= t < at[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (at[mid] <= (int)t) lo = mid;
      else hi = mid;
    }
    return (int)lo;
  }
  __device__ __forceinline__ uint32_t end(int s) const { return at ? (uint32_t)max(at[s + 1], 0) : 0xffffffffu; }
};
// Copies the offsets into `room` where they fit; the caller synchronizes.
__device__ __forceinline__ BalanceSeq balance_seq(const BalanceArgs& a, int* room, uint32_t size) {
  BalanceSeq q{a.seq, a.S};
  if (a.seq && a.S < size) {
    for (uint32_t i = threadIdx.x; i <= a.S; i += blockDim.x) room[i] = a.seq[i];
    q.at = room;
  }
  return q;
}

// Documents with tokens, by the whole block.
__device__ __forceinline__ int balance_docs(const BalanceArgs& a, const int* tokens) {
  int docs = 0;
  for (uint32_t s0 = 0; s0 < a.S; s0 += blockDim.x)
    docs += __syncthreads_count(s0 + threadIdx.x < a.S && __ldcg(&tokens[min(s0 + threadIdx.x, a.S - 1)]) > 0);
  return docs;
}

// True in every thread of the block that is the last of nb to come here; what
// the others wrote before is then visible to it.
__device__ __forceinline__ bool balance_last(unsigned* ticket, uint32_t nb) {
  __shared__ unsigned got;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) got = atomicAdd(ticket, 1u);
  __syncthreads();
  __threadfence();
  return got == nb - 1;
}

// Each of these kernels waits for the work before it and only then lets the
// next one start, so that a kernel of the chain may read the caller's inputs
// (though not what the chain writes) before its own wait.
__global__ void __launch_bounds__(bal::THREADS) balance_clear_kernel(const BalanceArgs a) {
  pdl_wait();
  pdl_trigger();
  const BalanceWork w = balance_work(a);
  const uint64_t step = (uint64_t)gridDim.x * bal::THREADS;
  for (uint64_t i = (uint64_t)blockIdx.x * bal::THREADS + threadIdx.x; i < (uint64_t)a.S * a.E; i += step) {
    w.sum[i] = w.rest[i] = 0;
    a.counts[i] = 0;
  }
  for (uint64_t i = (uint64_t)blockIdx.x * bal::THREADS + threadIdx.x; i < 2ull * a.S + 1; i += step) w.tokens[i] = 0;
}

// Counts of a tile of 256 tokens: through shared memory where the tile lies in
// one document, straight to the document's row where it does not.
__global__ void __launch_bounds__(bal::THREADS) balance_count_kernel(const BalanceArgs a) {
  using namespace bal;
  __shared__ int hist[kBalanceMaxExperts];
  __shared__ int doc[COUNT_TOKENS];
  __shared__ int room[SEQ_SMEM];
  __shared__ int top[WARPS];
  const BalanceWork w = balance_work(a);
  const uint32_t t0 = blockIdx.x * COUNT_TOKENS, t = t0 + threadIdx.x, n = min(COUNT_TOKENS, a.T - t0);
  // every input is on its way before the first is waited for
  int route[COUNT_AHEAD];
#pragma unroll
  for (uint32_t j = 0; j < COUNT_AHEAD; j++) {
    const uint32_t r = threadIdx.x + j * THREADS;
    route[j] = r < n * a.k ? __ldg(&a.idx[(uint64_t)t0 * a.k + r]) : -1;
  }
  const bool token = t < a.T && balance_token(a, t);
  const BalanceSeq q = balance_seq(a, room, SEQ_SMEM);
  __syncthreads();
  const int s = token ? q.doc(t) : -1;
  doc[threadIdx.x] = s;
  for (uint32_t e = threadIdx.x; e < a.E; e += THREADS) hist[e] = 0;
  // the tile's one document: the largest of all, equal to every one that is not padding
  int one = s;
#pragma unroll
  for (int d = 16; d; d >>= 1) one = max(one, __shfl_xor_sync(0xffffffffu, one, d));
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = one;
  __syncthreads();
  for (uint32_t i = 0; i < WARPS; i++) one = max(one, top[i]);
  const bool single = __syncthreads_and(s < 0 || s == one);
  const int live = __syncthreads_count(s >= 0);
  pdl_wait();
  pdl_trigger();
  if (live) {
    if (single) {
      if (threadIdx.x == 0) atomicAdd(&w.tokens[one], live);
    } else if (s >= 0) {
      atomicAdd(&w.tokens[s], 1);
    }
    auto count = [&](uint32_t r, int e) {
      if (e < 0 || e >= (int)a.E) return;
      const int d = doc[r / a.k];
      if (d < 0) return;
      if (single) atomicAdd(&hist[e], 1);
      else atomicAdd(&a.counts[(uint64_t)d * a.E + e], 1);
    };
#pragma unroll
    for (uint32_t j = 0; j < COUNT_AHEAD; j++) count(threadIdx.x + j * THREADS, route[j]);
    for (uint32_t r = threadIdx.x + COUNT_AHEAD * THREADS; r < n * a.k; r += THREADS)
      count(r, __ldg(&a.idx[(uint64_t)t0 * a.k + r]));
    __syncthreads();
    if (single)
      for (uint32_t e = threadIdx.x; e < a.E; e += THREADS)
        if (hist[e]) atomicAdd(&a.counts[(uint64_t)one * a.E + e], hist[e]);
  }
}

// A document's average count.
__device__ __forceinline__ int balance_ref(const BalanceArgs& a, int tokens) {
  return (int)((long long)tokens * a.k / a.E);
}

// A token's logits in L lanes, V each, in pieces of 16 bytes: piece j of lane
// l is the token's (j L + l)-th.
template <int DT, int L, int V>
struct BalanceToken {
  using D = Fp8Type<DT>;
  using T = typename D::T;
  static constexpr int PER = 16 / (int)sizeof(T), GROUPS = 32 / L;
  static_assert(V % PER == 0, "whole pieces");
  float z[V];  // logits, then e^(logit - largest)
  // the gradient is z * slope * (count - mean), slope = coef / sum; slope is 0
  // for padding and for a row with nothing open, NaN for one that holds a NaN
  // or +inf
  float slope, mean;

  static __device__ __forceinline__ uint32_t lane() { return threadIdx.x % L; }
  static __device__ __forceinline__ uint32_t group() { return (threadIdx.x & 31) / L; }
  static __device__ __forceinline__ uint32_t mask() {
    return L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << (group() * L);
  }
  static __device__ __forceinline__ uint32_t expert(int j) {
    return (uint32_t)((j / PER * L + (int)lane()) * PER + j % PER);
  }
  // `whole`: E = L V and rows start at multiples of 16 bytes
  __device__ __forceinline__ void load(const BalanceArgs& a, uint32_t t, bool whole) {
    const T* x = static_cast<const T*>(a.logits) + t * a.ldl;
    if (whole) {
      const uint4* src = reinterpret_cast<const uint4*>(x) + lane();
#pragma unroll
      for (int j = 0; j < V / PER; j++) {
        const uint4 raw = __ldg(src + j * L);
#pragma unroll
        for (int i = 0; i < PER; i++) z[j * PER + i] = D::up(reinterpret_cast<const T*>(&raw)[i]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) z[j] = expert(j) < a.E ? D::up(x[expert(j)]) : -__int_as_float(0x7f800000);
    }
  }
  __device__ __forceinline__ void nothing() {
    slope = mean = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) z[j] = 0.0f;
  }
  // The exponentials and the gradient's terms of a token; adds its
  // probabilities to psum.  cnt are the counts less their document's average,
  // so that count - mean loses no more than the counts' spread to rounding.
  // e^x is 2^(x log2 e) on the special-function unit, x <= 0 the difference to
  // the largest logit: off by 2^-22 of itself and 2^-24 |x| log2 e, far below
  // what the same errors in sum and mean leave (expf: 29.3 against 27.9 us at
  // 65,536 x 128, the gradient's error against 64 bits the same).
  __device__ __forceinline__ void softmax(const float (&cnt)[V], float (&psum)[V], float coef, int* bad) {
    const float inf = __int_as_float(0x7f800000);
    float m = -inf, sum = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) m = fmaxf(m, z[j]);
#pragma unroll
    for (int d = L / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(mask(), m, d));
    bool odd = false;
    if (!(m > -inf && m < inf)) {  // +inf, or nothing but -inf and NaN
#pragma unroll
      for (int j = 0; j < V; j++) odd |= !(z[j] < inf);
      odd = __any_sync(mask(), odd);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) {
        z[j] = ex2_approx((z[j] - m) * 1.4426950408889634f);
        sum += z[j];
        dot = fmaf(z[j], cnt[j], dot);
      }
#pragma unroll
      for (int d = L / 2; d; d >>= 1) {
        sum += __shfl_xor_sync(mask(), sum, d);
        dot += __shfl_xor_sync(mask(), dot, d);
      }
      odd = !(sum == sum);  // a NaN among finite logits
    }
    if (sum > 0.0f) {
      const float inv = 1.0f / sum;
      slope = coef * inv;
      mean = dot * inv;
#pragma unroll
      for (int j = 0; j < V; j++) psum[j] = fmaf(z[j], inv, psum[j]);
    } else {
      nothing();
      if (odd) {
        slope = __int_as_float(0x7fc00000);
        if (lane() == 0) *bad = 1;
      }
    }
  }
  __device__ __forceinline__ void write(const BalanceArgs& a, uint32_t t, const float (&cnt)[V], bool whole) const {
    T* g = static_cast<T*>(a.grad) + t * a.ldg;
    __align__(16) T out[V];
#pragma unroll
    for (int j = 0; j < V; j++) out[j] = D::down(z[j] * slope * (cnt[j] - mean));
    if (whole) {
      uint4* dst = reinterpret_cast<uint4*>(g) + lane();
#pragma unroll
      for (int j = 0; j < V / PER; j++) dst[j * L] = *reinterpret_cast<const uint4*>(&out[j * PER]);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (expert(j) < a.E) g[expert(j)] = out[j];
    }
  }
  static __device__ __forceinline__ bool whole_in(const BalanceArgs& a) {
    return a.E == L * V && !(reinterpret_cast<uintptr_t>(a.logits) & 15u) && a.ldl * sizeof(T) % 16 == 0;
  }
  static __device__ __forceinline__ bool whole_out(const BalanceArgs& a) {
    return a.E == L * V && !(reinterpret_cast<uintptr_t>(a.grad) & 15u) && a.ldg * sizeof(T) % 16 == 0;
  }
  // grad_scale alpha E / k for S' documents; over n twice for one of n tokens
  static __device__ __forceinline__ float factor(const BalanceArgs& a, int docs) {
    return a.grad_scale * a.alpha * (float)a.E / (float)a.k / (float)max(docs, 1);
  }
};

// Blocks of the kernel below that fit an SM (registers).
__host__ __device__ constexpr int bal_blocks(int v) { return v <= 8 ? 4 : 1; }

// A warp takes 32 / L tokens at once and `run` in a row for each lane group,
// the next token's logits loaded while one is worked on; the group's document,
// its counts and the sums of its probabilities stay in registers until the
// document ends.
template <int DT, int L, int V>
__global__ void __launch_bounds__(bal::THREADS, bal_blocks(V)) balance_tokens_kernel(const BalanceArgs a, uint32_t run) {
  using namespace bal;
  using K = BalanceToken<DT, L, V>;
  __shared__ float red[WARPS][L * V];
  __shared__ int red_doc[WARPS];
  __shared__ int room[SEQ_SMEM];
  const BalanceWork w = balance_work(a);
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool whole_in = K::whole_in(a), whole_out = K::whole_out(a);
  const uint32_t first_t = (blockIdx.x * WARPS + warp) * run * K::GROUPS + K::group();
  K next;
  bool next_token = false;
  if (first_t < a.T) {
    next.load(a, first_t, whole_in);
    next_token = balance_token(a, first_t);
  }
  const BalanceSeq q = balance_seq(a, room, SEQ_SMEM);
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const float all = K::factor(a, balance_docs(a, w.tokens));
  float cnt[V], psum[V], coef = 0.0f;
  int held = -1;      // the document that cnt and psum belong to
  int now = -1;       // the document of the group's tokens
  uint32_t end = 0;   // where that is to be looked up again
  auto flush = [&]() {
    if (held < 0) return;
#pragma unroll
    for (int j = 0; j < V; j++)
      balance_add(w, (uint64_t)held * a.E + K::expert(j), psum[j]);
  };
#pragma unroll
  for (int j = 0; j < V; j++) cnt[j] = psum[j] = 0.0f;
  for (uint32_t i = 0; i < run; i++) {
    const uint32_t t = first_t + i * K::GROUPS;
    if (t >= a.T) break;
    K tok = next;
    const int s = next_token ? (t >= end ? q.doc(t) : now) : -1;
    if (i + 1 < run && t + K::GROUPS < a.T) {
      next.load(a, t + K::GROUPS, whole_in);
      next_token = balance_token(a, t + K::GROUPS);
    }
    if (s >= 0) {
      if (s != now) {
        now = s;
        end = q.end(s);
      }
      if (s != held) {
        flush();
        held = s;
        const int tokens = __ldcg(&w.tokens[s]), ref = balance_ref(a, tokens);
        coef = all / (float)tokens / (float)tokens;
#pragma unroll
        for (int j = 0; j < V; j++) {
          psum[j] = 0.0f;
          cnt[j] = K::expert(j) < a.E ? (float)(__ldcg(&a.counts[(uint64_t)s * a.E + K::expert(j)]) - ref) : 0.0f;
        }
      }
      tok.softmax(cnt, psum, coef, &w.bad[s]);
    } else {
      tok.nothing();
    }
    if (a.grad) tok.write(a, t, cnt, whole_out);
  }
  // one row of sums a warp where all its groups hold the same document
  const int first = __shfl_sync(0xffffffffu, held, 0);
  const bool same = __all_sync(0xffffffffu, held == first || held < 0) && first >= 0;
  if (same) {
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int d = L; d < 32; d <<= 1) psum[j] += __shfl_xor_sync(0xffffffffu, psum[j], d);
      if (K::group() == 0) red[warp][K::expert(j)] = psum[j];
    }
  } else {
    flush();
  }
  if (lane == 0) red_doc[warp] = same ? first : -1;
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < a.E; e += THREADS) {
    float sum = 0.0f;
    for (uint32_t i = 0; i < WARPS; i++) {
      const int s = red_doc[i];
      if (s >= 0) sum += red[i][e];
      if (s >= 0 && (i + 1 == WARPS || red_doc[i + 1] != s)) {
        balance_add(w, (uint64_t)s * a.E + e, sum);
        sum = 0.0f;
      }
    }
  }
}

// A document's mean probability of an expert, from its sum in units of 2^-40
// and 2^-80, and the entry's part of the loss.
__device__ __forceinline__ double balance_entry(const BalanceArgs& a, uint64_t i, unsigned long long sum,
                                                unsigned long long rest, int n, bool bad, int count) {
  constexpr double unit = 1.0 / (double)bal::UNIT;
  double p = n > 0 ? ((double)sum + (double)rest * unit) * unit / n : 0.0;
  if (bad) p = __longlong_as_double(0x7ff8000000000000ll);
  a.prob[i] = (float)p;
  return n > 0 ? p * count * ((double)a.E / ((double)a.k * n)) : 0.0;
}

template <uint32_t WARPS>
__device__ __forceinline__ double balance_block_sum(double v) {
  __shared__ double warp_sum[WARPS];
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (uint32_t i = 0; i < WARPS; i++) v += warp_sum[i];
  return v;
}

// Mean probabilities and the loss: a partial sum for each block, added by the last.
__global__ void __launch_bounds__(bal::THREADS) balance_loss_kernel(const BalanceArgs a) {
  using namespace bal;
  pdl_wait();
  pdl_trigger();
  const BalanceWork w = balance_work(a);
  double sum = 0.0;
  for (uint64_t i = (uint64_t)blockIdx.x * THREADS + threadIdx.x; i < (uint64_t)a.S * a.E; i += gridDim.x * THREADS) {
    const uint32_t s = i >> 32 ? (uint32_t)(i / a.E) : (uint32_t)i / a.E;
    sum += balance_entry(a, i, __ldcg(&w.sum[i]), __ldcg(&w.rest[i]), __ldcg(&w.tokens[s]), __ldcg(&w.bad[s]) != 0,
                         __ldcg(&a.counts[i]));
  }
  sum = balance_block_sum<WARPS>(sum);
  if (threadIdx.x == 0) w.part[blockIdx.x] = sum;
  if (balance_last(w.ticket, gridDim.x)) {
    sum = balance_block_sum<WARPS>(threadIdx.x < gridDim.x ? __ldcg(&w.part[threadIdx.x]) : 0.0);
    const int docs = balance_docs(a, w.tokens);
    if (threadIdx.x == 0) *a.loss = (float)(sum * a.alpha / max(docs, 1));
  }
}

// Everything by one block: counts and sums in shared memory, the sums as four
// words of 20 bits each, of 2^-20, 2^-40, 2^-60 and 2^-80 (at most 2^10 tokens:
// all stay below 2^31), whose atomics are native.
struct BalanceOne {
  int seq[bal::ONE_TABLE + 1];
  int tokens[bal::ONE_TABLE], bad[bal::ONE_TABLE];
  int doc[bal::ONE_TOKENS];
  int counts[bal::ONE_TABLE];
  uint32_t sum[4][bal::ONE_TABLE];
};
template <int DT, int L, int V>
__global__ void __launch_bounds__(bal::ONE_THREADS, 1) balance_one_kernel(const BalanceArgs a) {
  using namespace bal;
  using K = BalanceToken<DT, L, V>;
  extern __shared__ __align__(16) uint8_t one_smem[];
  BalanceOne& m = *reinterpret_cast<BalanceOne*>(one_smem);
  pdl_wait();
  pdl_trigger();
  constexpr uint32_t STRIDE = ONE_THREADS / 32 * K::GROUPS;
  const uint32_t first_t = threadIdx.x / L;
  const bool whole_in = K::whole_in(a), whole_out = K::whole_out(a);
  K next;
  if (first_t < a.T) next.load(a, first_t, whole_in);
  const BalanceSeq q = balance_seq(a, m.seq, ONE_TABLE + 1);
  const uint32_t table = a.S * a.E;
  for (uint32_t i = threadIdx.x; i < table; i += ONE_THREADS) m.counts[i] = m.sum[0][i] = m.sum[1][i] = m.sum[2][i] = m.sum[3][i] = 0;
  for (uint32_t i = threadIdx.x; i < a.S; i += ONE_THREADS) m.tokens[i] = m.bad[i] = 0;
  __syncthreads();
  {
    const int s = threadIdx.x < a.T && balance_token(a, threadIdx.x) ? q.doc(threadIdx.x) : -1;
    m.doc[threadIdx.x] = s;
    const uint32_t alike = __match_any_sync(0xffffffffu, s);  // one add for each document of a warp
    if (s >= 0 && (threadIdx.x & 31) == __ffs(alike) - 1) atomicAdd(&m.tokens[s], __popc(alike));
  }
  __syncthreads();
  for (uint32_t r = threadIdx.x; r < a.T * a.k; r += ONE_THREADS) {
    const int d = m.doc[r / a.k], e = __ldg(&a.idx[r]);
    if (d >= 0 && e >= 0 && e < (int)a.E) atomicAdd(&m.counts[d * a.E + e], 1);
  }
  int docs = 0;
  for (uint32_t s0 = 0; s0 < a.S; s0 += ONE_THREADS)
    docs += __syncthreads_count(s0 + threadIdx.x < a.S && m.tokens[min(s0 + threadIdx.x, a.S - 1)] > 0);
  const float all = K::factor(a, docs);
  for (uint32_t t = first_t; t < a.T; t += STRIDE) {
    K tok = next;
    if (t + STRIDE < a.T) next.load(a, t + STRIDE, whole_in);
    const int s = m.doc[t], ref = s >= 0 ? balance_ref(a, m.tokens[s]) : 0;
    float cnt[V], psum[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      psum[j] = 0.0f;
      cnt[j] = s >= 0 && K::expert(j) < a.E ? (float)(m.counts[s * a.E + K::expert(j)] - ref) : 0.0f;
    }
    if (s >= 0) {
      const float n = (float)m.tokens[s];
      tok.softmax(cnt, psum, all / n / n, &m.bad[s]);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const uint32_t at = s * a.E + K::expert(j);
        if (psum[j] >= 1.0f / 65536.0f) {  // a whole number of 2^-40 (digit by digit for all: 7.7 against 7.1 us, 80 x 128)
          const unsigned long long u = __float2ull_rn(psum[j] * UNIT);
          atomicAdd(&m.sum[0][at], (uint32_t)(u >> 20));
          atomicAdd(&m.sum[1][at], (uint32_t)u & 0xfffffu);
        } else if (psum[j] > 0.0f) {
          float u = psum[j] * DIGIT;  // exact digits but for the last one's rounding
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t d = i < 3 ? __float2uint_rd(u) : __float2uint_rn(u);
            if (d) atomicAdd(&m.sum[i][at], d);
            u = (u - (float)d) * DIGIT;
          }
        }
      }
    } else {
      tok.nothing();
    }
    if (a.grad) tok.write(a, t, cnt, whole_out);
  }
  __syncthreads();
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < table; i += ONE_THREADS) {
    const uint32_t s = i / a.E;
    const unsigned long long whole = ((unsigned long long)m.sum[0][i] << 20) + m.sum[1][i];
    const unsigned long long rest = ((unsigned long long)m.sum[2][i] << 20) + m.sum[3][i];
    sum += balance_entry(a, i, whole, rest, m.tokens[s], m.bad[s] != 0, m.counts[i]);
    a.counts[i] = m.counts[i];
  }
  sum = balance_block_sum<ONE_THREADS / 32>(sum);
  if (threadIdx.x == 0) *a.loss = (float)(sum * a.alpha / max(docs, 1));
}

template <int DT, int L, int V>
static cudaError_t launch_balance(const BalanceArgs& a, cudaStream_t st) {
  using namespace bal;
  const uint64_t table = (uint64_t)a.S * a.E;
  if ((uint64_t)a.T * std::max(a.E, 64u) <= kBalanceOneLogits && a.T <= ONE_TOKENS && table <= ONE_TABLE) {
    static std::atomic<uint64_t> attr_done{0};
    if (cudaError_t e = smem_attr_per_device(balance_one_kernel<DT, L, V>, (int)sizeof(BalanceOne), attr_done);
        e != cudaSuccess)
      return e;
    return launch_pdl(balance_one_kernel<DT, L, V>, dim3(1), dim3(ONE_THREADS), sizeof(BalanceOne), st, a);
  }
  const dim3 t(THREADS);
  const uint32_t clear = (uint32_t)std::min<uint64_t>((std::max<uint64_t>(table, 2ull * a.S + 1) + THREADS - 1) / THREADS, 1024);
  cudaError_t e = launch_pdl(balance_clear_kernel, dim3(clear), t, 0, st, a);
  const uint32_t count = (a.T + COUNT_TOKENS - 1) / COUNT_TOKENS;
  if (e == cudaSuccess && count) e = launch_pdl(balance_count_kernel, dim3(count), t, 0, st, a);
  if (e == cudaSuccess && a.T) {
    // runs as long as all blocks that fit the GPU still have one
    const uint32_t at_once = WARPS * (32 / L), wave = (uint32_t)num_sms() * bal_blocks(V) * at_once;
    const uint32_t run = std::min(MAX_RUN, (a.T + wave - 1) / wave), tile = at_once * run;
    e = launch_pdl(balance_tokens_kernel<DT, L, V>, dim3((a.T + tile - 1) / tile), t, 0, st, a, run);
  }
  if (e == cudaSuccess) e = launch_pdl(balance_loss_kernel, dim3(a.loss_blocks), t, 0, st, a);
  return e;
}

// Eight values a lane: sixteen (eight lanes a token, half the instructions) need
// so many registers that fewer blocks fit, 31 against 27 us at 65,536 x 128.
template <int DT>
static cudaError_t launch_balance_experts(const BalanceArgs& a, cudaStream_t st) {
  if (a.E <= 64) return launch_balance<DT, 8, 8>(a, st);
  if (a.E <= 128) return launch_balance<DT, 16, 8>(a, st);
  if (a.E <= 256) return launch_balance<DT, 32, 8>(a, st);
  return launch_balance<DT, 32, 32>(a, st);
}

cudaError_t launch_router_balance(BalanceArgs a, cudaStream_t st) {
  a.loss_blocks = balance_loss_blocks(a.S, a.E);
  if (a.dtype == TS_DTYPE_F16) return launch_balance_experts<TS_DTYPE_F16>(a, st);
  if (a.dtype == TS_DTYPE_BF16) return launch_balance_experts<TS_DTYPE_BF16>(a, st);
  return launch_balance_experts<TS_DTYPE_F32>(a, st);
}

}  // namespace ts

// k_balance.cu — the router's balance loss, per-expert counts and gradient
// over packed documents (formulas: ts_cuda_op_router_balance in the header).
//
// The gradient needs every count of its document but no probability of other
// tokens, so counts are taken first (they read T k indices only) and one pass
// over the logits then gives the probabilities' sums and the gradient: each
// logit is read once and each gradient written once, which is what bounds it.
//
// Probabilities are summed as 64-bit integers in units of 2^-40 across blocks:
// integer sums do not depend on the order of the atomics, 2^23 tokens stay
// below 2^63, and a term's rounding error is 2^-41.  Inside a block they are
// f32 sums of at most 16 tokens a lane in a fixed order.
//
// Four phases (clear, count, tokens, loss), each written for `nb` blocks:
// four launches for large calls, or one cluster of eight blocks with the
// cluster's barrier between phases, where launches cost more than they do.
#include "ts_fp8.cuh"

#include <algorithm>

namespace ts {

namespace bal {
constexpr uint32_t THREADS = 256, WARPS = 8, CLUSTER = 8;
constexpr uint32_t COUNT_TOKENS = 256;  // tokens of a counting tile
constexpr uint32_t RUN = 4;             // tokens a lane group takes in a row
constexpr uint32_t MAX_LOSS_BLOCKS = 128;
constexpr float UNIT = 1099511627776.0f;  // 2^40
}  // namespace bal

static uint32_t balance_loss_blocks(uint32_t S, uint32_t E) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(bal::MAX_LOSS_BLOCKS, (uint64_t)S * E / 1024));
}

// Work area: sums u64 [S][E], partial losses f64 [blocks], tokens i32 [S],
// poisoned i32 [S], then documents with tokens and two tickets.
struct BalanceWork {
  unsigned long long* sum;
  double* part;
  int* tokens;
  int* bad;
  int* docs;
  unsigned* ticket;
};
__device__ __forceinline__ BalanceWork balance_work(const BalanceArgs& a) {
  BalanceWork w;
  w.sum = static_cast<unsigned long long*>(a.work);
  w.part = reinterpret_cast<double*>(w.sum + (uint64_t)a.S * a.E);
  w.tokens = reinterpret_cast<int*>(w.part + a.loss_blocks);
  w.bad = w.tokens + a.S;
  w.docs = w.bad + a.S;
  w.ticket = reinterpret_cast<unsigned*>(w.docs + 1);
  return w;
}
size_t balance_work_bytes(uint32_t S, uint32_t E) {
  return (size_t)S * E * 8 + balance_loss_blocks(S, E) * 8 + (size_t)S * 8 + 12;
}

// The document of token t, or -1: padding, or outside [seq[0], seq[S]).
__device__ __forceinline__ int balance_doc(const BalanceArgs& a, uint32_t t) {
  if (a.mask && !a.mask[t]) return -1;
  if (!a.seq) return 0;
  if ((int)t < a.seq[0] || (int)t >= a.seq[a.S]) return -1;
  uint32_t lo = 0, hi = a.S;  // seq[lo] <= t < seq[hi]
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.seq[mid] <= (int)t) lo = mid;
    else hi = mid;
  }
  return (int)lo;
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

__device__ __forceinline__ void balance_clear(const BalanceArgs& a, uint32_t bid, uint32_t nb) {
  const BalanceWork w = balance_work(a);
  const uint64_t step = (uint64_t)nb * bal::THREADS;
  for (uint64_t i = bid * bal::THREADS + threadIdx.x; i < (uint64_t)a.S * a.E; i += step) {
    w.sum[i] = 0;
    a.counts[i] = 0;
  }
  for (uint64_t i = bid * bal::THREADS + threadIdx.x; i < 2ull * a.S + 3; i += step) w.tokens[i] = 0;
}

// Counts of tiles of 256 tokens: through shared memory where the tile lies in
// one document, straight to the document's row where it does not.  The last
// block counts the documents that have tokens.
__device__ __forceinline__ void balance_count(const BalanceArgs& a, uint32_t bid, uint32_t nb) {
  using namespace bal;
  __shared__ int hist[kBalanceMaxExperts];
  __shared__ int doc[COUNT_TOKENS];
  const BalanceWork w = balance_work(a);
  for (uint32_t t0 = bid * COUNT_TOKENS; t0 < a.T; t0 += nb * COUNT_TOKENS) {
    const uint32_t t = t0 + threadIdx.x, n = min(COUNT_TOKENS, a.T - t0);
    const int s = t < a.T ? balance_doc(a, t) : -1;
    doc[threadIdx.x] = s;
    for (uint32_t e = threadIdx.x; e < a.E; e += THREADS) hist[e] = 0;
    // the tile's one document: the largest of all, equal to every one that is not padding
    int one = s;
#pragma unroll
    for (int d = 16; d; d >>= 1) one = max(one, __shfl_xor_sync(0xffffffffu, one, d));
    __shared__ int top[WARPS];
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = one;
    __syncthreads();
    for (uint32_t i = 0; i < WARPS; i++) one = max(one, top[i]);
    const bool single = __syncthreads_and(s < 0 || s == one);
    const int live = __syncthreads_count(s >= 0);
    if (live) {
      if (single) {
        if (threadIdx.x == 0) atomicAdd(&w.tokens[one], live);
      } else if (s >= 0) {
        atomicAdd(&w.tokens[s], 1);
      }
      for (uint32_t r = threadIdx.x; r < n * a.k; r += THREADS) {
        const int d = doc[r / a.k];
        if (d < 0) continue;
        const int e = a.idx[(uint64_t)t0 * a.k + r];
        if (e < 0 || e >= (int)a.E) continue;
        if (single) atomicAdd(&hist[e], 1);
        else atomicAdd(&a.counts[(uint64_t)d * a.E + e], 1);
      }
      __syncthreads();
      if (single)
        for (uint32_t e = threadIdx.x; e < a.E; e += THREADS)
          if (hist[e]) atomicAdd(&a.counts[(uint64_t)one * a.E + e], hist[e]);
    }
    __syncthreads();
  }
  if (balance_last(&w.ticket[0], nb)) {
    int used = 0;
    for (uint32_t s0 = 0; s0 < a.S; s0 += THREADS)
      used += __syncthreads_count(s0 + threadIdx.x < a.S && __ldcg(&w.tokens[min(s0 + threadIdx.x, a.S - 1)]) > 0);
    if (threadIdx.x == 0) *w.docs = used;
  }
}

// L lanes hold a token's logits, V each, in pieces of 16 bytes: piece j of
// lane l is the token's (j L + l)-th.  A warp takes 32 / L tokens at once and
// RUN in a row for each lane group; the group's document, its counts and the
// sums of its probabilities stay in registers until the document ends.
template <int DT, int L, int V>
__device__ __forceinline__ void balance_tokens(const BalanceArgs& a, uint32_t bid, uint32_t nb) {
  using namespace bal;
  using D = Fp8Type<DT>;
  using T = typename D::T;
  constexpr int PER = 16 / (int)sizeof(T), GROUPS = 32 / L;
  constexpr uint32_t TILE = WARPS * GROUPS * RUN;
  __shared__ float red[WARPS][L * V];
  __shared__ int red_doc[WARPS];
  const BalanceWork w = balance_work(a);
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L, grp = lane / L;
  const uint32_t mask = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << (grp * L);
  const float inf = __int_as_float(0x7f800000);
  const bool vec_in = !(reinterpret_cast<uintptr_t>(a.logits) & 15u) && a.ldl * sizeof(T) % 16 == 0;
  const bool vec_out = !(reinterpret_cast<uintptr_t>(a.grad) & 15u) && a.ldg * sizeof(T) % 16 == 0;
  const float all = a.grad_scale * a.alpha * (float)a.E / (float)a.k / (float)max(__ldcg(w.docs), 1);
  auto expert = [&](int j) { return (uint32_t)((j / PER * L + (int)l) * PER + j % PER); };
  float cnt[V], psum[V];
  for (uint32_t t0 = bid * TILE; t0 < a.T; t0 += nb * TILE) {
    int held = -1;  // the document that cnt and psum belong to
    float coef = 0.0f;
    auto flush = [&]() {
      if (held < 0) return;
#pragma unroll
      for (int j = 0; j < V; j++)
        if (psum[j] > 0.0f) atomicAdd(&w.sum[(uint64_t)held * a.E + expert(j)], __float2ull_rn(psum[j] * UNIT));
    };
#pragma unroll
    for (int j = 0; j < V; j++) psum[j] = 0.0f;
    for (uint32_t i = 0; i < RUN; i++) {
      const uint32_t t = t0 + (warp * RUN + i) * GROUPS + grp;
      if (t >= a.T) break;
      float z[V];
      const T* x = static_cast<const T*>(a.logits) + t * a.ldl;
#pragma unroll
      for (int j = 0; j < V; j += PER) {
        const uint32_t e = expert(j);
        if (vec_in && e + PER <= a.E) {
          const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + e));
#pragma unroll
          for (int i2 = 0; i2 < PER; i2++) z[j + i2] = D::up(reinterpret_cast<const T*>(&raw)[i2]);
        } else {
#pragma unroll
          for (int i2 = 0; i2 < PER; i2++) z[j + i2] = e + i2 < a.E ? D::up(x[e + i2]) : -inf;
        }
      }
      const int s = balance_doc(a, t);
      float scale = 0.0f, mean = 0.0f, fill = 0.0f;
      if (s >= 0) {
        if (s != held) {
          flush();
          held = s;
          const float n = (float)__ldcg(&w.tokens[s]);
          coef = all / n / n;
#pragma unroll
          for (int j = 0; j < V; j++) {
            psum[j] = 0.0f;
            cnt[j] = expert(j) < a.E ? (float)__ldcg(&a.counts[(uint64_t)s * a.E + expert(j)]) : 0.0f;
          }
        }
        float m = -inf;
#pragma unroll
        for (int j = 0; j < V; j++) m = fmaxf(m, z[j]);
#pragma unroll
        for (int d = L / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, d));
        float sum = 0.0f, dot = 0.0f;
        bool odd = false;
        if (!(m > -inf && m < inf)) {  // +inf, or nothing but -inf and NaN
#pragma unroll
          for (int j = 0; j < V; j++) odd |= !(z[j] < inf);
          odd = __any_sync(mask, odd);
        } else {
#pragma unroll
          for (int j = 0; j < V; j++) {
            z[j] = expf(z[j] - m);
            sum += z[j];
            dot = fmaf(z[j], cnt[j], dot);
          }
#pragma unroll
          for (int d = L / 2; d; d >>= 1) {
            sum += __shfl_xor_sync(mask, sum, d);
            dot += __shfl_xor_sync(mask, dot, d);
          }
          odd = !(sum == sum);  // a NaN among finite logits
        }
        if (odd) {
          if (l == 0) w.bad[s] = 1;
          fill = __int_as_float(0x7fc00000);
        } else if (sum > 0.0f) {
          const float inv = 1.0f / sum;
          mean = dot * inv;
          scale = coef;
#pragma unroll
          for (int j = 0; j < V; j++) {
            z[j] *= inv;
            psum[j] += z[j];
          }
        }
      }
      if (!a.grad) continue;
      T* g = static_cast<T*>(a.grad) + t * a.ldg;
#pragma unroll
      for (int j = 0; j < V; j += PER) {
        const uint32_t e = expert(j);
        uint4 raw;
        T* out = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i2 = 0; i2 < PER; i2++)
          out[i2] = D::down(scale != 0.0f ? scale * z[j + i2] * (cnt[j + i2] - mean) : fill);
        if (vec_out && e + PER <= a.E) {
          *reinterpret_cast<uint4*>(g + e) = raw;
        } else {
#pragma unroll
          for (int i2 = 0; i2 < PER; i2++)
            if (e + i2 < a.E) g[e + i2] = out[i2];
        }
      }
    }
    // one row of sums a warp where all its groups hold the same document
    const int first = __shfl_sync(0xffffffffu, held, 0);
    const bool same = __all_sync(0xffffffffu, held == first || held < 0) && first >= 0;
    if (same) {
#pragma unroll
      for (int j = 0; j < V; j++) {
#pragma unroll
        for (int d = L; d < 32; d <<= 1) psum[j] += __shfl_xor_sync(0xffffffffu, psum[j], d);
        if (grp == 0) red[warp][expert(j)] = psum[j];
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
          atomicAdd(&w.sum[(uint64_t)s * a.E + e], __float2ull_rn(sum * UNIT));
          sum = 0.0f;
        }
      }
    }
    __syncthreads();
  }
}

// Mean probabilities and the loss: a partial sum for each block, added by the last.
__device__ __forceinline__ void balance_loss(const BalanceArgs& a, uint32_t bid, uint32_t nb) {
  using namespace bal;
  __shared__ double warp_sum[WARPS];
  const BalanceWork w = balance_work(a);
  auto block_sum = [&](double v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (uint32_t i = 0; i < WARPS; i++) v += warp_sum[i];
    return v;
  };
  double sum = 0.0;
  if (bid < a.loss_blocks) {
    for (uint64_t i = bid * THREADS + threadIdx.x; i < (uint64_t)a.S * a.E; i += a.loss_blocks * THREADS) {
      const uint32_t s = (uint32_t)(i / a.E);
      const int n = __ldcg(&w.tokens[s]);
      double p = n > 0 ? (double)__ldcg(&w.sum[i]) * (1.0 / (double)UNIT) / n : 0.0;
      if (__ldcg(&w.bad[s])) p = __longlong_as_double(0x7ff8000000000000ll);
      a.prob[i] = (float)p;
      if (n > 0) sum += p * __ldcg(&a.counts[i]) * ((double)a.E / ((double)a.k * n));
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) w.part[bid] = sum;
  }
  if (balance_last(&w.ticket[1], nb)) {
    sum = block_sum(threadIdx.x < a.loss_blocks ? __ldcg(&w.part[threadIdx.x]) : 0.0);
    if (threadIdx.x == 0) *a.loss = (float)(sum * a.alpha / max(__ldcg(w.docs), 1));
  }
}

__global__ void __launch_bounds__(bal::THREADS) balance_clear_kernel(const BalanceArgs a) {
  pdl_trigger();
  pdl_wait();
  balance_clear(a, blockIdx.x, gridDim.x);
}
__global__ void __launch_bounds__(bal::THREADS) balance_count_kernel(const BalanceArgs a) {
  pdl_trigger();
  pdl_wait();
  balance_count(a, blockIdx.x, gridDim.x);
}
template <int DT, int L, int V>
__global__ void __launch_bounds__(bal::THREADS) balance_tokens_kernel(const BalanceArgs a) {
  pdl_trigger();
  pdl_wait();
  balance_tokens<DT, L, V>(a, blockIdx.x, gridDim.x);
}
__global__ void __launch_bounds__(bal::THREADS) balance_loss_kernel(const BalanceArgs a) {
  pdl_trigger();
  pdl_wait();
  balance_loss(a, blockIdx.x, gridDim.x);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// All phases by one cluster.
template <int DT, int L, int V>
__global__ void __launch_bounds__(bal::THREADS) balance_cluster_kernel(const BalanceArgs a) {
  pdl_trigger();
  pdl_wait();
  balance_clear(a, blockIdx.x, bal::CLUSTER);
  cluster_sync();
  balance_count(a, blockIdx.x, bal::CLUSTER);
  cluster_sync();
  balance_tokens<DT, L, V>(a, blockIdx.x, bal::CLUSTER);
  cluster_sync();
  balance_loss(a, blockIdx.x, bal::CLUSTER);
}

template <int DT, int L, int V>
static cudaError_t launch_balance(const BalanceArgs& a, cudaStream_t st) {
  using namespace bal;
  const uint64_t table = (uint64_t)a.S * a.E;
  if ((uint64_t)a.T * std::max(a.E, 64u) <= kBalanceClusterLogits && table <= kBalanceClusterLogits / 4) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CLUSTER);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CLUSTER;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, balance_cluster_kernel<DT, L, V>, a);
  }
  constexpr uint32_t TILE = WARPS * (32 / L) * RUN;
  const dim3 t(THREADS);
  const uint32_t clear = (uint32_t)std::min<uint64_t>((std::max<uint64_t>(table, 2ull * a.S + 3) + THREADS - 1) / THREADS, 1024);
  cudaError_t e = launch_pdl(balance_clear_kernel, dim3(clear), t, 0, st, a);
  const uint32_t count = std::max(1u, (a.T + COUNT_TOKENS - 1) / COUNT_TOKENS);
  if (e == cudaSuccess) e = launch_pdl(balance_count_kernel, dim3(count), t, 0, st, a);
  if (e == cudaSuccess && a.T) e = launch_pdl(balance_tokens_kernel<DT, L, V>, dim3((a.T + TILE - 1) / TILE), t, 0, st, a);
  if (e == cudaSuccess) e = launch_pdl(balance_loss_kernel, dim3(a.loss_blocks), t, 0, st, a);
  return e;
}

template <int DT>
static cudaError_t launch_balance_experts(const BalanceArgs& a, cudaStream_t st) {
  if (a.E <= 128) return launch_balance<DT, 8, 16>(a, st);
  if (a.E <= 256) return launch_balance<DT, 16, 16>(a, st);
  if (a.E <= 512) return launch_balance<DT, 32, 16>(a, st);
  return launch_balance<DT, 32, 32>(a, st);
}

cudaError_t launch_router_balance(BalanceArgs a, cudaStream_t st) {
  a.loss_blocks = balance_loss_blocks(a.S, a.E);
  if (a.dtype == TS_DTYPE_F16) return launch_balance_experts<TS_DTYPE_F16>(a, st);
  if (a.dtype == TS_DTYPE_BF16) return launch_balance_experts<TS_DTYPE_BF16>(a, st);
  return launch_balance_experts<TS_DTYPE_F32>(a, st);
}

}  // namespace ts

// k_balance.cu — the router's balance loss, per-expert counts and gradient
// over packed documents (formulas: ts_cuda_op_router_balance in the header).
//
// The gradient needs every count of its document but no probability of other
// tokens, so counts are taken first and one pass over the logits then gives
// the probabilities' sums and the gradient.  Probabilities are summed as
// 64-bit integers in units of 2^-40: integer sums do not depend on the order
// of the atomics, 2^23 tokens stay below 2^63, and a term's rounding error is
// 2^-41 against an average probability of at least 2^-10.
#include "ts_fp8.cuh"

#include <algorithm>

namespace ts {

// Work area: sums u64 [S][E], tokens i32 [S], poisoned i32 [S].
struct BalanceWork {
  unsigned long long* sum;
  int* tokens;
  int* bad;
  __host__ __device__ BalanceWork(void* p, uint32_t S, uint32_t E)
      : sum(static_cast<unsigned long long*>(p)),
        tokens(reinterpret_cast<int*>(sum + (uint64_t)S * E)),
        bad(tokens + S) {}
};
size_t balance_work_bytes(uint32_t S, uint32_t E) { return (size_t)S * E * 8 + (size_t)S * 8; }

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

__global__ void __launch_bounds__(256) balance_count_kernel(const BalanceArgs a) {
  const BalanceWork w(a.work, a.S, a.E);
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.T) return;
  const int s = balance_doc(a, t);
  if (s < 0) return;
  atomicAdd(&w.tokens[s], 1);
  for (uint32_t j = 0; j < a.k; j++) {
    const int e = a.idx[(uint64_t)t * a.k + j];
    if (e >= 0 && e < (int)a.E) atomicAdd(&a.counts[(uint64_t)s * a.E + e], 1);
  }
}

// One warp for each token.
template <int DT>
__global__ void __launch_bounds__(256) balance_token_kernel(const BalanceArgs a) {
  using D = Fp8Type<DT>;
  __shared__ int docs;
  const BalanceWork w(a.work, a.S, a.E);
  if (threadIdx.x == 0) docs = 0;
  __syncthreads();
  for (uint32_t s = threadIdx.x; s < a.S; s += 256)
    if (w.tokens[s] > 0) atomicAdd(&docs, 1);
  __syncthreads();
  const uint32_t t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= a.T) return;
  const int s = balance_doc(a, t);
  const auto* z = reinterpret_cast<const typename D::T*>(a.logits) + t * a.ldl;
  auto* g = reinterpret_cast<typename D::T*>(a.grad) + t * a.ldg;
  if (s < 0) {
    if (a.grad)
      for (uint32_t e = lane; e < a.E; e += 32) g[e] = D::down(0.0f);
    return;
  }
  const float inf = __int_as_float(0x7f800000);
  float mx = -inf;
  bool bad = false;
  for (uint32_t e = lane; e < a.E; e += 32) {
    const float v = D::up(z[e]);
    bad |= !(v < inf);
    mx = fmaxf(mx, v);
  }
  bad = __any_sync(0xffffffffu, bad);
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  if (bad) {
    if (lane == 0) w.bad[s] = 1;
    if (a.grad)
      for (uint32_t e = lane; e < a.E; e += 32) g[e] = D::down(__int_as_float(0x7fc00000));
    return;
  }
  const bool none = mx == -inf;  // no expert is open to this token
  const int* cnt = a.counts + (uint64_t)s * a.E;
  float sum = 0.0f, dot = 0.0f;
  for (uint32_t e = lane; e < a.E; e += 32) {
    const float p = none ? 0.0f : expf(D::up(z[e]) - mx);
    sum += p;
    dot = fmaf(p, (float)cnt[e], dot);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    dot += __shfl_xor_sync(0xffffffffu, dot, d);
  }
  const float inv = none ? 0.0f : 1.0f / sum;
  const float mean = dot * inv, n = (float)w.tokens[s];
  const float c = a.grad_scale * a.alpha * (float)a.E / ((float)a.k * (float)docs * n) / n;
  for (uint32_t e = lane; e < a.E; e += 32) {
    const float p = none ? 0.0f : expf(D::up(z[e]) - mx) * inv;
    atomicAdd(&w.sum[(uint64_t)s * a.E + e], (unsigned long long)__float2ull_rn(p * 1099511627776.0f));
    if (a.grad) g[e] = D::down(c * p * ((float)cnt[e] - mean));
  }
}

// One block: the mean probabilities and the loss.
__global__ void __launch_bounds__(1024) balance_loss_kernel(const BalanceArgs a) {
  __shared__ double part[1024];
  __shared__ int docs;
  const BalanceWork w(a.work, a.S, a.E);
  if (threadIdx.x == 0) docs = 0;
  __syncthreads();
  for (uint32_t s = threadIdx.x; s < a.S; s += 1024)
    if (w.tokens[s] > 0) atomicAdd(&docs, 1);
  double sum = 0.0;
  for (uint64_t i = threadIdx.x; i < (uint64_t)a.S * a.E; i += 1024) {
    const uint32_t s = (uint32_t)(i / a.E);
    const int n = w.tokens[s];
    double p = n > 0 ? (double)w.sum[i] * (1.0 / 1099511627776.0) / n : 0.0;
    if (w.bad[s]) p = __longlong_as_double(0x7ff8000000000000ll);
    a.prob[i] = (float)p;
    if (n > 0) sum += p * a.counts[i] * ((double)a.E / ((double)a.k * n));
  }
  part[threadIdx.x] = sum;
  __syncthreads();
  for (uint32_t d = 512; d; d >>= 1) {
    if (threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) *a.loss = (float)(part[0] * a.alpha / max(docs, 1));
}

cudaError_t launch_router_balance(const BalanceArgs& a, cudaStream_t st) {
  cudaError_t e = cudaMemsetAsync(a.work, 0, balance_work_bytes(a.S, a.E), st);
  if (e == cudaSuccess) e = cudaMemsetAsync(a.counts, 0, (size_t)a.S * a.E * 4, st);
  if (e != cudaSuccess) return e;
  if (a.T) {
    balance_count_kernel<<<(a.T + 255) / 256, 256, 0, st>>>(a);
    const uint32_t grid = (a.T + 7) / 8;
    if (a.dtype == TS_DTYPE_F16) balance_token_kernel<TS_DTYPE_F16><<<grid, 256, 0, st>>>(a);
    else if (a.dtype == TS_DTYPE_BF16) balance_token_kernel<TS_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
    else balance_token_kernel<TS_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  }
  balance_loss_kernel<<<1, 1024, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace ts

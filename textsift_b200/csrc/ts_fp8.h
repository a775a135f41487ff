// ts_fp8.h — launchers of the 8-bit floating point operators and the router
// balance (internal to the library; the C ABI is in ops_fp8.cu).
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace ts {

constexpr uint32_t kFp8Block = 128;       // values that share a scale
constexpr uint32_t kFp8MatvecRows = 16;   // largest M of the single-token form
constexpr uint32_t kFp8MaxSize = 0x7fffff00u;  // largest M, N, K and E N of the products
__host__ __device__ constexpr uint32_t fp8_blocks(uint32_t n) { return n / kFp8Block + (n % kFp8Block != 0); }
// Values i .. i + 15 all lie below n, any n: i + 16 may not fit 32 bits.
__host__ __device__ constexpr bool fp8_whole(uint32_t i, uint32_t n) { return i < n && n - i >= 16; }
static_assert(fp8_whole(0, 16) && !fp8_whole(0, 15) && !fp8_whole(16, 16) && !fp8_whole(0xfffffff0u, 0xffffffffu) &&
                  fp8_whole(0xffffffe0u, 0xffffffffu),
              "ends of rows");

// Error flag of the kernels of this file on the current device (bounded waits
// that ran out), in device memory; null when it cannot be looked up.
int* fp8_err_flag();

struct Fp8QuantArgs {
  const void* x = nullptr;
  int dtype = 0;
  uint64_t ldx = 0;
  uint32_t rows = 0, cols = 0;
  uint8_t* codes = nullptr;
  uint64_t ldc = 0;
  float* scales = nullptr;
  uint64_t lds = 0;
};
cudaError_t launch_fp8_quant_rows(const Fp8QuantArgs& a, cudaStream_t st);
cudaError_t launch_fp8_quant_cols(const Fp8QuantArgs& a, cudaStream_t st);
cudaError_t launch_fp8_transpose(const uint8_t* codes, uint64_t ldw, const float* scales, uint32_t E, uint32_t N,
                                 uint32_t K, uint8_t* codes_t, uint64_t ldt, float* scales_t, cudaStream_t st);

struct Fp8MmArgs {
  const uint8_t* a = nullptr;
  uint64_t lda = 0;
  const float* as = nullptr;
  uint64_t ldas = 0;
  const uint8_t* w = nullptr;
  uint64_t ldw = 0;
  const float* ws = nullptr;
  uint64_t ldws = 0;
  int w_block = 128;               // 128: [E][nb][kb] scales; 1: a row operand's [kb][ldws]
  const uint16_t* bias = nullptr;  // fp16 [E][N] or null
  const int* seg = nullptr;        // [E + 1] or null
  uint32_t E = 1;
  void* out = nullptr;
  int out_dtype = 0;
  uint64_t ldo = 0;
  int accumulate = 0;
  uint32_t M = 0, N = 0, K = 0;
  int* err = nullptr;
};
cudaError_t launch_fp8_matmul(const Fp8MmArgs& a, cudaStream_t st);
// What that launches on a GPU of `sms` (8 or more) SMs, by sizes, w_block and segments
// alone: the sum of nothing, the single-token form, CTA pairs on 256 x 256
// tiles, single CTAs on 128 x 128 or 128 x 64, clusters that split k.
enum class Fp8Form { empty, matvec, pairs, wide, narrow, split2, split4, split8 };
Fp8Form fp8_matmul_form(const Fp8MmArgs& a, uint32_t sms);

// x of a floating type, quantised on the way, or codes (x_dtype TS_DTYPE_U8)
// with their scales xs.
struct Fp8MvArgs {
  const void* x = nullptr;
  int x_dtype = 0;
  uint64_t ldx = 0;
  const float* xs = nullptr;
  uint64_t ldxs = 0;
  const uint8_t* w = nullptr;
  uint64_t ldw = 0;
  const float* ws = nullptr;
  const uint16_t* bias = nullptr;
  void* out = nullptr;
  int out_dtype = 0;
  uint64_t ldo = 0;
  int accumulate = 0;
  uint32_t M = 0, N = 0, K = 0;
};
cudaError_t launch_fp8_matvec(const Fp8MvArgs& a, cudaStream_t st);

struct BalanceArgs {
  const void* logits = nullptr;
  int dtype = 0;
  uint64_t ldl = 0;
  const int* idx = nullptr;
  const uint8_t* mask = nullptr;
  const int* seq = nullptr;
  uint32_t S = 1, T = 0, E = 0, k = 0;
  float alpha = 0.0f, grad_scale = 1.0f;
  int* counts = nullptr;
  float* prob = nullptr;
  float* loss = nullptr;
  void* grad = nullptr;
  uint64_t ldg = 0;
  void* work = nullptr;
  uint32_t loss_blocks = 1;  // set by the launcher
};
constexpr uint32_t kBalanceMaxExperts = 1024, kBalanceMaxK = 64, kBalanceMaxTokens = 1u << 23;
// Calls of at most this many logits may run as one block.
constexpr uint64_t kBalanceOneLogits = 1u << 16;
size_t balance_work_bytes(uint32_t S, uint32_t E);
cudaError_t launch_router_balance(BalanceArgs a, cudaStream_t st);

}  // namespace ts

// ops_fp8.cu — the C ABI of the 8-bit floating point operators and of the
// router balance: argument checks, then the launchers of ts_fp8.h.  None of
// them allocates or synchronizes.
#include "textsift_cuda.h"
#include "ts_fp8.h"
#include "ts_kernels.h"
#include "ts_simt.h"

#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <unordered_map>

namespace {

// Errors go to the library's per-thread message (ts_cuda_last_error).
int fp8_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  ts::set_last_error(buf);
  return code;
}

int fp8_done(const char* what, cudaError_t e) {
  return e == cudaSuccess ? TS_OK : fp8_fail(TS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool is_float(int32_t dtype) {
  return dtype == TS_DTYPE_F16 || dtype == TS_DTYPE_BF16 || dtype == TS_DTYPE_F32;
}
size_t float_bytes(int32_t dtype) { return dtype == TS_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// The error flag is one for a device and all its streams, so whichever check
// finds it set cannot tell whose work failed.  Errors found are counted, and
// every stream is told of those it has not heard of.  A flag raised between
// the copy and the clearing below is not lost either: it belongs to the error
// that is counted after them, before its own stream can check.
struct OpErrors {
  std::mutex lock;
  struct Device {
    uint64_t found = 0;
    std::unordered_map<unsigned long long, uint64_t> told;  // by stream id; only streams that were told of any
  };
  std::unordered_map<int, Device> devices;
};
OpErrors& op_errors() {
  static OpErrors* e = new OpErrors;  // checks at exit may come after static destructors
  return *e;
}

// Codes of rows of `cols` values, ld bytes apart.
int check_codes(const char* what, const uint8_t* codes, uint64_t ld, uint32_t cols) {
  if (ld < cols) return fp8_fail(TS_ERR_ARG, "%s: rows of codes overlap (%llu < %u)", what, (unsigned long long)ld, cols);
  if (!aligned(codes, 16) || ld % 16)
    return fp8_fail(TS_ERR_UNSUPPORTED, "%s: rows of codes must start at multiples of 16 bytes", what);
  return TS_OK;
}

}  // namespace

extern "C" {

int ts_cuda_op_quant_fp8(const void* d_x, int32_t x_dtype, uint64_t ldx, uint32_t rows, uint32_t cols,
                         int32_t transpose, uint8_t* d_codes, uint64_t ldc, float* d_scales, uint64_t lds,
                         void* stream) {
  const char* me = "ts_cuda_op_quant_fp8";
  if (!is_float(x_dtype)) return fp8_fail(TS_ERR_ARG, "%s: x_dtype must be F16, BF16 or F32", me);
  if (rows == 0 || cols == 0) return TS_OK;
  if (!d_x || !d_codes || !d_scales) return fp8_fail(TS_ERR_ARG, "%s: null pointer", me);
  if (ldx < cols) return fp8_fail(TS_ERR_ARG, "%s: rows of x overlap", me);
  if (!aligned(d_x, float_bytes(x_dtype)) || !aligned(d_scales, 4))
    return fp8_fail(TS_ERR_ARG, "%s: x and scales must be aligned to their type", me);
  const uint32_t R = transpose ? cols : rows, C = transpose ? rows : cols;
  if (int rc = check_codes(me, d_codes, ldc, C)) return rc;
  if (lds < R) return fp8_fail(TS_ERR_ARG, "%s: blocks of scales overlap", me);
  ts::Fp8QuantArgs a;
  a.x = d_x; a.dtype = x_dtype; a.ldx = ldx; a.rows = rows; a.cols = cols;
  a.codes = d_codes; a.ldc = ldc; a.scales = d_scales; a.lds = lds;
  cudaStream_t st = (cudaStream_t)stream;
  return fp8_done(me, transpose ? ts::launch_fp8_quant_cols(a, st) : ts::launch_fp8_quant_rows(a, st));
}

int ts_cuda_op_transpose_fp8(const uint8_t* d_codes, uint64_t ldw, const float* d_scales, uint32_t E, uint32_t N,
                             uint32_t K, uint8_t* d_codes_t, uint64_t ldt, float* d_scales_t, void* stream) {
  const char* me = "ts_cuda_op_transpose_fp8";
  if (E == 0 || N == 0 || K == 0) return TS_OK;
  if (!d_codes || !d_scales || !d_codes_t || !d_scales_t) return fp8_fail(TS_ERR_ARG, "%s: null pointer", me);
  if (!aligned(d_scales, 4) || !aligned(d_scales_t, 4))
    return fp8_fail(TS_ERR_ARG, "%s: scales must be aligned to their type", me);
  if (E > 65535) return fp8_fail(TS_ERR_UNSUPPORTED, "%s: more than 65535 experts", me);
  if (int rc = check_codes(me, d_codes, ldw, K)) return rc;
  if (int rc = check_codes(me, d_codes_t, ldt, N)) return rc;
  return fp8_done(me, ts::launch_fp8_transpose(d_codes, ldw, d_scales, E, N, K, d_codes_t, ldt, d_scales_t,
                                               (cudaStream_t)stream));
}

int ts_cuda_op_matmul_fp8(const uint8_t* d_a, uint64_t lda, const float* d_as, uint64_t ldas, const uint8_t* d_w,
                          uint64_t ldw, const float* d_ws, uint64_t ldws, int32_t w_block, const uint16_t* d_bias,
                          const int32_t* d_seg, uint32_t E, void* d_out, int32_t out_dtype, uint64_t ldo,
                          int32_t accumulate, uint32_t M, uint32_t N, uint32_t K, void* stream) {
  const char* me = "ts_cuda_op_matmul_fp8";
  if (!is_float(out_dtype)) return fp8_fail(TS_ERR_ARG, "%s: out_dtype must be F16, BF16 or F32", me);
  if (accumulate && out_dtype != TS_DTYPE_F32) return fp8_fail(TS_ERR_ARG, "%s: only F32 accumulates", me);
  if (w_block != 128 && w_block != 1) return fp8_fail(TS_ERR_ARG, "%s: w_block must be 128 or 1", me);
  if (E == 0 || (E > 1 && !d_seg)) return fp8_fail(TS_ERR_ARG, "%s: E must be 1 without segments", me);
  if (w_block == 1 && (E != 1 || d_seg)) return fp8_fail(TS_ERR_ARG, "%s: w_block 1 takes no segments", me);
  if (E > 1024) return fp8_fail(TS_ERR_UNSUPPORTED, "%s: more than 1024 experts", me);
  if (M > ts::kFp8MaxSize || N > ts::kFp8MaxSize || K > ts::kFp8MaxSize || (uint64_t)E * N > ts::kFp8MaxSize)
    return fp8_fail(TS_ERR_UNSUPPORTED, "%s: sizes must stay below 2^31", me);
  if (M == 0 || N == 0) return TS_OK;
  if (!d_out || (K && (!d_a || !d_as || !d_w || !d_ws))) return fp8_fail(TS_ERR_ARG, "%s: null pointer", me);
  if (ldo < N) return fp8_fail(TS_ERR_ARG, "%s: rows of out overlap", me);
  if (!aligned(d_out, float_bytes(out_dtype)) || !aligned(d_as, 4) || !aligned(d_ws, 4) || !aligned(d_bias, 2) ||
      !aligned(d_seg, 4))
    return fp8_fail(TS_ERR_ARG, "%s: out, scales, bias and segments must be aligned to their type", me);
  if (K) {
    if (int rc = check_codes(me, d_a, lda, K)) return rc;
    if (int rc = check_codes(me, d_w, ldw, K)) return rc;
  }
  if (ldas < M || (w_block == 1 && ldws < N)) return fp8_fail(TS_ERR_ARG, "%s: blocks of scales overlap", me);
  ts::Fp8MmArgs a;
  a.a = d_a; a.lda = lda; a.as = d_as; a.ldas = ldas; a.w = d_w; a.ldw = ldw; a.ws = d_ws; a.ldws = ldws;
  a.w_block = w_block; a.bias = d_bias; a.seg = d_seg; a.E = E; a.out = d_out; a.out_dtype = out_dtype; a.ldo = ldo;
  a.accumulate = accumulate; a.M = M; a.N = N; a.K = K;
  a.err = ts::fp8_err_flag();
  if (!a.err) return fp8_fail(TS_ERR_CUDA, "%s: no error flag on this device", me);
  return fp8_done(me, ts::launch_fp8_matmul(a, (cudaStream_t)stream));
}

int ts_cuda_selftest_matmul_fp8_form(uint32_t M, uint32_t N, uint32_t K, int32_t w_block, int32_t segments, uint32_t E,
                                     uint32_t sms) {
  const char* me = "ts_cuda_selftest_matmul_fp8_form";
  if (M == 0 || N == 0 || E == 0) return fp8_fail(TS_ERR_ARG, "%s: sizes must be positive", me);
  if (w_block != 128 && w_block != 1) return fp8_fail(TS_ERR_ARG, "%s: w_block must be 128 or 1", me);
  if (sms != 0 && sms < 8) return fp8_fail(TS_ERR_ARG, "%s: sms must be 0 or 8 at least", me);
  ts::Fp8MmArgs a;
  static const int some[1] = {0};  // stands for segments, which are not read
  a.M = M; a.N = N; a.K = K; a.w_block = w_block; a.seg = segments ? some : nullptr; a.E = E;
  return (int)ts::fp8_matmul_form(a, sms ? sms : (uint32_t)ts::num_sms());
}

int ts_cuda_op_matvec_fp8(const void* d_x, int32_t x_dtype, uint64_t ldx, const uint8_t* d_w, uint64_t ldw,
                          const float* d_ws, const uint16_t* d_bias, void* d_out, int32_t out_dtype, uint64_t ldo,
                          uint32_t M, uint32_t N, uint32_t K, void* stream) {
  const char* me = "ts_cuda_op_matvec_fp8";
  if (!is_float(x_dtype) || !is_float(out_dtype))
    return fp8_fail(TS_ERR_ARG, "%s: x_dtype and out_dtype must be F16, BF16 or F32", me);
  if (M > ts::kFp8MatvecRows) return fp8_fail(TS_ERR_UNSUPPORTED, "%s: at most %u rows", me, ts::kFp8MatvecRows);
  if (N > ts::kFp8MaxSize || K > ts::kFp8MaxSize) return fp8_fail(TS_ERR_UNSUPPORTED, "%s: sizes must stay below 2^31", me);
  if (M == 0 || N == 0) return TS_OK;
  if (!d_out || (K && (!d_x || !d_w || !d_ws))) return fp8_fail(TS_ERR_ARG, "%s: null pointer", me);
  if (ldx < K || ldo < N) return fp8_fail(TS_ERR_ARG, "%s: rows of x or out overlap", me);
  if (!aligned(d_x, float_bytes(x_dtype)) || !aligned(d_out, float_bytes(out_dtype)) || !aligned(d_ws, 4) ||
      !aligned(d_bias, 2))
    return fp8_fail(TS_ERR_ARG, "%s: x, out, scales and bias must be aligned to their type", me);
  if (K)
    if (int rc = check_codes(me, d_w, ldw, K)) return rc;
  ts::Fp8MvArgs a;
  a.x = d_x; a.x_dtype = x_dtype; a.ldx = ldx; a.w = d_w; a.ldw = ldw; a.ws = d_ws; a.bias = d_bias; a.out = d_out;
  a.out_dtype = out_dtype; a.ldo = ldo; a.M = M; a.N = N; a.K = K;
  return fp8_done(me, ts::launch_fp8_matvec(a, (cudaStream_t)stream));
}

size_t ts_cuda_router_balance_work(uint32_t n_seqs, uint32_t E) { return ts::balance_work_bytes(n_seqs, E); }

int ts_cuda_op_router_balance(const void* d_logits, int32_t dtype, uint64_t ldl, const int32_t* d_idx,
                              const uint8_t* d_mask, const int32_t* d_seq, uint32_t n_seqs, uint32_t T, uint32_t E,
                              uint32_t k, float alpha, float grad_scale, int32_t* d_counts, float* d_prob,
                              float* d_loss, void* d_grad, uint64_t ldg, void* d_work, size_t work_bytes,
                              void* stream) {
  const char* me = "ts_cuda_op_router_balance";
  if (!is_float(dtype)) return fp8_fail(TS_ERR_ARG, "%s: dtype must be F16, BF16 or F32", me);
  if (E == 0 || k == 0 || n_seqs == 0) return fp8_fail(TS_ERR_ARG, "%s: E, k and n_seqs must be positive", me);
  if (n_seqs > 1 && !d_seq) return fp8_fail(TS_ERR_ARG, "%s: n_seqs must be 1 without d_seq", me);
  if (E > ts::kBalanceMaxExperts || k > ts::kBalanceMaxK || T > ts::kBalanceMaxTokens || n_seqs > ts::kBalanceMaxTokens)
    return fp8_fail(TS_ERR_UNSUPPORTED, "%s: at most %u experts, %u routes a token and %u tokens", me,
                    ts::kBalanceMaxExperts, ts::kBalanceMaxK, ts::kBalanceMaxTokens);
  if (!d_counts || !d_prob || !d_loss || !d_work || (T && (!d_logits || !d_idx)))
    return fp8_fail(TS_ERR_ARG, "%s: null pointer", me);
  if (work_bytes < ts::balance_work_bytes(n_seqs, E)) return fp8_fail(TS_ERR_ARG, "%s: d_work is too small", me);
  if (!aligned(d_work, 8) || !aligned(d_logits, float_bytes(dtype)) || !aligned(d_grad, float_bytes(dtype)) ||
      !aligned(d_idx, 4) || !aligned(d_seq, 4) || !aligned(d_counts, 4) || !aligned(d_prob, 4) || !aligned(d_loss, 4))
    return fp8_fail(TS_ERR_ARG, "%s: buffers must be aligned to their type, d_work to 8 bytes", me);
  if (ldl < E || (d_grad && ldg < E)) return fp8_fail(TS_ERR_ARG, "%s: rows of logits or gradient overlap", me);
  ts::BalanceArgs a;
  a.logits = d_logits; a.dtype = dtype; a.ldl = ldl; a.idx = d_idx; a.mask = d_mask; a.seq = d_seq; a.S = n_seqs;
  a.T = T; a.E = E; a.k = k; a.alpha = alpha; a.grad_scale = grad_scale; a.counts = d_counts; a.prob = d_prob;
  a.loss = d_loss; a.grad = d_grad; a.ldg = ldg; a.work = d_work;
  return fp8_done(me, ts::launch_router_balance(a, (cudaStream_t)stream));
}

int ts_cuda_op_check(void* stream) {
  const char* me = "ts_cuda_op_check";
  cudaStream_t st = (cudaStream_t)stream;
  int* flag = ts::fp8_err_flag();
  int err = 0, dev = 0;
  unsigned long long id = 0;
  if (!flag) return fp8_fail(TS_ERR_CUDA, "%s: no error flag on this device", me);
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaStreamGetId(st, &id);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);  // before the lock: others need not wait for this stream
  if (e != cudaSuccess) return fp8_done(me, e);
  OpErrors& errors = op_errors();
  std::lock_guard<std::mutex> hold(errors.lock);
  OpErrors::Device& d = errors.devices[dev];
  e = cudaMemcpyAsync(&err, flag, 4, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && err) {
    e = cudaMemsetAsync(flag, 0, 4, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess) d.found++;
  }
  if (e != cudaSuccess) return fp8_done(me, e);
  const auto heard = d.told.find(id);
  if (d.found == (heard == d.told.end() ? 0 : heard->second)) return TS_OK;
  d.told[id] = d.found;
  return fp8_fail(TS_ERR_DEVICE, "%s: device error flag (bounded wait timed out) on a stream of this device", me);
}

int ts_cuda_selftest_op_wait_timeout(uint32_t limit_us, int32_t* d_result, void* stream) {
  const char* me = "ts_cuda_selftest_op_wait_timeout";
  if (limit_us == 0 || limit_us > 1000000u) return fp8_fail(TS_ERR_ARG, "%s: limit_us must be in [1, 1000000]", me);
  if (!aligned(d_result, 4)) return fp8_fail(TS_ERR_ARG, "%s: d_result must be aligned to its type", me);
  int* flag = ts::fp8_err_flag();
  if (!flag) return fp8_fail(TS_ERR_CUDA, "%s: no error flag on this device", me);
  return fp8_done(me, ts::launch_wait_selftest(flag, 1000ull * limit_us, d_result, (cudaStream_t)stream));
}

}  // extern "C"

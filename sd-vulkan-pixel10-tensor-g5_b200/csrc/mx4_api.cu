// mx4_api.cu — C entry points of the MXFP4 operators (include/sdg.h): quantise, read back, linear, GroupNorm
// into an MXFP4 operand.
#include <cstdio>
#include <mutex>
#include <string>

#include "../../include/sdg.h"
#include "mx4.cuh"
#include "sdg_kernels.h"

namespace sdg {
int op_fail(int code, const std::string& msg);
}

namespace {

using sdg::op_fail;

// The word the kernels' bounded waits report to when the caller passes none: zero-initialised device memory of the
// library, looked up once per device; sdg_mx4_status reads and clears it. The look-up may load the module, so it runs with
// this thread's stream-capture mode relaxed: a first call inside a capture is fine.
static __device__ int g_mx4_err[64];
std::mutex g_mu;
int* g_err_dev[64] = {nullptr};

int* default_err_word() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_err_dev[dev]) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    const bool swapped = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_mx4_err) == cudaSuccess) g_err_dev[dev] = static_cast<int*>(p);
    if (swapped) cudaThreadExchangeStreamCaptureMode(&mode);
  }
  return g_err_dev[dev];
}

int status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return SDG_OK;
  if (e == cudaErrorInvalidValue) return op_fail(SDG_ERR_SHAPE, std::string(what) + ": unsupported shape or arguments");
  return op_fail(SDG_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t elem_bytes(int dtype) { return dtype == sdg::kF32 ? 4 : 2; }
// Rows and columns that 32-bit row, column and tile numbers hold with room for a tile behind the last.
constexpr int kMaxK = 1 << 23, kMaxRows = 1 << 30;
bool bad_size(int M, int K) { return M <= 0 || K <= 0 || M > kMaxRows || K > kMaxK; }

int linear_check(const char* what, int M, int K, const uint8_t* wcodes, const uint8_t* wscales, const float* bias, int N,
                 const void* residual, int act, int dtype, const void* y) {
  const std::string w(what);
  if (!wcodes || !wscales || !y || bad_size(M, K) || bad_size(N, K) || act < 0 || act > 2)
    return op_fail(SDG_ERR_ARG, w + ": bad arguments");
  if (dtype != sdg::kF16 && dtype != sdg::kBF16) return op_fail(SDG_ERR_ARG, w + ": dtype must be fp16 or bf16");
  if (act == 2 && residual) return op_fail(SDG_ERR_ARG, w + ": GEGLU takes no residual");
  if (act == 2 ? N % 32 : N % 8)
    return op_fail(SDG_ERR_SHAPE, w + (act == 2 ? ": GEGLU needs N a multiple of 32" : ": N must be a multiple of 8"));
  if (!aligned(wcodes, 16) || !aligned(wscales, 16) || !aligned(y, 16) || !aligned(residual, 16) || !aligned(bias, 4))
    return op_fail(SDG_ERR_ARG, w + ": weight, scale, residual and output pointers must be 16-byte aligned");
  return SDG_OK;
}

// Waits for the stream, then reads and clears an error word: SDG_ERR_DEVICE with its code, if it held one.
int take_code(int* word, cudaStream_t s, const char* what) {
  int v = 0;
  cudaError_t e = cudaMemcpyAsync(&v, word, sizeof v, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && v != 0) {
    e = cudaMemsetAsync(word, 0, sizeof v, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) return status(e, what);
  if (v == 0) return SDG_OK;
  char buf[128];
  snprintf(buf, sizeof buf, "%s: device error word 0x%x (a kernel's bounded wait expired)", what, v);
  return op_fail(SDG_ERR_DEVICE, buf);
}

// The codes' part of the scratch, rounded up so that the scales behind it are aligned.
size_t code_space(int M, int K) { return ((size_t)M * (sdg::mx_kp(K) / 2) + 511) / 512 * 512; }

int linear_run(sdg::Mx4LinearArgs a, int M, int K, const uint8_t* wcodes, const uint8_t* wscales, const float* bias, int N,
               const void* residual, int act, int dtype, void* y, int* err_word, cudaStream_t s) {
  a.wcodes = wcodes; a.wscales = wscales;
  a.M = M; a.N = N; a.K = K; a.bias = bias; a.residual = residual; a.act = act; a.dtype = dtype; a.y = y;
  int* err = err_word ? err_word : default_err_word();
  if (!err) return op_fail(SDG_ERR_CUDA, "linear_mx4: no device error word");
  return status(sdg::launch_mx4_linear(a, err, s), "linear_mx4");
}

}  // namespace

extern "C" {

SDG_API size_t sdg_mx4_code_bytes(int M, int K) {
  return bad_size(M, K) ? 0 : (size_t)M * (sdg::mx_kp(K) / 2);
}
SDG_API size_t sdg_mx4_scale_bytes(int M, int K) {
  return bad_size(M, K) ? 0 : (size_t)sdg::mx_rtiles(M) * sdg::mx_ktiles(K) * sdg::kMxTileBytes;
}

SDG_API int sdg_quantize_mx4(const void* x, int dtype, int M, int K, int64_t ldx, uint8_t* codes, uint8_t* scales,
                             void* stream) {
  if (!x || !codes || !scales || bad_size(M, K) || ldx < 0)
    return op_fail(SDG_ERR_ARG, "quantize_mx4: bad arguments");
  if (dtype < sdg::kF16 || dtype > sdg::kF32) return op_fail(SDG_ERR_ARG, "quantize_mx4: dtype must be fp16, bf16 or fp32");
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(x, elem_bytes(dtype)))
    return op_fail(SDG_ERR_ARG, "quantize_mx4: codes and scales must be 16-byte aligned, x aligned to its type");
  return status(sdg::launch_mx4_quantize(x, dtype, M, K, ldx, codes, scales, static_cast<cudaStream_t>(stream)),
                "quantize_mx4");
}

SDG_API int sdg_dequantize_mx4(const uint8_t* codes, const uint8_t* scales, int M, int K, int dtype, void* y,
                               void* stream) {
  if (!y || !codes || !scales || bad_size(M, K))
    return op_fail(SDG_ERR_ARG, "dequantize_mx4: bad arguments");
  if (dtype < sdg::kF16 || dtype > sdg::kF32)
    return op_fail(SDG_ERR_ARG, "dequantize_mx4: dtype must be fp16, bf16 or fp32");
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(y, elem_bytes(dtype)))
    return op_fail(SDG_ERR_ARG, "dequantize_mx4: codes and scales must be 16-byte aligned, y aligned to its type");
  return status(sdg::launch_mx4_dequantize(codes, scales, M, K, dtype, y, static_cast<cudaStream_t>(stream)),
                "dequantize_mx4");
}

SDG_API int sdg_linear_mx4(const uint8_t* xcodes, const uint8_t* xscales, int M, int K, const uint8_t* wcodes,
                           const uint8_t* wscales, const float* bias, int N, const void* residual, int act, int dtype,
                           void* y, int* err_word, void* stream) {
  int st = linear_check("linear_mx4", M, K, wcodes, wscales, bias, N, residual, act, dtype, y);
  if (st) return st;
  if (!xcodes || !xscales || !aligned(xcodes, 16) || !aligned(xscales, 16))
    return op_fail(SDG_ERR_ARG, "linear_mx4: x codes and scales must be 16-byte aligned device pointers");
  sdg::Mx4LinearArgs a;
  a.xcodes = xcodes;
  a.xscales = xscales;
  return linear_run(a, M, K, wcodes, wscales, bias, N, residual, act, dtype, y, err_word,
                    static_cast<cudaStream_t>(stream));
}

SDG_API int sdg_linear_mx4_x(const void* x, int M, int K, int64_t ldx, const uint8_t* wcodes, const uint8_t* wscales,
                             const float* bias, int N, const void* residual, int act, int dtype, void* y, void* scratch,
                             size_t scratch_bytes, int* err_word, void* stream) {
  int st = linear_check("linear_mx4", M, K, wcodes, wscales, bias, N, residual, act, dtype, y);
  if (st) return st;
  const size_t need = sdg_linear_mx4_scratch_bytes(x, M, K, ldx, N);
  if (!x || ldx < 0 || !aligned(x, 2) || (need && (!scratch || !aligned(scratch, 16) || scratch_bytes < need)))
    return op_fail(SDG_ERR_ARG, "linear_mx4: bad x, or scratch smaller than sdg_linear_mx4_scratch_bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  sdg::Mx4LinearArgs a;
  if (need == 0) {
    a.x = x;
    a.ldx = ldx;
  } else {
    uint8_t* xc = static_cast<uint8_t*>(scratch);
    uint8_t* xs = xc + code_space(M, K);
    st = status(sdg::launch_mx4_quantize(x, dtype, M, K, ldx, xc, xs, s), "linear_mx4");
    if (st) return st;
    a.xcodes = xc;
    a.xscales = xs;
  }
  return linear_run(a, M, K, wcodes, wscales, bias, N, residual, act, dtype, y, err_word, s);
}

SDG_API int sdg_selftest_stalled_linear_mx4(const void* x, const uint8_t* xscales, int M, int K, const uint8_t* wcodes,
                                            const uint8_t* wscales, int N, const void* residual, void* y, int form,
                                            int stall_who, int stall_iter, int wait_limit_us, int* err_word,
                                            void* stream) {
  const char* what = "selftest_stalled_linear_mx4";
  int st = linear_check(what, M, K, wcodes, wscales, nullptr, N, residual, 0, sdg::kF16, y);
  if (st) return st;
  if (!x || !aligned(x, 16) || !aligned(xscales, 16) || stall_iter < 0 || stall_who < 0 || stall_who > 1 ||
      wait_limit_us <= 0 || wait_limit_us > 2000000)
    return op_fail(SDG_ERR_ARG, std::string(what) + ": bad arguments");
  sdg::Mx4LinearArgs a;
  if (xscales) {
    a.xcodes = static_cast<const uint8_t*>(x);
    a.xscales = xscales;
  } else {
    if (!sdg::mx4_linear_takes_x(x, M, K, K, N)) return op_fail(SDG_ERR_ARG, std::string(what) + ": not a fused product");
    a.x = x;
    a.ldx = K;
  }
  a.M = M; a.N = N; a.K = K; a.wcodes = wcodes; a.wscales = wscales; a.residual = residual; a.y = y;
  const sdg::Mx4Form f = sdg::mx4_linear_form(a);
  if (f == sdg::kMx4Rows || (int)f != form || (stall_who && f != sdg::kMx4Fused && f != sdg::kMx4Pair))
    return op_fail(SDG_ERR_ARG, std::string(what) + ": the product does not run in that form");
  a.test_stall_iter = stall_iter;
  a.test_stall_who = stall_who;
  a.wait_limit_ns = 1000ull * (unsigned long long)wait_limit_us;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int* err = err_word ? err_word : default_err_word();
  if (!err) return op_fail(SDG_ERR_CUDA, std::string(what) + ": no device error word");
  st = status(sdg::launch_mx4_linear(a, err, s), what);
  return st || !err_word ? st : take_code(err_word, s, what);
}

SDG_API int sdg_mx4_status(void* stream) {
  const char* what = "mx4_status";
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(s, &cap);
  if (e == cudaErrorStreamCaptureImplicit || (e == cudaSuccess && cap != cudaStreamCaptureStatusNone))
    return op_fail(SDG_ERR_ARG, std::string(what) + ": the stream is being captured");
  if (e != cudaSuccess) return status(e, what);
  int* word = default_err_word();
  if (!word) return op_fail(SDG_ERR_CUDA, std::string(what) + ": no device error word");
  return take_code(word, s, what);
}

SDG_API size_t sdg_linear_mx4_scratch_bytes(const void* x, int M, int K, int64_t ldx, int N) {
  if (bad_size(M, K) || N <= 0 || sdg::mx4_linear_takes_x(x, M, K, ldx, N)) return 0;
  return code_space(M, K) + sdg_mx4_scale_bytes(M, K);
}

SDG_API size_t sdg_groupnorm_mx4_scratch_bytes(int B, int HW, int C, int groups) {
  if (B <= 0 || HW <= 0 || C <= 0 || groups <= 0) return 0;
  return sdg::mx4_groupnorm_scratch_bytes(B, HW, C, groups);
}

SDG_API int sdg_groupnorm_mx4(const void* x, int dtype, int B, int HW, int C, int groups, const float* gamma,
                              const float* beta, float eps, int silu, uint8_t* codes, uint8_t* scales,
                              float* stats_scratch, void* stream) {
  if (!x || !gamma || !beta || !codes || !scales || !stats_scratch || B <= 0 || HW <= 0 || C <= 0 || groups <= 0)
    return op_fail(SDG_ERR_ARG, "groupnorm_mx4: bad arguments");
  if (dtype != sdg::kF16 && dtype != sdg::kBF16) return op_fail(SDG_ERR_ARG, "groupnorm_mx4: dtype must be fp16 or bf16");
  if (C % 8 || C % groups || C > 4096 || B > 65535 || (int64_t)B * HW > kMaxRows)
    return op_fail(SDG_ERR_SHAPE, "groupnorm_mx4: C must be a multiple of 8 and of groups, at most 4096; B at most 65535, B * HW at most 2^30");
  if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(stats_scratch, 8) || !aligned(gamma, 4) ||
      !aligned(beta, 4))
    return op_fail(SDG_ERR_ARG, "groupnorm_mx4: x, codes and scales must be 16-byte aligned");
  sdg::Mx4GroupNormArgs a;
  a.x = x; a.dtype = dtype; a.B = B; a.HW = HW; a.C = C; a.groups = groups;
  a.gamma = gamma; a.beta = beta; a.eps = eps; a.silu = silu;
  a.codes = codes; a.scales = scales; a.stats = stats_scratch;
  return status(sdg::launch_mx4_groupnorm(a, static_cast<cudaStream_t>(stream)), "groupnorm_mx4");
}

}  // extern "C"

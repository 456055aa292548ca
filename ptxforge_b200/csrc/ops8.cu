// ops8.cu -- the 8-bit operators of the C ABI (include/pf_b200.h): int8 store and restore, the int8 product with
// token and channel scales, the fused product with an 8-bit checkpoint, and its gradients.
//
// None needs a pf_ctx: operands and workspaces are the caller's, every launch goes on the caller's stream, nothing is
// allocated and nothing is kept from one call for the next but each device's properties.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "pf_b200.h"
#include "gemm8_simple.cuh"
#include "host_util.cuh"
#include "quant_s8.cuh"

// Bounded waits that ran out, of every kernel here: bits are only ever set, until pf_ops8_status clears them, so calls
// that overlap on the GPU may share it.
static __device__ unsigned ops8_status_word;

namespace {

using pf::DeviceGuard;
typedef __nv_bfloat16 bf16;

constexpr int kMaxDevices = 64;
constexpr int kMaxSumK = 131071;  // K * 128 * 128 stays below 2^31

struct Device {
  std::mutex mu;
  bool ready = false;
  int cc_major = 0, num_sms = 0;
  unsigned *status = nullptr;
};
Device g_devices[kMaxDevices];

struct Err {
  char *text;
  size_t len;
  int operator()(int code, const char *fmt, ...) const {
    if (text && len) {
      va_list ap;
      va_start(ap, fmt);
      vsnprintf(text, len, fmt, ap);
      va_end(ap);
    }
    return code;
  }
};

// The device's properties, looked up once; a failed look-up is tried again by the next call.
int device_of(int device, const Err &err, Device **out) {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n || device >= kMaxDevices) {
    cudaGetLastError();
    return err(PF_ENODEV, "no CUDA device %d", device);
  }
  Device &d = g_devices[device];
  std::lock_guard<std::mutex> lk(d.mu);
  if (!d.ready) {
    DeviceGuard g(device);
    void *p = nullptr;
    cudaError_t e = cudaDeviceGetAttribute(&d.cc_major, cudaDevAttrComputeCapabilityMajor, device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&d.num_sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess && d.cc_major == 10) e = cudaGetSymbolAddress(&p, ops8_status_word);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return err(PF_ECUDA, "set-up on device %d failed: %s", device, cudaGetErrorString(e));
    }
    d.status = static_cast<unsigned *>(p);
    d.ready = true;
  }
  if (d.cc_major != 10) return err(PF_ENODEV, "device %d is not an sm_100 GPU", device);
  *out = &d;
  return PF_OK;
}

int stream_of(int device, void *stream, const Err &err, cudaStream_t *out) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  *out = s;
  // A capturing stream cannot be asked for its device; one of another device fails the launch itself.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(s, &capture);
  if (e == cudaSuccess && capture == cudaStreamCaptureStatusActive) return PF_OK;
  int at = -1;
  if (e == cudaSuccess) e = cudaStreamGetDevice(s, &at);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return err(PF_EINVAL, "stream is not a valid CUDA stream: %s", cudaGetErrorString(e));
  }
  if (at != device) return err(PF_EINVAL, "stream belongs to device %d, not device %d", at, device);
  return PF_OK;
}

int launched(const Err &err) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PF_OK : err(PF_ECUDA, "launch: %s", cudaGetErrorString(e));
}

template <class... P>
bool any_null(const P *...p) {
  return (... || (p == nullptr));
}

unsigned blocks_of(long long n, int per) { return static_cast<unsigned>((n + per - 1) / per); }

template <class T>
void quantize(const void *X, long long ldx, int rows, int cols, int axis, int8_t *Q, long long ldq, float *scale,
              cudaStream_t s) {
  const T *x = static_cast<const T *>(X);
  if (axis == 1) {
    pf::quantize_rows_s8<T><<<rows, 256, 0, s>>>(x, ldx, cols, Q, ldq, scale);
  } else {
    pf::scale_cols_s8<T><<<blocks_of(cols, 32), dim3(32, 8), 0, s>>>(x, ldx, rows, cols, scale);
    pf::quantize_cols_s8<T><<<rows, 256, 0, s>>>(x, ldx, cols, scale, Q, ldq);
  }
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// The parts of the backward pass's workspace, in order, each 256-byte aligned.
struct BackwardSpace {
  size_t dz, a, partial, total;
  int parts;
  BackwardSpace(int M, int N, int K) {
    parts = (M + pf::kDzRows - 1) / pf::kDzRows;
    dz = 0;
    a = dz + round256(size_t(M) * N * sizeof(bf16));
    partial = a + round256(size_t(M) * K * sizeof(bf16));
    total = partial + round256(size_t(parts) * N * sizeof(float));
  }
};

template <class T, class Acc, class Store>
void product(const pf::Strided<T> &g, int M, int N, int K, const Store &store, cudaStream_t s) {
  pf::gemm8_simple<T, Acc><<<dim3(blocks_of(M, 64), blocks_of(N, 64)), 256, 0, s>>>(g, M, N, K, store);
}

}  // namespace

extern "C" {

int pf_quantize_s8(int device, pf_dtype src, int rows, int cols, const void *X, long long ldx, int axis,
                   signed char *codes, long long ld_codes, float *scale, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (rows < 0 || cols < 0) return err(PF_EINVAL, "rows and cols must not be negative (got %d, %d)", rows, cols);
  if (src != PF_F32 && src != PF_BF16) return err(PF_EINVAL, "the source type must be f32 or bf16");
  if (axis != 0 && axis != 1) return err(PF_EINVAL, "axis must be 1 (a scale for each row) or 0 (for each column), got %d", axis);
  if (rows == 0 || cols == 0) return PF_OK;
  if (any_null(X, codes, scale)) return err(PF_EINVAL, "null argument");
  if (ldx < cols || ld_codes < cols) return err(PF_EINVAL, "a row stride is below cols");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  int8_t *q = reinterpret_cast<int8_t *>(codes);
  if (src == PF_F32) quantize<float>(X, ldx, rows, cols, axis, q, ld_codes, scale, s);
  else quantize<bf16>(X, ldx, rows, cols, axis, q, ld_codes, scale, s);
  return launched(err);
}

int pf_dequantize_s8(int device, int rows, int cols, const signed char *codes, long long ld_codes, const float *scale,
                     int axis, pf_dtype dst, void *X, long long ldx, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (rows < 0 || cols < 0) return err(PF_EINVAL, "rows and cols must not be negative (got %d, %d)", rows, cols);
  if (dst != PF_F32 && dst != PF_BF16) return err(PF_EINVAL, "the destination type must be f32 or bf16");
  if (axis != 0 && axis != 1) return err(PF_EINVAL, "axis must be 1 (a scale for each row) or 0 (for each column), got %d", axis);
  if (rows == 0 || cols == 0) return PF_OK;
  if (any_null(codes, scale, X)) return err(PF_EINVAL, "null argument");
  if (ldx < cols || ld_codes < cols) return err(PF_EINVAL, "a row stride is below cols");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  const int8_t *q = reinterpret_cast<const int8_t *>(codes);
  if (dst == PF_F32) pf::dequantize_s8<float><<<rows, 256, 0, s>>>(q, ld_codes, cols, scale, axis, static_cast<float *>(X), ldx);
  else pf::dequantize_s8<bf16><<<rows, 256, 0, s>>>(q, ld_codes, cols, scale, axis, static_cast<bf16 *>(X), ldx);
  return launched(err);
}

int pf_gemm_s8(int device, int M, int N, int K, const signed char *A, long long lda, const signed char *B, long long ldb,
               const float *scale_a, const float *scale_b, const float *bias, int gelu, pf_dtype out, void *C,
               long long ldc, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (M < 0 || N < 0) return err(PF_EINVAL, "M and N must not be negative (got %d, %d)", M, N);
  if (K < 1 || K > kMaxSumK)
    return err(PF_EINVAL, "K must be 1 to %d, so that a sum of int8 products fits 32 bits (got %d)", kMaxSumK, K);
  if (out != PF_F32 && out != PF_BF16) return err(PF_EINVAL, "the output type must be f32 or bf16");
  if (M == 0 || N == 0) return PF_OK;
  if (any_null(A, B, C) || any_null(scale_a, scale_b)) return err(PF_EINVAL, "null argument");
  if (lda < K || ldb < N || ldc < N) return err(PF_EINVAL, "a row stride is below the row's length");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  const pf::Strided<int8_t> op{reinterpret_cast<const int8_t *>(A), reinterpret_cast<const int8_t *>(B), lda, 1, ldb, 1};
  product<int8_t, int>(op, M, N, K, pf::StoreS8{scale_a, scale_b, bias, gelu, out == PF_F32, C, ldc}, s);
  return launched(err);
}

int pf_gemm_bias_gelu_checkpoint(int device, int M, int N, int K, const void *A, const void *B, const float *bias,
                                 void *C, signed char *a_codes, float *a_scale, unsigned char *grad_codes, void *stream,
                                 char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (M < 0 || N < 1 || K < 1) return err(PF_EINVAL, "M must not be negative, N and K positive (got %d, %d, %d)", M, N, K);
  if (N % 8 || K % 8) return err(PF_ESHAPE, "rows of A, B and C must be multiples of 16 bytes (N=%d, K=%d)", N, K);
  if (M == 0) return PF_OK;
  if (any_null(A, B, C) || any_null(bias) || any_null(grad_codes)) return err(PF_EINVAL, "null argument");
  if ((a_codes == nullptr) != (a_scale == nullptr)) return err(PF_EINVAL, "a_codes and a_scale go together");
  if (!pf::aligned16(A) || !pf::aligned16(B) || !pf::aligned16(C) || !pf::aligned16(grad_codes) || !pf::aligned16(a_codes))
    return err(PF_EINVAL, "operands must be 16-byte aligned");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  if (a_codes) quantize<bf16>(A, K, M, K, 1, reinterpret_cast<int8_t *>(a_codes), K, a_scale, s);
  const pf::Strided<bf16> op{static_cast<const bf16 *>(A), static_cast<const bf16 *>(B), K, 1, N, 1};
  product<bf16, float>(op, M, N, K, pf::StoreCheckpoint{bias, static_cast<bf16 *>(C), grad_codes, N}, s);
  return launched(err);
}

size_t pf_gemm_bias_gelu_backward_workspace(int M, int N, int K) {
  return M < 1 || N < 1 || K < 1 ? 0 : BackwardSpace(M, N, K).total;
}

int pf_gemm_bias_gelu_backward(int device, int M, int N, int K, const void *dC, const void *B, const signed char *a_codes,
                               const float *a_scale, const unsigned char *grad_codes, void *dA, void *dB, float *dbias,
                               void *workspace, size_t workspace_bytes, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (M < 0 || N < 1 || K < 1) return err(PF_EINVAL, "M must not be negative, N and K positive (got %d, %d, %d)", M, N, K);
  if (N % 8 || K % 8) return err(PF_ESHAPE, "rows of dC, B and the gradients must be multiples of 16 bytes (N=%d, K=%d)", N, K);
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  if (M == 0) {  // no tokens: the sums over them are zero
    cudaError_t e = cudaSuccess;
    if (dB) e = cudaMemsetAsync(dB, 0, size_t(N) * K * sizeof(bf16), s);
    if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, size_t(N) * sizeof(float), s);
    return e == cudaSuccess ? PF_OK : err(PF_ECUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
  }
  if (any_null(dC) || any_null(grad_codes) || (dA && !B) || (dB && (!a_codes || !a_scale)))
    return err(PF_EINVAL, "null argument");
  const BackwardSpace w(M, N, K);
  if (!workspace || workspace_bytes < w.total)
    return err(PF_EINVAL, "the workspace holds %zu bytes, %zu are needed", workspace ? workspace_bytes : size_t(0), w.total);
  if (!pf::aligned16(dC) || !pf::aligned16(B) || !pf::aligned16(a_codes) || !pf::aligned16(grad_codes) ||
      !pf::aligned16(dA) || !pf::aligned16(dB) || reinterpret_cast<uintptr_t>(workspace) % 256)
    return err(PF_EINVAL, "operands must be 16-byte aligned, the workspace 256-byte aligned");
  char *base = static_cast<char *>(workspace);
  bf16 *dz = reinterpret_cast<bf16 *>(base + w.dz), *a = reinterpret_cast<bf16 *>(base + w.a);
  float *partial = reinterpret_cast<float *>(base + w.partial);
  pf::gelu_backward_dz<<<dim3(blocks_of(N, 256), w.parts), 256, 0, s>>>(
      static_cast<const bf16 *>(dC), grad_codes, dB ? a_scale : nullptr, M, N, dz, partial);
  if (dbias) pf::sum_partials<<<blocks_of(N, 256), 256, 0, s>>>(partial, w.parts, N, dbias);
  if (dA) {
    const pf::Strided<bf16> op{dz, static_cast<const bf16 *>(B), N, 1, 1, N};
    product<bf16, float>(op, M, K, N, pf::StoreBf16{dB ? a_scale : nullptr, static_cast<bf16 *>(dA), K}, s);
  }
  if (dB) {
    pf::input_of_codes<<<M, 256, 0, s>>>(reinterpret_cast<const int8_t *>(a_codes), a_scale, K, a);
    const pf::Strided<bf16> op{a, dz, 1, K, N, 1};
    product<bf16, float>(op, K, N, M, pf::StoreBf16{nullptr, static_cast<bf16 *>(dB), N}, s);
  }
  return launched(err);
}

int pf_dequantize_gelu_grad(int device, long long count, const unsigned char *codes, pf_dtype dst, void *X, void *stream,
                            char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (count < 0) return err(PF_EINVAL, "count must not be negative (got %lld)", count);
  if (dst != PF_F32 && dst != PF_BF16) return err(PF_EINVAL, "the destination type must be f32 or bf16");
  if (count == 0) return PF_OK;
  if (any_null(codes) || any_null(X)) return err(PF_EINVAL, "null argument");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  const unsigned grid = static_cast<unsigned>(std::min<long long>((count + 255) / 256, 1 << 20));
  if (dst == PF_F32) pf::dequantize_grad<float><<<grid, 256, 0, s>>>(codes, count, static_cast<float *>(X));
  else pf::dequantize_grad<bf16><<<grid, 256, 0, s>>>(codes, count, static_cast<bf16 *>(X));
  return launched(err);
}

int pf_ops8_status(int device, unsigned *err_word, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (!err_word) return err(PF_EINVAL, "null argument");
  Device *d;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(err_word, d->status, sizeof *err_word, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess) e = cudaMemset(d->status, 0, sizeof *err_word);
  return e == cudaSuccess ? PF_OK : err(PF_ECUDA, "status read: %s", cudaGetErrorString(e));
}

}  // extern "C"

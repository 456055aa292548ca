// quant_s8.cuh -- int8 codes with one fp32 scale for each row (token) or column (channel) of a matrix, and the
// 8-bit GELU derivative of the training checkpoint.
//
//   s = max(max |x| / 127, 2^-126) over the row or column;  q = rint(x / s), in [-127, 127];  x~ = q s
//
// The quotient is the real one rounded once to the nearest whole number (ties to even), so the codes do not
// depend on how the division is done.  A row (column) that holds an infinity or a NaN gets the scale NaN and
// codes 0: what is computed from it comes out NaN instead of plausible.
//
// GELU derivative d = gelu_tanh'(z), in (-0.1290, 1.1290): code = rint(200 d) + 26, so 26 is exactly 0 (a dead
// unit), 226 exactly 1 (a saturated one), codes run from 0 to 252 and 255 stands for NaN.  A fixed step needs no
// scale to be found or kept; it errs by at most 0.0025, less than z itself kept in 8 bits would make d err.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

namespace pf {

constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126: scales stay normal numbers
constexpr float kGradSteps = 200.f;
constexpr int kGradZero = 26;
constexpr int kGradNan = 255;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// |x| as ordered bits: finite < infinity < NaN, so a maximum over them keeps what is not finite.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The scale of a row (column) from its largest abs_bits.
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 127.f), kLeastScale);
}

// rint(x / s) for a scale from scale_of.  x * (1 / s) is within 3e-5 of the quotient (|quotient| < 128, two
// roundings of 2^-24 relative); only a value that near to a half step may round to the wrong side, and there the
// sign of x - (k + 1/2) s, which one fused multiply-add gives exactly, decides.  A NaN scale gives code 0.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  const float t = x * inv;
  float r = rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) < 3e-5f) {
    const float k = floorf(t);
    const float e = fmaf(-(k + 0.5f), s, x);
    r = e > 0.f ? k + 1.f : e < 0.f ? k : rintf(k + 0.5f);
  }
  const int q = __float2int_rn(r);  // NaN -> 0
  return max(-127, min(127, q));
}

__device__ __forceinline__ float grad_value(uint32_t code) {
  const float d = __fdiv_rn(static_cast<float>(static_cast<int>(code) - kGradZero), kGradSteps);
  return code == kGradNan ? __uint_as_float(0x7FC00000u) : d;
}

// Largest abs_bits of a block's threads (`sh`: one word for each warp); the result is everybody's.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *sh) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) m = max(m, sh[w]);
  return m;
}

// A scale for each row: one block a row.
template <class T>
__global__ void quantize_rows_s8(const T *X, long long ldx, int cols, int8_t *Q, long long ldq, float *scale) {
  __shared__ uint32_t sh[32];
  const long long r = blockIdx.x;
  const T *x = X + r * ldx;
  uint32_t m = 0;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) m = max(m, abs_bits(to_f32(x[c])));
  const float s = scale_of(block_max(m, sh)), inv = __fdiv_rn(1.f, s);
  for (int c = threadIdx.x; c < cols; c += blockDim.x)
    Q[r * ldq + c] = static_cast<int8_t>(code_of(to_f32(x[c]), s, inv));
  if (threadIdx.x == 0) scale[r] = s;
}

// A scale for each column: 32 columns a block of 32 x 8 threads.
template <class T>
__global__ void scale_cols_s8(const T *X, long long ldx, int rows, int cols, float *scale) {
  __shared__ uint32_t sh[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x;
  uint32_t m = 0;
  if (c < cols)
    for (long long r = threadIdx.y; r < rows; r += 8) m = max(m, abs_bits(to_f32(X[r * ldx + c])));
  sh[threadIdx.y][threadIdx.x] = m;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) m = max(m, sh[i][threadIdx.x]);
    scale[c] = scale_of(m);
  }
}
template <class T>
__global__ void quantize_cols_s8(const T *X, long long ldx, int cols, const float *scale, int8_t *Q, long long ldq) {
  const long long r = blockIdx.x;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const float s = scale[c];
    Q[r * ldq + c] = static_cast<int8_t>(code_of(to_f32(X[r * ldx + c]), s, __fdiv_rn(1.f, s)));
  }
}

template <class T>
__global__ void dequantize_s8(const int8_t *Q, long long ldq, int cols, const float *scale, int by_row, T *X,
                              long long ldx) {
  const long long r = blockIdx.x;
  for (int c = threadIdx.x; c < cols; c += blockDim.x)
    X[r * ldx + c] = from_f32<T>(static_cast<float>(Q[r * ldq + c]) * scale[by_row ? r : c]);
}

template <class T>
__global__ void dequantize_grad(const uint8_t *D, long long n, T *X) {
  for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * blockDim.x)
    X[i] = from_f32<T>(grad_value(D[i]));
}

// Rows of bytes that start anywhere -> rows of whole 16-byte words.  Each word is put together from the aligned
// 4-byte words that hold its bytes; a word with no byte of the row is not read.  What follows a row's end is whatever
// shares its last word, and is never used.
__global__ void align_rows(const uint8_t *X, long long ld, int cols, uint4 *Y, long long ld_y) {
  const long long r = blockIdx.x;
  const uintptr_t row = reinterpret_cast<uintptr_t>(X + r * ld);
  const unsigned shift = 8 * static_cast<unsigned>(row & 3);
  const uint32_t *x = reinterpret_cast<const uint32_t *>(row & ~uintptr_t(3));
  const int words = static_cast<int>((cols + (row & 3) + 3) / 4);
  for (int i = threadIdx.x; i * 16 < cols; i += blockDim.x) {
    uint32_t v[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] = i * 4 + j < words ? __ldg(x + i * 4 + j) : 0u;
    Y[r * ld_y + i] = make_uint4(__funnelshift_r(v[0], v[1], shift), __funnelshift_r(v[1], v[2], shift),
                                 __funnelshift_r(v[2], v[3], shift), __funnelshift_r(v[3], v[4], shift));
  }
}

// The input's scale split into s = m 2^e, so that the backward pass rounds once where it could round twice: the
// tensor cores take q 2^e, which is exact in bf16 (7 bits), and round(m dz), whose product is q s dz; dA, which
// has no use for m, is divided by it at the end.  1 <= m < 2, so a token of tiny or no input keeps its dA.  A scale
// that is not finite goes to e alone: dB is NaN then, dA is not.
struct SplitScale {
  float m, e;
};
__device__ __forceinline__ SplitScale split_scale(float s) {
  const uint32_t b = __float_as_uint(s), field = b & 0x7F800000u;
  if (field == 0u || field == 0x7F800000u) return {1.f, field == 0u ? s : __uint_as_float(0x7FC00000u)};
  return {__uint_as_float((b & 0x007FFFFFu) | 0x3F800000u), __uint_as_float(b & 0xFF800000u)};
}

// m dz = m dC d~ (rounded once to bf16) and, from the unrounded dz, the column sums of `kDzRows` rows in fp32:
// partial[blockIdx.y][column].  a_scale may be null: m = 1.
constexpr int kDzRows = 128;
__global__ void gelu_backward_dz(const __nv_bfloat16 *dC, const uint8_t *D, const float *a_scale, int M, int N,
                                 __nv_bfloat16 *dz, float *partial) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= N) return;
  const int r1 = min(M, static_cast<int>(blockIdx.y + 1) * kDzRows);
  float sum = 0.f;
  for (int r = blockIdx.y * kDzRows; r < r1; ++r) {
    const long long i = static_cast<long long>(r) * N + c;
    const float v = to_f32(dC[i]) * grad_value(D[i]);
    dz[i] = __float2bfloat16_rn(a_scale ? v * split_scale(a_scale[r]).m : v);
    sum += v;
  }
  partial[static_cast<long long>(blockIdx.y) * N + c] = sum;
}
// q 2^e in bf16, exact.
__global__ void input_of_codes(const int8_t *Q, const float *a_scale, int K, __nv_bfloat16 *X) {
  const long long r = blockIdx.x;
  const float e = split_scale(a_scale[r]).e;
  for (int c = threadIdx.x; c < K; c += blockDim.x) X[r * K + c] = __float2bfloat16_rn(static_cast<float>(Q[r * K + c]) * e);
}
// dbias: the partial column sums added in row order.
__global__ void sum_partials(const float *partial, int parts, int N, float *out) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= N) return;
  float sum = 0.f;
  for (int p = 0; p < parts; ++p) sum += partial[static_cast<long long>(p) * N + c];
  out[c] = sum;
}

}  // namespace pf

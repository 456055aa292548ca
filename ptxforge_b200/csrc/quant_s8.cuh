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

#include "sm100.cuh"

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

// The input's scale split into s = m 2^e, so that the backward pass rounds once where it could round twice: the
// tensor cores take q 2^e, which is exact in bf16 (7 bits), and round(m dz), whose product is q s dz; dA, which
// has no use for m, is divided by it at the end.  1/2 <= m < 1, so a token of tiny or no input keeps its dA, and m dz is
// finite where dz is; but 1 <= m < 2 from 2^121 on (inputs past 3.376e38), where 127 2^e would not be finite otherwise.  A
// scale that is not finite goes to e alone: dB is NaN then, dA is not.
struct SplitScale {
  float m, e;
};
__device__ __forceinline__ SplitScale split_scale(float s) {
  const uint32_t b = __float_as_uint(s), field = b & 0x7F800000u;
  if (field == 0u || field == 0x7F800000u) return {1.f, field == 0u ? s : __uint_as_float(0x7FC00000u)};
  const bool below = field < (121u + 127u) << 23;
  return {__uint_as_float((b & 0x007FFFFFu) | (below ? 0x3F000000u : 0x3F800000u)),
          __uint_as_float((b & 0xFF800000u) + (below ? 1u << 23 : 0u))};
}

// The whole numbers that four codes in a word stand for: grad codes code - 26 (NaN for 255) in steps of 1 or of 1 / 256,
// or int8 codes.  A byte put under the exponent of 2^23 is the float 2^23 + byte, under that of 2^15 2^15 + byte / 256.
constexpr float kGradUnit = 1.f / 256;
template <bool kInUnits = false>
__device__ __forceinline__ void grad_steps4(uint32_t w, float (&k)[4]) {
  constexpr float UNIT = kInUnits ? kGradUnit : 1.f;
  constexpr uint32_t BASE = kInUnits ? 0x47000000u : 0x4B000000u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = __byte_perm(w, BASE, 0x7650 | j);
    k[j] = b == (BASE | kGradNan) ? __uint_as_float(0x7FC00000u) : __uint_as_float(b) - (8388608.f + kGradZero) * UNIT;
  }
}
__device__ __forceinline__ void codes4(uint32_t w, float (&q)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    q[j] = __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4B000000u, 0x7650 | j)) - (8388608.f + 128.f);
}
// k / 200 rounded once, for every k of a code: a product by 1 / 200 and one correction by what it leaves.
__device__ __forceinline__ float grad_value(float k) {
  const float q = k * (1.f / kGradSteps);
  return fmaf(fmaf(-kGradSteps, q, k), 1.f / kGradSteps, q);
}

// ------------------------------------------------------------------------------------------------
// vectors of kVec values of a row: 16 bytes of them at once, or one
// ------------------------------------------------------------------------------------------------
template <int kBytes>
struct Word;
template <>
struct Word<1> { typedef uint8_t type; };
template <>
struct Word<2> { typedef uint16_t type; };
template <>
struct Word<4> { typedef uint32_t type; };
template <>
struct Word<8> { typedef uint2 type; };
template <>
struct Word<16> { typedef uint4 type; };

template <class T, int kVec>
struct Values {
  typename Word<sizeof(T) * kVec>::type w;
  __device__ __forceinline__ void load(const T *p) { w = *reinterpret_cast<const typename Word<sizeof(T) * kVec>::type *>(p); }
  __device__ __forceinline__ float operator[](int j) const { return to_f32(reinterpret_cast<const T *>(&w)[j]); }
};

// Largest |x| of vectors, NaN where there is one; eight bf16 values go two to an instruction.
template <class T, int kVec>
struct Largest {
  uint32_t m = 0;
  __device__ __forceinline__ void take(const Values<T, kVec> &x) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) m = max(m, abs_bits(x[j]));
  }
  __device__ __forceinline__ uint32_t bits() const { return m; }
};
template <>
struct Largest<__nv_bfloat16, 8> {
  __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
  __device__ __forceinline__ void take(const Values<__nv_bfloat16, 8> &x) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&x.w);
#pragma unroll
    for (int j = 0; j < 4; ++j) m = __hmax2_nan(m, __habs2(p[j]));
  }
  __device__ __forceinline__ uint32_t bits() const {
    return max(abs_bits(__low2float(m)), abs_bits(__high2float(m)));
  }
};

// The same, a column each.
template <class T, int kVec>
struct ColumnLargest {
  uint32_t m[kVec] = {};
  __device__ __forceinline__ void take(const Values<T, kVec> &x) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) m[j] = max(m[j], abs_bits(x[j]));
  }
  __device__ __forceinline__ uint32_t bits(int j) const { return m[j]; }
};
template <>
struct ColumnLargest<__nv_bfloat16, 8> {
  __nv_bfloat162 m[4];
  __device__ __forceinline__ ColumnLargest() {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = __floats2bfloat162_rn(0.f, 0.f);
  }
  __device__ __forceinline__ void take(const Values<__nv_bfloat16, 8> &x) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&x.w);
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = __hmax2_nan(m[j], __habs2(p[j]));
  }
  __device__ __forceinline__ uint32_t bits(int j) const {
    return abs_bits(j & 1 ? __high2float(m[j / 2]) : __low2float(m[j / 2]));
  }
};

// Codes of kVec values with the scales s[j] (one for all where kOne).  1.5 2^23 + x / s holds the code in its low byte,
// rounded to the nearest whole number by the addition; vectors with a value near a half step are done again by
// code_of, as are those with a scale that is NaN (`bad`), whose codes are 0.
template <class T, int kVec, bool kOne>
__device__ __forceinline__ void store_codes(const Values<T, kVec> &x, const float *s, const float *inv, bool bad, int8_t *q) {
  constexpr float magic = 12582912.f;
  uint32_t r[kVec];
  float far = 0.f;
  if constexpr (kVec == 1) {
    const float t = x[0] * inv[0], y = t + magic;
    far = fabsf(t - (y - magic));
    r[0] = __float_as_uint(y);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; j += 2) {
      const float2 i2 = kOne ? make_float2(inv[0], inv[0]) : make_float2(inv[j], inv[j + 1]);
      const float2 t = __fmul2_rn(make_float2(x[j], x[j + 1]), i2);
      const float2 y = __fadd2_rn(t, make_float2(magic, magic));
      const float2 n = __fadd2_rn(make_float2(magic, magic), make_float2(-y.x, -y.y));  // minus the whole number
      const float2 d = __fadd2_rn(t, n);
      far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
      r[j] = __float_as_uint(y.x);
      r[j + 1] = __float_as_uint(y.y);
    }
  }
  if (bad || far > 0.5f - 3e-5f) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) r[j] = static_cast<uint32_t>(code_of(x[j], s[kOne ? 0 : j], inv[kOne ? 0 : j]));
  }
  if constexpr (kVec == 1) {
    *q = static_cast<int8_t>(r[0]);
  } else {
    uint32_t w[kVec / 4];
#pragma unroll
    for (int j = 0; j < kVec; j += 4)
      w[j / 4] = __byte_perm(__byte_perm(r[j], r[j + 1], 0x0040), __byte_perm(r[j + 2], r[j + 3], 0x0040), 0x5410);
    if constexpr (kVec == 4) *reinterpret_cast<uint32_t *>(q) = w[0];
    else *reinterpret_cast<uint2 *>(q) = make_uint2(w[0], w[1]);
  }
}

// ------------------------------------------------------------------------------------------------
// a scale for each row
// ------------------------------------------------------------------------------------------------
// blockDim.x threads a row and blockDim.y rows a block (a warp's 32 threads where there are several), kHeld vectors a
// thread held in registers: one pass over X.  What a longer row has beyond them is read again (from L2).
template <class T, int kVec, int kHeld>
__global__ void __launch_bounds__(512) quantize_rows_s8(const T *X, long long ldx, int rows, int cols, int8_t *Q,
                                                        long long ldq, float *scale) {
  __shared__ uint32_t sh[16];
  grid_launch_dependents();
  grid_dependency_wait();
  const long long r = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (r >= rows) return;  // whole warps: blockDim.y > 1 only with a warp a row
  const T *x = X + r * ldx;
  const int vecs = cols / kVec, step = blockDim.x;
  Values<T, kVec> held[kHeld];
  Largest<T, kVec> largest;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int v = threadIdx.x + i * step;
    if (v < vecs) held[i].load(x + static_cast<long long>(v) * kVec);
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (static_cast<int>(threadIdx.x) + i * step < vecs) largest.take(held[i]);
  for (int v = threadIdx.x + kHeld * step; v < vecs; v += step) {
    Values<T, kVec> y;
    y.load(x + static_cast<long long>(v) * kVec);
    largest.take(y);
  }
  uint32_t m = __reduce_max_sync(0xffffffffu, largest.bits());
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) m = max(m, sh[w]);
  }
  const float s = scale_of(m), inv = __fdiv_rn(1.f, s);
  int8_t *q = Q + r * ldq;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int v = threadIdx.x + i * step;
    if (v < vecs) store_codes<T, kVec, true>(held[i], &s, &inv, s != s, q + static_cast<long long>(v) * kVec);
  }
  for (int v = threadIdx.x + kHeld * step; v < vecs; v += step) {
    Values<T, kVec> y;
    y.load(x + static_cast<long long>(v) * kVec);
    store_codes<T, kVec, true>(y, &s, &inv, s != s, q + static_cast<long long>(v) * kVec);
  }
  if (threadIdx.x == 0) scale[r] = s;
}

// ------------------------------------------------------------------------------------------------
// a scale for each column
// ------------------------------------------------------------------------------------------------
// Up to 4096 aligned rows: a cluster takes a strip of 128 bytes of columns, each of its CTAs a share of the rows, which
// comes to shared memory by TMA, all boxes on their way at once, and stays there: one pass over X.  The column maxima are
// joined through distributed shared memory.
constexpr int kColBox = 64, kColMostBoxes = 8, kColMostRows = 8 * kColBox * kColMostBoxes;
template <class T>
__global__ void __launch_bounds__(256, 3) quantize_strips_s8(const __grid_constant__ CUtensorMap map, int rows, int cols,
                                                             int8_t *Q, long long ldq, float *scale, unsigned *status,
                                                             unsigned long long timeout_ns) {
  constexpr int kVec = 16 / sizeof(T), W = 128 / sizeof(T), LANES = W / kVec, STEP = 256 / LANES;  // LANES = 8, STEP = 32
  typedef Values<T, kVec> Vec;
  extern __shared__ uint8_t smem_raw[];
  T *slab = reinterpret_cast<T *>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
  __shared__ uint32_t amax[W];
  __shared__ float scales[2][W];
  __shared__ uint64_t full[kColMostBoxes];
  __shared__ int abort_word;
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
  const int rank = static_cast<int>(cluster_ctarank());
  const int r0 = rows * rank / static_cast<int>(splits), n = rows * (rank + 1) / static_cast<int>(splits) - r0;
  const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES;
  const int c0 = static_cast<int>(blockIdx.x / splits) * W, c = c0 + lane * kVec;
  const int boxes = (n + kColBox - 1) / kColBox;
  grid_launch_dependents();
  if (threadIdx.x < W) amax[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map);
    for (int b = 0; b < boxes; ++b) mbar_init(&full[b], 1);
    abort_word = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  grid_dependency_wait();
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int b = 0; b < boxes; ++b) {
      mbar_arrive_expect_tx(&full[b], kColBox * 128);
      tma_load_2d(slab + b * kColBox * W, &map, &full[b], c0, r0 + b * kColBox);
    }
  }
  ColumnLargest<T, kVec> largest;
  for (int b = 0; b < boxes; ++b) {
    if (!mbar_wait(&full[b], 0, timeout_ns, &abort_word)) {
      atomicOr(status, 1u);
      abort_word = 1;
    }
#pragma unroll
    for (int k = 0; k < kColBox / STEP; ++k) {
      const int r = b * kColBox + k * STEP + first;
      Vec y;
      y.load(slab + r * W + lane * kVec);
      if (r < n) largest.take(y);
    }
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    // the lanes of a warp that hold the same columns first, then one of them for the warp
    uint32_t m = largest.bits(j);
#pragma unroll
    for (int d = LANES; d < 32; d *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) < LANES) atomicMax(&amax[lane * kVec + j], m);
  }
  __syncwarp();
  cluster_sync();
  // a thread a column: every CTA's maximum, all loads on their way at once
  if (threadIdx.x < W) {
    uint32_t all = 0;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k)
      if (k < splits) all = max(all, ld_cluster(mapa_shared(smem_u32(&amax[threadIdx.x]), k)));
    const float s = scale_of(all);
    scales[0][threadIdx.x] = s;
    scales[1][threadIdx.x] = __fdiv_rn(1.f, s);
    if (rank == 0 && c0 + static_cast<int>(threadIdx.x) < cols) scale[c0 + threadIdx.x] = s;
  }
  __syncthreads();
  cluster_arrive_relaxed();  // the others' maxima were read
  if (c < cols) {  // whole vectors: cols is a multiple of kVec
    float s[kVec], inv[kVec];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      s[j] = scales[0][lane * kVec + j], inv[j] = scales[1][lane * kVec + j];
      bad |= s[j] != s[j];
    }
    int8_t *q = Q + r0 * ldq + c;
#pragma unroll 4
    for (int r = first; r < n; r += STEP) {
      Vec y;
      y.load(slab + r * W + lane * kVec);
      store_codes<T, kVec, false>(y, s, inv, bad, q + r * ldq);
    }
  }
  __syncwarp();
  cluster_wait();  // nobody leaves while its maxima may be read
}

// Any matrix, two passes: 32 vectors of columns x kColRows rows a block.  First the largest abs_bits of each column into
// `scale` (zeroed before; a maximum of bits does not depend on the order), then the codes, then the scales over the bits.
constexpr int kColRows = 128;
template <class T, int kVec>
__global__ void __launch_bounds__(256) amax_cols_s8(const T *X, long long ldx, int rows, int cols, int col_blocks, uint32_t *amax) {
  __shared__ uint32_t sh[8][32 * kVec];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int rb = blockIdx.x / col_blocks, c0 = (blockIdx.x - rb * col_blocks) * 32 * kVec, c = c0 + lane * kVec;
  const int r1 = min(static_cast<long long>(rows), (rb + 1ll) * kColRows);
  ColumnLargest<T, kVec> largest;
  if (c < cols) {
#pragma unroll 8
    for (int r = rb * kColRows + row; r < r1; r += 8) {
      Values<T, kVec> y;
      y.load(X + r * ldx + c);
      largest.take(y);
    }
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) sh[row][lane * kVec + j] = largest.bits(j);
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * kVec; i += 256)
    if (c0 + i < cols) {
      uint32_t all = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) all = max(all, sh[k][i]);
      atomicMax(amax + c0 + i, all);
    }
}
template <class T, int kVec>
__global__ void __launch_bounds__(256) codes_cols_s8(const T *X, long long ldx, int rows, int cols, int col_blocks,
                                                     const uint32_t *amax, int8_t *Q, long long ldq) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int rb = blockIdx.x / col_blocks, c = ((blockIdx.x - rb * col_blocks) * 32 + lane) * kVec;
  if (c >= cols) return;
  const int r1 = min(static_cast<long long>(rows), (rb + 1ll) * kColRows);
  float s[kVec], inv[kVec];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    s[j] = scale_of(amax[c + j]), inv[j] = __fdiv_rn(1.f, s[j]);
    bad |= s[j] != s[j];
  }
#pragma unroll 4
  for (int r = rb * kColRows + row; r < r1; r += 8) {
    Values<T, kVec> y;
    y.load(X + r * ldx + c);
    store_codes<T, kVec, false>(y, s, inv, bad, Q + r * ldq + c);
  }
}
// Scales of rows (columns) that hold nothing.
__global__ void __launch_bounds__(256) least_scales(float *scale, int n) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) scale[i] = kLeastScale;
}
__global__ void __launch_bounds__(256) scales_of_bits(uint32_t *amax, int n) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) amax[i] = __float_as_uint(scale_of(amax[i]));
}

// ------------------------------------------------------------------------------------------------
// back from codes
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void store_vec(__nv_bfloat16 *out, const float (&x)[8]) {
  *reinterpret_cast<uint4 *>(out) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                               pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void store_vec(float *out, const float (&x)[4]) {
  *reinterpret_cast<float4 *>(out) = make_float4(x[0], x[1], x[2], x[3]);
}
// What the codes of one vector stand for, by codes4 or grad_steps4.
template <int kVec, class Four>
__device__ __forceinline__ void load_codes(const void *p, float (&q)[kVec], Four four) {
  typename Word<kVec>::type w = *reinterpret_cast<const typename Word<kVec>::type *>(p);
  const uint32_t *words = reinterpret_cast<const uint32_t *>(&w);
#pragma unroll
  for (int i = 0; i < kVec / 4; ++i) {
    float a[4];
    four(words[i], a);
#pragma unroll
    for (int j = 0; j < 4; ++j) q[i * 4 + j] = a[j];
  }
}

// Scale of a row or of the columns; kInput: the part 2^e of a row's (split_scale), which keeps the values exact in bf16.
// kVec: 16 bytes of values, or 1.  blockDim.x threads a row, blockDim.y rows a block.
template <class T, int kVec, bool kByRow, bool kInput = false>
__device__ __forceinline__ void restore_row(const int8_t *q, int cols, const float *scale, T *x, int first, int step) {
  float s = kByRow ? *scale : 0.f;
  if constexpr (kInput) s = split_scale(s).e;
  if constexpr (kVec > 1) {
#pragma unroll 4
    for (int c = first * kVec; c < cols; c += step * kVec) {
      float v[kVec];
      load_codes(q + c, v, [](uint32_t w, float (&a)[4]) { codes4(w, a); });
      if constexpr (kByRow) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] *= s;
      } else if ((reinterpret_cast<uintptr_t>(scale) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < kVec; j += 4) {
          const float4 a = *reinterpret_cast<const float4 *>(scale + c + j);
          v[j] *= a.x, v[j + 1] *= a.y, v[j + 2] *= a.z, v[j + 3] *= a.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] *= scale[c + j];
      }
      store_vec(x + c, v);
    }
  } else {
    for (int c = first; c < cols; c += step) x[c] = from_f32<T>(static_cast<float>(q[c]) * (kByRow ? s : scale[c]));
  }
}
template <class T, int kVec, bool kByRow>
__global__ void __launch_bounds__(256) dequantize_s8(const int8_t *Q, long long ldq, int rows, int cols, const float *scale,
                                                     T *X, long long ldx) {
  grid_launch_dependents();
  grid_dependency_wait();
  const long long r = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (r < rows) restore_row<T, kVec, kByRow>(Q + r * ldq, cols, kByRow ? scale + r : scale, X + r * ldx, threadIdx.x, blockDim.x);
}

// kGradAhead vectors a thread, all on their way at once.
template <class T, int kVec, int kGradAhead>
__global__ void __launch_bounds__(256) dequantize_grad(const uint8_t *D, long long n, T *X) {
  grid_launch_dependents();
  grid_dependency_wait();
  const long long stride = static_cast<long long>(gridDim.x) * 256 * kVec * kGradAhead;
  for (long long base = blockIdx.x * (256ll * kVec * kGradAhead) + threadIdx.x * kVec; base < n; base += stride) {
    if constexpr (kVec > 1) {
      if (base + (kGradAhead - 1) * 256ll * kVec + kVec <= n) {
        float v[kGradAhead][kVec];
#pragma unroll
        for (int b = 0; b < kGradAhead; ++b)
          load_codes(D + base + b * 256 * kVec, v[b], [](uint32_t w, float (&a)[4]) { grad_steps4(w, a); });
#pragma unroll
        for (int b = 0; b < kGradAhead; ++b) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) v[b][j] = grad_value(v[b][j]);
          store_vec(X + base + b * 256 * kVec, v[b]);
        }
        continue;
      }
    }
    for (int b = 0; b < kGradAhead; ++b) {
      const long long i = base + b * 256 * kVec;
      for (long long j = i; j < n && j < i + kVec; ++j) {
        float k[4];
        grad_steps4(D[j], k);
        X[j] = from_f32<T>(grad_value(k[0]));
      }
    }
  }
}

// Rows of bytes that start anywhere -> rows of whole 16-byte words.  Each word is put together from the aligned
// 4-byte words that hold its bytes; a word with no byte of the row is not read.  What follows a row's end is whatever
// shares its last word, and is never used.
// One launch for two matrices: a block a row, the first rows_a of them of `a`.
struct AlignRows {
  const uint8_t *X;
  long long ld;
  int cols;
  uint4 *Y;
  long long ld_y;
};
__global__ void __launch_bounds__(128) align_rows(const AlignRows a, const AlignRows b, int rows_a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const bool second = static_cast<int>(blockIdx.x) >= rows_a;
  const uint8_t *X = second ? b.X : a.X;
  uint4 *Y = second ? b.Y : a.Y;
  const long long ld = second ? b.ld : a.ld, ld_y = second ? b.ld_y : a.ld_y;
  const long long r = static_cast<int>(blockIdx.x) - (second ? rows_a : 0);
  const int cols = second ? b.cols : a.cols;
  const uintptr_t row = reinterpret_cast<uintptr_t>(X + r * ld);
  const unsigned shift = 8 * static_cast<unsigned>(row & 3);
  const uint32_t *x = reinterpret_cast<const uint32_t *>(row & ~uintptr_t(3));
  const int words = static_cast<int>((cols + (row & 3) + 3) / 4);
  for (int i = threadIdx.x; i * 16 < cols; i += blockDim.x) {
    uint32_t v[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] = i * 4 + j < words ? x[i * 4 + j] : 0u;
    Y[r * ld_y + i] = make_uint4(__funnelshift_r(v[0], v[1], shift), __funnelshift_r(v[1], v[2], shift),
                                 __funnelshift_r(v[2], v[3], shift), __funnelshift_r(v[3], v[4], shift));
  }
}

// ------------------------------------------------------------------------------------------------
// the backward pass's elementwise part
// ------------------------------------------------------------------------------------------------
// Blocks below dz_blocks: m dz = m dC d~ (rounded once to bf16) of 256 columns x dz_rows rows and, from the unrounded dz,
// their column sums in fp32 (`sums` [row block][column]; with one row block that is dbias).  dC k / 256 is exact in fp32 (8
// by 8 bits) and finite where dC is, which dC k is not; so dz is rounded once, by 256 / 200.  The blocks after them: the
// input's q 2^e in bf16, exact, a row each.  a_scale may be null (m = 1, no input wanted).
constexpr int kDzCols = 256;
__global__ void __launch_bounds__(256) backward_operands(const __nv_bfloat16 *dC, const uint8_t *D, const float *a_scale,
                                                         int M, int N, int dz_blocks, int col_blocks, int dz_rows,
                                                         __nv_bfloat16 *dz,
                                                         float *sums, const int8_t *Q, int K, __nv_bfloat16 *input) {
  __shared__ float sh[8][kDzCols];
  grid_launch_dependents();
  grid_dependency_wait();
  if (static_cast<int>(blockIdx.x) >= dz_blocks) {
    const long long r = blockIdx.x - dz_blocks;
    restore_row<__nv_bfloat16, 8, true, true>(Q + r * K, K, a_scale + r, input + r * K, threadIdx.x, 256);
    return;
  }
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int rb = blockIdx.x / col_blocks;
  const int c = (blockIdx.x - rb * col_blocks) * kDzCols + lane * 8;
  float sum[8] = {};
  if (c < N) {
    const int r0 = rb * dz_rows + row, r1 = min(M, (rb + 1) * dz_rows);
    for (int r = r0; r < r1; r += 32) {
      // four rows on their way at once, the last ones too
      uint4 g[4];
      uint2 w[4];
      float m[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (r + b * 8 >= r1) break;
        const long long i = static_cast<long long>(r + b * 8) * N + c;
        g[b] = *reinterpret_cast<const uint4 *>(dC + i);
        w[b] = *reinterpret_cast<const uint2 *>(D + i);
        m[b] = a_scale ? a_scale[r + b * 8] : 1.f;
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (r + b * 8 >= r1) break;
        float k[8], v[8];
        load_codes(&w[b], k, [](uint32_t x, float (&a)[4]) { grad_steps4<true>(x, a); });
        const float f = a_scale ? split_scale(m[b]).m : 1.f;
        const uint32_t gw[4] = {g[b].x, g[b].y, g[b].z, g[b].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = __uint_as_float((j & 1) ? gw[j / 2] & 0xFFFF0000u : gw[j / 2] << 16);
          const float z = x * k[j] * (1.f / kGradUnit / kGradSteps);
          sum[j] += z;
          v[j] = z * f;
        }
        store_vec(dz + static_cast<long long>(r + b * 8) * N + c, v);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[row][lane * 8 + j] = sum[j];
  __syncthreads();
  const int col = (blockIdx.x - rb * col_blocks) * kDzCols + threadIdx.x;
  if (col < N) {
    float total = sh[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 8; ++i) total += sh[i][threadIdx.x];
    sums[static_cast<long long>(rb) * N + col] = total;
  }
}

// dbias: the row blocks' sums added, eight runs of them side by side, then the runs in order.
__global__ void __launch_bounds__(256) sum_row_blocks(const float *sums, int blocks, int N, float *out) {
  __shared__ float sh[8][32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < N) {
#pragma unroll 8
    for (int b = run; b < blocks; b += 8) sum += sums[static_cast<long long>(b) * N + c];
  }
  sh[run][lane] = sum;
  __syncthreads();
  if (run == 0 && c < N) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += sh[i][lane];
    out[c] = sum;
  }
}

}  // namespace pf

// gemm8_simple.cuh -- the products of the 8-bit operators on the CUDA cores: 64 x 64 tiles through shared memory,
// 4 x 4 outputs a thread, any sizes, strides and alignment.
#pragma once

#include "ops8_epilogue.cuh"

namespace pf {

// A(i, k) = A[i * a_row + k * a_k], B(k, j) = B[k * b_k + j * b_col].
template <class T>
struct Strided {
  const T *A, *B;
  long long a_row, a_k, b_k, b_col;
};

__device__ __forceinline__ int mac(int8_t a, int8_t b, int c) { return c + static_cast<int>(a) * static_cast<int>(b); }
__device__ __forceinline__ float mac(__nv_bfloat16 a, __nv_bfloat16 b, float c) { return fmaf(to_f32(a), to_f32(b), c); }

struct StoreS8 {
  const float *sa, *sb, *bias;
  int gelu, out_f32;
  void *C;
  long long ldc;
  __device__ __forceinline__ void operator()(int r, int c, int acc) const {
    float x = static_cast<float>(acc) * (sa[r] * sb[c]);
    if (bias) x += bias[c];
    if (gelu) x = gelu_of(x);
    const long long i = r * ldc + c;
    if (out_f32) static_cast<float *>(C)[i] = x;
    else static_cast<__nv_bfloat16 *>(C)[i] = __float2bfloat16_rn(x);
  }
};
struct StoreCheckpoint {
  const float *bias;
  __nv_bfloat16 *C;
  uint8_t *D;
  long long ld;
  __device__ __forceinline__ void operator()(int r, int c, float acc) const {
    const Gelu g = gelu_and_grad(acc + bias[c]);
    C[r * ld + c] = __float2bfloat16_rn(g.y);
    D[r * ld + c] = static_cast<uint8_t>(grad_code(g.d));
  }
};
struct StoreBf16 {
  const float *row_scale;  // null, or rows are divided by its m (split_scale)
  __nv_bfloat16 *C;
  long long ld;
  __device__ __forceinline__ void operator()(int r, int c, float acc) const {
    C[r * ld + c] = __float2bfloat16_rn(row_scale ? __fdiv_rn(acc, split_scale(row_scale[r]).m) : acc);
  }
};

template <class T, class Acc, class Store>
__global__ void __launch_bounds__(256) gemm8_simple(Strided<T> g, int M, int N, int K, Store store) {
  __shared__ T a[16][64 + 4 / sizeof(T)], b[16][64 + 4 / sizeof(T)];
  const long long m0 = static_cast<long long>(blockIdx.x) * 64, n0 = static_cast<long long>(blockIdx.y) * 64;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  Acc acc[4][4] = {};
  for (long long k0 = 0; k0 < K; k0 += 16) {
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int kk = i >> 6, j = i & 63;
      const long long k = k0 + kk;
      a[kk][j] = k < K && m0 + j < M ? g.A[(m0 + j) * g.a_row + k * g.a_k] : T(0);
      b[kk][j] = k < K && n0 + j < N ? g.B[k * g.b_k + (n0 + j) * g.b_col] : T(0);
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mac(a[kk][ty * 4 + i], b[kk][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const long long r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
      if (r < M && c < N) store(static_cast<int>(r), static_cast<int>(c), acc[i][j]);
    }
}

}  // namespace pf

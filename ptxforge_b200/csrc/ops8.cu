// ops8.cu -- the 8-bit operators of the C ABI (include/pf_b200.h): int8 store and restore, the int8 product with
// token and channel scales, the fused product with an 8-bit checkpoint, and its gradients.
//
// None needs a pf_ctx: operands and workspaces are the caller's, every launch goes on the caller's stream, nothing is
// allocated and nothing is kept from one call for the next but each device's properties.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <type_traits>

#include "pf_b200.h"
#include "gemm8_tc.cuh"
#include "host_util.cuh"
#include "ops8_epilogue.cuh"
#include "selftest.cuh"

// Bounded waits that ran out, of every kernel here: bits are only ever set, until pf_ops8_status clears those that it has
// read, so calls that overlap on the GPU, and with that, may share it.
static __device__ unsigned ops8_status_word;

namespace {

__global__ void clear_bits(unsigned *word, unsigned bits) { atomicAnd(word, ~bits); }

using pf::DeviceGuard;
typedef __nv_bfloat16 bf16;

constexpr int kMaxDevices = 64;
constexpr int kMostSize = 1 << 30;  // rows, columns, M, N, K: index arithmetic in 32 bits stays below 2^31
constexpr unsigned long long kWaitNs = 4000000000ull;  // bound of each device-side wait
constexpr int kMaxSumK = 131071;  // K * 128 * 128 stays below 2^31

// A device's properties and, for each tensor-core kernel that it has launched, the CTA pairs that fit at once (its
// shared-memory limit raised before).
struct KernelUnits {
  const void *func;
  int units;
};
struct Device {
  std::mutex mu;
  bool ready = false;
  int cc_major = 0, num_sms = 0;
  unsigned *status = nullptr;
  KernelUnits kernels[48];
  int n_kernels = 0;
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
  if (device < 0 || device >= kMaxDevices) return err(PF_ENODEV, "no CUDA device %d", device);
  Device &d = g_devices[device];
  std::lock_guard<std::mutex> lk(d.mu);
  if (!d.ready) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || device >= n) {
      cudaGetLastError();
      return err(PF_ENODEV, "no CUDA device %d", device);
    }
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

// Raises a kernel's shared-memory limit and, for a pair kernel, counts the pairs that fit on the device at once.
int kernel_units(Device &d, const void *func, int smem, int pair_threads, const Err &err, int *units) {
  std::lock_guard<std::mutex> lk(d.mu);
  for (int i = 0; i < d.n_kernels; ++i)
    if (d.kernels[i].func == func) {
      *units = d.kernels[i].units;
      return PF_OK;
    }
  cudaError_t e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int u = 0;
  if (e == cudaSuccess && pair_threads) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(2 * (d.num_sms / 2));
    cfg.blockDim = dim3(pair_threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&u, func, &cfg);
    if (e == cudaSuccess && u <= 0) e = cudaErrorLaunchOutOfResources;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return err(PF_ECUDA, "kernel set-up: %s", cudaGetErrorString(e));
  }
  if (d.n_kernels < static_cast<int>(sizeof d.kernels / sizeof d.kernels[0])) d.kernels[d.n_kernels++] = {func, u};
  *units = u;
  return PF_OK;
}

// Whether rows of `cols` values of `size` bytes, `ld` apart, can be read and written `vec` values at a time.
bool vectors_fit(const void *x, long long ld, int cols, int size, int vec) {
  return reinterpret_cast<uintptr_t>(x) % (size * vec) == 0 && ld % vec == 0 && cols % vec == 0;
}

template <class T, int kVec>
void quantize_rows(const T *x, long long ldx, int rows, int cols, int8_t *q, long long ldq, float *scale, cudaStream_t s) {
  // Many rows: a warp each where its registers hold the row, else a block each, eight vectors a thread -- much in flight
  // and few threads to join.  Few rows: as many threads a row as it can use, so that a lone one is spread over an SM.
  // Measured, us: 16384 x 4096 bf16 with 2 vectors a thread 52, with 8 43; 65536 x 512 fp32 with 2 and a block a row 69,
  // with 4 and a warp a row 26.  To both sides of 1,024 rows, many / few, X in L2: fp32 4096 columns, 512 rows 3.4 / 3.3, 1,024
  // 3.8 / 4.0, 4,096 10.1 / 11.8; 14336 columns the same within 2 %; bf16 4096 columns 7.8 / 4.2, 8.5 / 5.1, 14.5 / 12.6, so there
  // `few` would do up to some thousand rows.
  const int vecs = (cols + kVec - 1) / kVec;
  const auto launch = [&](auto kernel, dim3 block) {
    pf::launch_pdl(kernel, dim3(blocks_of(rows, block.y)), block, 0, s, x, ldx, rows, cols, q, ldq, scale);
  };
  const auto threads = [&](int held) { return dim3(std::min(512, (vecs + 32 * held - 1) / (32 * held) * 32)); };
  if (vecs <= 64) return launch(&pf::quantize_rows_s8<T, kVec, 2>, dim3(32, 8));
  if (rows >= 1024) {
    if (vecs <= 128) return launch(&pf::quantize_rows_s8<T, kVec, 4>, dim3(32, 8));
    return launch(&pf::quantize_rows_s8<T, kVec, 8>, vecs <= 256 ? dim3(32, 8) : threads(8));
  }
  if (vecs <= 512) return launch(&pf::quantize_rows_s8<T, kVec, 2>, threads(2));
  if (vecs <= 1024) return launch(&pf::quantize_rows_s8<T, kVec, 4>, threads(4));
  launch(&pf::quantize_rows_s8<T, kVec, 8>, threads(8));
}

// Strips of whole columns held in shared memory: 512 rows of 128 bytes a CTA, so that three CTAs share an SM, one's loads
// beside another's stores.  What bounds it is the chain of a CTA (load, maximum, exchange, codes), times how often the SMs are
// filled with CTAs: 4096 x 14336 in bf16 fills them 1.56 times, so twice, 69 us; in fp32 3.11 times, so four times, 78 us.  DRAM is
// busy for 26 and 43 %, L2 for 17 and 30 %, issue for 40 and 32 %.  fp32 with 256 rows a CTA in clusters of 16: 5 % more.
template <class T>
int quantize_strips(Device &d, const T *x, long long ldx, int rows, int cols, int8_t *q, long long ldq, float *scale,
                    cudaStream_t s, const Err &err) {
  constexpr int kRowBytes = 128, kPerCta = pf::kColBox * pf::kColMostBoxes;
  int splits = 1;
  while (rows > kPerCta * splits) splits *= 2;
  const int held = ((rows + splits - 1) / splits + pf::kColBox - 1) / pf::kColBox * pf::kColBox;
  const void *func = reinterpret_cast<const void *>(&pf::quantize_strips_s8<T>);
  int rc, units;
  if ((rc = kernel_units(d, func, 128 + kPerCta * kRowBytes, 0, err, &units))) return rc;
  CUtensorMap map;
  char msg[200];
  if (pf::encode_2d_msg(msg, sizeof msg, &map, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, x,
                        cols, rows, ldx * sizeof(T), kRowBytes / sizeof(T), pf::kColBox, CU_TENSOR_MAP_SWIZZLE_NONE))
    return err(PF_ECUDA, "%s", msg);
  pf::launch_cluster(&pf::quantize_strips_s8<T>, dim3(blocks_of(static_cast<long long>(cols) * sizeof(T), kRowBytes) * splits),
                     dim3(256), 128 + held * kRowBytes, splits, s, map, rows, cols, q, ldq, scale, d.status, kWaitNs);
  return PF_OK;
}

template <class T, int kVec>
int quantize_cols(const T *x, long long ldx, int rows, int cols, int8_t *q, long long ldq, float *scale, cudaStream_t s,
                  const Err &err) {
  uint32_t *amax = reinterpret_cast<uint32_t *>(scale);
  const cudaError_t e = cudaMemsetAsync(amax, 0, size_t(cols) * sizeof(float), s);
  if (e != cudaSuccess) return err(PF_ECUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
  const int col_blocks = static_cast<int>(blocks_of(cols, 32 * kVec));
  const long long blocks = static_cast<long long>(col_blocks) * blocks_of(rows, pf::kColRows);
  if (blocks > 0x7FFFFFFF) return err(PF_EINVAL, "more than 2^31 blocks");
  const dim3 grid(static_cast<unsigned>(blocks));
  pf::launch_pdl(&pf::amax_cols_s8<T, kVec>, grid, 256, 0, s, x, ldx, rows, cols, col_blocks, amax);
  pf::launch_pdl(&pf::codes_cols_s8<T, kVec>, grid, 256, 0, s, x, ldx, rows, cols, col_blocks, static_cast<const uint32_t *>(amax),
                 q, ldq);
  pf::launch_pdl(&pf::scales_of_bits, dim3(blocks_of(cols, 256)), 256, 0, s, amax, cols);
  return PF_OK;
}

template <class T>
int quantize(Device &d, const void *X, long long ldx, int rows, int cols, int axis, int8_t *Q, long long ldq, float *scale,
             cudaStream_t s, const Err &err) {
  constexpr int kVec = 16 / sizeof(T);
  const T *x = static_cast<const T *>(X);
  const bool wide = vectors_fit(X, ldx, cols, sizeof(T), kVec) && vectors_fit(Q, ldq, cols, 1, kVec);
  if (axis == 0) {
    if (wide && rows <= pf::kColMostRows) return quantize_strips<T>(d, x, ldx, rows, cols, Q, ldq, scale, s, err);
    return wide ? quantize_cols<T, kVec>(x, ldx, rows, cols, Q, ldq, scale, s, err)
                : quantize_cols<T, 1>(x, ldx, rows, cols, Q, ldq, scale, s, err);
  }
  if (wide) quantize_rows<T, kVec>(x, ldx, rows, cols, Q, ldq, scale, s);
  else quantize_rows<T, 1>(x, ldx, rows, cols, Q, ldq, scale, s);
  return PF_OK;
}

template <class T, int kVec>
void dequantize(const int8_t *q, long long ldq, int rows, int cols, const float *scale, int axis, T *x, long long ldx,
                cudaStream_t s) {
  int across = 8;  // threads a row
  while (across < 256 && across * kVec < cols) across *= 2;
  const dim3 block(across, 256 / across);
  const auto kernel = axis ? &pf::dequantize_s8<T, kVec, true> : &pf::dequantize_s8<T, kVec, false>;
  pf::launch_pdl(kernel, dim3(blocks_of(rows, block.y)), block, 0, s, q, ldq, rows, cols, scale, x, ldx);
}
template <class T>
void dequantize(const int8_t *q, long long ldq, int rows, int cols, const float *scale, int axis, void *X, long long ldx,
                cudaStream_t s) {
  T *x = static_cast<T *>(X);
  constexpr int kVec = 16 / sizeof(T);
  if (vectors_fit(q, ldq, cols, 1, kVec) && vectors_fit(X, ldx, cols, sizeof(T), kVec))
    dequantize<T, kVec>(q, ldq, rows, cols, scale, axis, x, ldx, s);
  else dequantize<T, 1>(q, ldq, rows, cols, scale, axis, x, ldx, s);
}

template <class T>
void dequantize_grad(const unsigned char *codes, long long n, void *X, cudaStream_t s) {
  T *x = static_cast<T *>(X);
  constexpr int kVec = 16 / sizeof(T);
  const bool wide = reinterpret_cast<uintptr_t>(codes) % kVec == 0 && pf::aligned16(X);
  // Four vectors a thread where that leaves enough blocks (16384 x 14336 to bf16: 129 us with one, 105 with four), one below.
  const bool ahead = wide && n >= 1024ll * 256 * 4 * kVec;
  const int per = 256 * (wide ? kVec : 1) * (ahead ? 4 : 1);
  const dim3 grid(static_cast<unsigned>(std::min<long long>((n + per - 1) / per, 1 << 30)));
  const auto kernel = ahead ? &pf::dequantize_grad<T, kVec, 4> : wide ? &pf::dequantize_grad<T, kVec, 1> : &pf::dequantize_grad<T, 1, 1>;
  pf::launch_pdl(kernel, grid, 256, 0, s, codes, n, x);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// The parts of the backward pass's workspace, in order, each 256-byte aligned.
struct BackwardSpace {
  size_t dz, a, partial, total;
  int col_blocks, rows, parts;
  BackwardSpace(int M, int N, int K) {
    // 128 rows a block of the elementwise kernel (and a part of dbias' sums); 32 where that makes too few blocks to keep
    // the memory busy.  With the launch that joins the parts, 32 / 128 rows, us: 1999 x 2048 6.3 / 9.0, 4096 x 2048 7.6 / 9.8,
    // 8192 x 2048 14.6 / 12.9, 2048 x 8192 13.4 / 13.4, 4096 x 8192 29.9 / 28.7, 16384 x 2048 32.7 / 28.5 (from some 512 blocks on 128
    // rows are as good).  Up to 128 tokens are one part, which needs no launch to join parts (a backward pass of
    // 77 x 512 x 512 waits for its launches: 16.8 us with three parts, 14.4 with one).
    col_blocks = (N + pf::kDzCols - 1) / pf::kDzCols;
    rows = M > 128 && (M + 127) / 128 * static_cast<long long>(col_blocks) < 1024 ? 32 : 128;
    parts = (M + rows - 1) / rows;
    dz = 0;
    a = dz + round256(size_t(M) * N * sizeof(bf16));
    partial = a + round256(size_t(M) * K * sizeof(bf16));
    total = partial + round256(size_t(parts) * N * sizeof(float));
  }
};

// TMA wants rows that start on 16-byte boundaries.  A product's operand that has others is copied, row by row, to the
// workspace.
struct ProductSpace {
  bool copy_a, copy_b;
  long long lda, ldb;  // row strides that the tensor maps use
  size_t b, total;
  static bool fits(const void *x, long long ld, int rows) { return pf::aligned16(x) && (rows == 1 || ld % 16 == 0); }
  static long long round16(long long n) { return (n + 15) / 16 * 16; }
  ProductSpace(int M, int N, int K, const void *A, long long lda_, const void *B, long long ldb_) {
    copy_a = !fits(A, lda_, M);
    copy_b = !fits(B, ldb_, K);
    lda = copy_a || M == 1 ? round16(K) : lda_;
    ldb = copy_b || K == 1 ? round16(N) : ldb_;
    b = copy_a ? round256(size_t(M) * lda) : 0;
    total = b + (copy_b ? round256(size_t(K) * ldb) : 0);
  }
};

// One product: out[t][c] = sum_r T(t, r) W(r, c).  A K-major operand is [t][r] or [c][r], an MN-major one [r][t] or
// [r][c], with row strides ldt, ldw in elements.
struct Product {
  int tokens, channels, sum;
  const void *T, *W;
  long long ldt, ldw;
  // The part from channel c0, token t0 on.
  template <class Op>
  Product part(int c0, int t0) const {
    return {tokens - t0, channels - c0, sum,
            static_cast<const char *>(T) + (Op::T_K ? t0 * ldt : t0) * Op::ELEM,
            static_cast<const char *>(W) + (Op::W_K ? c0 * ldw : c0) * Op::ELEM, ldt, ldw};
  }
};

template <int kElem>
CUtensorMapDataType map_type() {
  return kElem == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
}

template <class Op>
int operand_maps(const Product &g, const Err &err, CUtensorMap *w, CUtensorMap *t) {
  constexpr int e = Op::ELEM;
  char msg[200];
  if (pf::encode_2d_msg(msg, sizeof msg, w, map_type<e>(), g.W, Op::W_K ? g.sum : g.channels,
                        Op::W_K ? g.channels : g.sum, g.ldw * e, Op::W_BOX0, Op::W_BOX1, CU_TENSOR_MAP_SWIZZLE_128B) ||
      pf::encode_2d_msg(msg, sizeof msg, t, map_type<e>(), g.T, Op::T_K ? g.sum : g.tokens, Op::T_K ? g.tokens : g.sum,
                        g.ldt * e, Op::T_BOX0, Op::T_BOX1, CU_TENSOR_MAP_SWIZZLE_128B))
    return err(PF_ECUDA, "%s", msg);
  return PF_OK;
}

constexpr int kSmemPerSm = 227 * 1024;  // of one SM, for the CTAs that share it
constexpr int kOneStatic = 3 * 1024;    // of gemm8_one: barriers and token scalars

// What a product costs, in us on a B200, by the measurements below; it is used to choose a kernel, never to skip work.
//   one CTA, T tokens a tile, S splits: an SM takes in 92 KB/us of operands with one CTA, 130 with more (a k-block is 16 KB
//   of W and T / 8 KB of T), or all of them W from HBM at 6.7 GB/ms; 3.5 for the launch, T / 40 for T tokens' epilogue
//   (with splits 0.7 + T / 125 for the exchange and a share of that); CTAs that do not fit at once start 3 later.
//   pair: 0.28 a k-block and wave, 11.5 for the launch and the last epilogue.
// Measured / by this rule, bf16, M x N x K: 1024 x 2048 x 8192 T128 S2 36 / 38, S1 50 / 51, pair 49 / 47;
// 512 x 4096 x 4096 T128 S2 23 / 23, pair 30 / 29; 256 x 4096 x 4096 T128 S4 16 / 15, T64 S2 17 / 17; 1024^3 T64 S2 9.4 / 9.4;
// 2048^3 pair 20 / 20, T128 S1 24 / 24.  int8: 2048^2 x 128 T128 S1 8.8 / 8.8, x 1024 10.2 / 12.2, x 4096 pair 18.9 / 20.5.
// The pair's rule is good for the few waves that it decides and no more: many full waves take a third longer (a k-block costs 0.37 at
// the chip's sustained rate), and short sums wait for the epilogue, which it leaves out: 8192^2 x 256 int8 56 / 19, with
// GELU 72 / 19, bf16 checkpoint 87 / 27.
struct Choice {
  int tokens = 0, splits = 1;
  double us = 1e30;
};
int k_blocks_of(int sum, int elem) { return (sum + 128 / elem - 1) / (128 / elem); }
Choice choose_one(const Device &d, int tokens, int channels, int sum, int elem, int least_tokens) {
  Choice best;
  const int kb = k_blocks_of(sum, elem);
  const double hbm = double(channels) * sum * elem / 6.7e6;
  for (int T = least_tokens; T <= 128; T *= 2) {
    if (tokens > 65535ll * T) continue;  // the grid's second dimension
    const double tiles = std::ceil(channels / 128.0) * std::ceil(tokens / double(T));
    for (int S = 1; S <= 8 && kb >= 2 * S - 1; S *= 2) {
      const double ctas = std::ceil(tiles * S / d.num_sms), blocks = (kb + S - 1) / S;
      const double in = ctas * blocks * (16 + T / 8) / (ctas > 1 ? 130 : 92);
      const double epilogue = S == 1 ? T / 40.0 : 0.7 + T / 125.0 + T / (40.0 * S);
      const double late = std::ceil(ctas / (T <= 64 ? 3 : 2)) - 1;
      const double us = 3.5 + std::max(in, hbm) + epilogue * (1 + 0.5 * std::min(ctas - 1, 2.0)) + 3 * late;
      if (us < best.us) best = {T, S, us};
    }
  }
  return best;
}
// n1 tiles of k1 k-blocks, then n2 of k2, dealt to the pairs in turn: the pair with the most.
double pair_us(const Device &d, long long n1, int k1, long long n2, int k2) {
  const long long pairs = d.num_sms / 2, over = (n1 + n2) % pairs;
  double most = 0;
  // a short last wave goes to the one-CTA kernel (run_pair): about half a wave and a launch
  const bool cut = n1 + n2 > pairs && 2 * over <= pairs && over <= n2;
  const long long n = n1 + n2 - (cut ? over : 0);
  for (long long p = 0; p < pairs; ++p) {
    const long long all = n > p ? (n - 1 - p) / pairs + 1 : 0, one = n1 > p ? (n1 - 1 - p) / pairs + 1 : 0;
    most = std::max(most, double(one) * k1 + double(all - one) * k2);
  }
  return 11.5 + 0.28 * (most + (cut && over ? 0.5 * k2 : 0.0));
}
long long pair_tiles(const Product &g) { return (g.channels + 255ll) / 256 * ((g.tokens + 255ll) / 256); }

template <class Op, class Epi>
int run_one(Device &d, const Product &g, int splits, const typename Epi::Args &args, cudaStream_t s, const Err &err) {
  CUtensorMap w, t;
  int rc, units;
  if ((rc = operand_maps<Op>(g, err, &w, &t))) return rc;
  const void *func = reinterpret_cast<const void *>(&pf::gemm8_one<Op, Epi>);
  if ((rc = kernel_units(d, func, kSmemPerSm - kOneStatic, 0, err, &units))) return rc;
  pf::Gemm8Params p = {};
  p.channels = g.channels;
  p.tokens = g.tokens;
  p.c_tiles = (g.channels + 127) / 128;
  p.t_tiles = (g.tokens + Op::TOKENS - 1) / Op::TOKENS;
  p.k_blocks = (g.sum + Op::BK - 1) / Op::BK;
  p.status = d.status;
  p.timeout_ns = kWaitNs;
  const long long tiles = static_cast<long long>(p.c_tiles) * p.t_tiles;
  // As deep a pipeline as lets the CTAs of one SM share its memory, at least what the split sums need; no deeper than
  // keeps the memory busy, so that the next launch finds room to start beside the last CTAs (int8 1 x 14336 x 4096, two CTAs
  // an SM: 6 stages 13.3 us, 4 12.9; 37 x 4096 x 14336, one: 6 14.4, 8 14.7).
  const int per_sm = static_cast<int>(std::min<long long>(4, (tiles * splits + d.num_sms - 1) / d.num_sms));
  const int room = (kSmemPerSm / per_sm - kOneStatic - 2048) / Op::STAGE_BYTES;  // alignment, and 1 KB of the system's
  const int least = std::max(2, (Op::TOKENS * 512 + Op::STAGE_BYTES - 1) / Op::STAGE_BYTES);
  const int busy = per_sm == 1 ? 6 : per_sm == 2 ? 4 : 3;
  p.stages = std::max(least, std::min({room, busy, (p.k_blocks + splits - 1) / splits}));
  pf::launch_cluster(&pf::gemm8_one<Op, Epi>, dim3(p.c_tiles * splits, p.t_tiles), dim3(pf::kOneThreads),
                     1024 + p.stages * Op::STAGE_BYTES, splits, s, w, t, p, args);
  return launched(err);
}

template <int kElem, bool kWK, bool kTK, class Epi>
int run_best_one(Device &d, const Product &g, const typename Epi::Args &args, cudaStream_t s, const Err &err) {
  using pf::Operands;
  const Choice c = choose_one(d, g.tokens, g.channels, g.sum, kElem, kTK ? 16 : 128 / kElem);
  if constexpr (kTK) {
    if (c.tokens == 16) return run_one<Operands<kElem, kWK, kTK, 16, 1>, Epi>(d, g, c.splits, args, s, err);
    if (c.tokens == 32) return run_one<Operands<kElem, kWK, kTK, 32, 1>, Epi>(d, g, c.splits, args, s, err);
  }
  if (c.tokens == 64) return run_one<Operands<kElem, kWK, kTK, 64, 1>, Epi>(d, g, c.splits, args, s, err);
  return run_one<Operands<kElem, kWK, kTK, 128, 1>, Epi>(d, g, c.splits, args, s, err);
}

// One product's part of a pair launch.
template <int kElem, bool kWK, bool kTK, class Epi_>
struct PairJob {
  static constexpr int ELEM = kElem;
  static constexpr bool WK = kWK, TK = kTK;
  typedef Epi_ Epi;
  typedef pf::Operands<kElem, kWK, kTK, 128, 2> Op;
  typedef pf::Job<Op, Epi> Kernel;
  Product g;
  typename Epi::Args args;
  CUtensorMap w, t;
  pf::Gemm8Params p = {};
  int prepare(Device &d, const Err &err) {
    int rc;
    if ((rc = operand_maps<Op>(g, err, &w, &t))) return rc;
    p.channels = g.channels;
    p.tokens = g.tokens;
    p.c_tiles = (g.channels + 255) / 256;
    p.t_tiles = (g.tokens + 255) / 256;
    p.k_blocks = (g.sum + Op::BK - 1) / Op::BK;
    p.group = std::min(16, p.c_tiles);
    p.status = d.status;
    p.timeout_ns = kWaitNs;
    const long long tiles = static_cast<long long>(p.c_tiles) * p.t_tiles;
    if (tiles > (1ll << 29)) return err(PF_EINVAL, "more than 2^29 tiles of 256 x 256");
    p.tiles = static_cast<int>(tiles);
    return PF_OK;
  }
};

// Whole waves of 256 x 256 tiles by the pair kernel.  Where the last wave would leave more than half of the pairs idle, its
// tiles (a rectangle: the last token columns of the raster's last group) go to the one-CTA kernel, which spreads them
// over the whole GPU: dB of 4096 x 14336 from 8192 tokens, 896 tiles on 74 pairs: 826 us in whole waves, 651 so.
// `first`: a product whose tiles come before `last`'s, or null.
template <int kEpiWarps, class First, class Last>
int run_pair_with(Device &d, First *first, Last &last, cudaStream_t s, const Err &err) {
  // Stages of two 128-byte atoms of the sum; sustained 16384 x 14336 x 4096 checkpoint, us: 3 of two 1475, 6 of one 1565; 3 of two
  // 1454, 2 of three 1600.
  constexpr int kStages = 3;
  typedef typename Last::Kernel J;
  using Cfg = pf::PairConfig<J, kStages, kEpiWarps>;
  constexpr bool kTwo = !std::is_same<First, Last>::value;
  const int before = kTwo ? first->p.tiles : 0;
  const void *func;
  if constexpr (kTwo) func = reinterpret_cast<const void *>(&pf::gemm8_pair<kStages, kEpiWarps, typename First::Kernel, J>);
  else func = reinterpret_cast<const void *>(&pf::gemm8_pair<kStages, kEpiWarps, J, pf::NoJob>);
  int rc, units;
  if ((rc = kernel_units(d, func, Cfg::SMEM_BYTES, Cfg::THREADS, err, &units))) return rc;
  pf::Gemm8Params &p = last.p;
  const int tiles = before + p.tiles, over = tiles % units, rows = p.c_tiles - (p.c_tiles - 1) / p.group * p.group;
  int columns = (over + rows - 1) / rows;
  if (tiles < units || 2 * columns * rows > units || columns >= p.t_tiles) columns = 0;
  p.tiles -= columns * rows;
  const dim3 grid(2 * std::min(tiles - columns * rows, units));
  if constexpr (kTwo)
    pf::launch_pdl(&pf::gemm8_pair<kStages, kEpiWarps, typename First::Kernel, J>, grid, Cfg::THREADS, Cfg::SMEM_BYTES, s, first->w,
                   first->t, last.w, last.t, first->p, p, first->args, last.args);
  else
    pf::launch_pdl(&pf::gemm8_pair<kStages, kEpiWarps, J, pf::NoJob>, grid, Cfg::THREADS, Cfg::SMEM_BYTES, s, last.w, last.t, last.w,
                   last.t, p, p, last.args, pf::NoJob::Args{});
  if ((rc = launched(err)) || columns == 0) return rc;
  const int c0 = (p.c_tiles - rows) * 256, t0 = (p.t_tiles - columns) * 256;
  return run_best_one<Last::ELEM, Last::WK, Last::TK, typename Last::Epi>(d, last.g.template part<typename Last::Op>(c0, t0),
                                                                          last.args.part(c0, t0), s, err);
}

// 16 epilogue warps where the epilogue is what a launch waits for: few k-blocks a tile, or one or two tiles a pair, whose
// last epilogue nothing covers.  8 otherwise: they take less power, which long launches run out of.  Measured, 8 / 16
// warps, us: checkpoint 8192^2 x 1024 140 / 120, int8 with GELU 101 / 80, bf16 2048^3 21.4 / 19.9; sustained 16384 x 14336 x
// 4096 checkpoint 1492 / 1526, int8 716 / 726.
template <class First, class Last>
int run_pair(Device &d, First *first, Last &last, cudaStream_t s, const Err &err) {
  int rc;
  if ((rc = last.prepare(d, err))) return rc;
  if constexpr (!std::is_same<First, Last>::value)
    if ((rc = first->prepare(d, err))) return rc;
  const int tiles = last.p.tiles + (std::is_same<First, Last>::value ? 0 : first->p.tiles);
  return k_blocks_of(last.g.sum, Last::ELEM) < 32 || tiles <= d.num_sms ? run_pair_with<16>(d, first, last, s, err)
                                                                        : run_pair_with<8>(d, first, last, s, err);
}

// Elements, W's and T's order, epilogue -> the kernel for the sizes.
template <int kElem, bool kWK, bool kTK, class Epi>
int product(Device &d, const Product &g, const typename Epi::Args &args, cudaStream_t s, const Err &err) {
  const Choice one = choose_one(d, g.tokens, g.channels, g.sum, kElem, kTK ? 16 : 128 / kElem);
  if (pair_us(d, 0, 0, pair_tiles(g), k_blocks_of(g.sum, kElem)) < one.us) {
    PairJob<kElem, kWK, kTK, Epi> job{g, args};
    return run_pair(d, &job, job, s, err);
  }
  return run_best_one<kElem, kWK, kTK, Epi>(d, g, args, s, err);
}

// dA and dB: one pair launch over both where that is estimated to be shorter than each by its own best kernel.
template <class EpiA, class EpiB>
int two_products(Device &d, const Product &ga, const typename EpiA::Args &aa, const Product &gb, const typename EpiB::Args &ab,
                 cudaStream_t s, const Err &err) {
  const auto alone = [&](const Product &g, int least) {
    return std::min(choose_one(d, g.tokens, g.channels, g.sum, 2, least).us, pair_us(d, 0, 0, pair_tiles(g), k_blocks_of(g.sum, 2)));
  };
  const double both = pair_us(d, pair_tiles(ga), k_blocks_of(ga.sum, 2), pair_tiles(gb), k_blocks_of(gb.sum, 2));
  if (both < alone(ga, 16) + alone(gb, 64)) {
    PairJob<2, true, true, EpiA> a{ga, aa};
    PairJob<2, false, false, EpiB> b{gb, ab};
    return run_pair(d, &a, b, s, err);
  }
  const int rc = product<2, true, true, EpiA>(d, ga, aa, s, err);
  return rc ? rc : product<2, false, false, EpiB>(d, gb, ab, s, err);
}

}  // namespace

extern "C" {

int pf_quantize_s8(int device, pf_dtype src, int rows, int cols, const void *X, long long ldx, int axis,
                   signed char *codes, long long ld_codes, float *scale, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (rows < 0 || cols < 0 || rows > kMostSize || cols > kMostSize)
    return err(PF_EINVAL, "rows and cols must be 0 to 2^30 (got %d, %d)", rows, cols);
  if (src != PF_F32 && src != PF_BF16) return err(PF_EINVAL, "the source type must be f32 or bf16");
  if (axis != 0 && axis != 1) return err(PF_EINVAL, "axis must be 1 (a scale for each row) or 0 (for each column), got %d", axis);
  const int lines = axis ? rows : cols;
  if (lines == 0) return PF_OK;
  const bool no_values = rows == 0 || cols == 0;  // each line's scale is the least one
  if (any_null(scale) || (!no_values && any_null(X, codes))) return err(PF_EINVAL, "null argument");
  if (ldx < cols || ld_codes < cols) return err(PF_EINVAL, "a row stride is below cols");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  if (no_values) {
    pf::launch_pdl(&pf::least_scales, dim3(blocks_of(lines, 256)), 256, 0, s, scale, lines);
    return launched(err);
  }
  int8_t *q = reinterpret_cast<int8_t *>(codes);
  rc = src == PF_F32 ? quantize<float>(*d, X, ldx, rows, cols, axis, q, ld_codes, scale, s, err)
                     : quantize<bf16>(*d, X, ldx, rows, cols, axis, q, ld_codes, scale, s, err);
  return rc ? rc : launched(err);
}

int pf_dequantize_s8(int device, int rows, int cols, const signed char *codes, long long ld_codes, const float *scale,
                     int axis, pf_dtype dst, void *X, long long ldx, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (rows < 0 || cols < 0 || rows > kMostSize || cols > kMostSize)
    return err(PF_EINVAL, "rows and cols must be 0 to 2^30 (got %d, %d)", rows, cols);
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
  if (dst == PF_F32) dequantize<float>(q, ld_codes, rows, cols, scale, axis, X, ldx, s);
  else dequantize<bf16>(q, ld_codes, rows, cols, scale, axis, X, ldx, s);
  return launched(err);
}

size_t pf_gemm_s8_workspace(int M, int N, int K, const signed char *A, long long lda, const signed char *B,
                            long long ldb) {
  return M < 1 || N < 1 || K < 1 ? 0 : ProductSpace(M, N, K, A, lda, B, ldb).total;
}

int pf_gemm_s8(int device, int M, int N, int K, const signed char *A, long long lda, const signed char *B, long long ldb,
               const float *scale_a, const float *scale_b, const float *bias, int gelu, pf_dtype out, void *C,
               long long ldc, void *workspace, size_t workspace_bytes, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (M < 0 || N < 0 || M > kMostSize || N > kMostSize) return err(PF_EINVAL, "M and N must be 0 to 2^30 (got %d, %d)", M, N);
  if (K < 1 || K > kMaxSumK)
    return err(PF_EINVAL, "K must be 1 to %d, so that a sum of int8 products fits 32 bits (got %d)", kMaxSumK, K);
  if (out != PF_F32 && out != PF_BF16) return err(PF_EINVAL, "the output type must be f32 or bf16");
  if (M == 0 || N == 0) return PF_OK;
  if (any_null(A, B) || any_null(scale_a, scale_b) || any_null(C)) return err(PF_EINVAL, "null argument");
  if (lda < K || ldb < N || ldc < N) return err(PF_EINVAL, "a row stride is below the row's length");
  const ProductSpace w(M, N, K, A, lda, B, ldb);
  if (w.total && (!workspace || workspace_bytes < w.total))
    return err(PF_EINVAL, "the workspace holds %zu bytes, %zu are needed", workspace ? workspace_bytes : size_t(0), w.total);
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return err(PF_EINVAL, "the workspace must be 256-byte aligned");
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  Product p{M, N, K, A, B, lda, ldb};
  char *base = static_cast<char *>(workspace);
  if (w.total) {
    if (static_cast<long long>(M) + K > 0x7FFFFFFF) return err(PF_EINVAL, "more than 2^31 rows to align");
    const pf::AlignRows a{reinterpret_cast<const uint8_t *>(A), lda, K, reinterpret_cast<uint4 *>(base), w.lda / 16};
    const pf::AlignRows b{reinterpret_cast<const uint8_t *>(B), ldb, N, reinterpret_cast<uint4 *>(base + w.b), w.ldb / 16};
    const int rows_a = w.copy_a ? M : 0;
    pf::launch_pdl(&pf::align_rows, dim3(rows_a + (w.copy_b ? K : 0)), 128, 0, s, a, b, rows_a);
    if (w.copy_a) p.T = base;
    if (w.copy_b) p.W = base + w.b;
  }
  p.ldt = w.lda;
  p.ldw = w.ldb;
  if (out == PF_F32)
    return product<1, false, true, pf::EpilogueS8<float>>(
        *d, p, {scale_a, scale_b, bias, static_cast<float *>(C), ldc, gelu}, s, err);
  return product<1, false, true, pf::EpilogueS8<bf16>>(*d, p, {scale_a, scale_b, bias, static_cast<bf16 *>(C), ldc, gelu},
                                                       s, err);
}

int pf_gemm_bias_gelu_checkpoint(int device, int M, int N, int K, const void *A, const void *B, const float *bias,
                                 void *C, signed char *a_codes, float *a_scale, unsigned char *grad_codes, void *stream,
                                 char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (M < 0 || N < 1 || K < 1 || M > kMostSize || N > kMostSize || K > kMostSize)
    return err(PF_EINVAL, "M must be 0 to 2^30, N and K 1 to 2^30 (got %d, %d, %d)", M, N, K);
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
  if (a_codes && (rc = quantize<bf16>(*d, A, K, M, K, 1, reinterpret_cast<int8_t *>(a_codes), K, a_scale, s, err))) return rc;
  return product<2, false, true, pf::EpilogueCheckpoint>(*d, Product{M, N, K, A, B, K, N},
                                                         {bias, static_cast<bf16 *>(C), grad_codes, N}, s, err);
}

size_t pf_gemm_bias_gelu_backward_workspace(int M, int N, int K) {
  return M < 1 || N < 1 || K < 1 || M > kMostSize || N > kMostSize || K > kMostSize ? 0 : BackwardSpace(M, N, K).total;
}

int pf_gemm_bias_gelu_backward(int device, int M, int N, int K, const void *dC, const void *B, const signed char *a_codes,
                               const float *a_scale, const unsigned char *grad_codes, void *dA, void *dB, float *dbias,
                               void *workspace, size_t workspace_bytes, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (M < 0 || N < 1 || K < 1 || M > kMostSize || N > kMostSize || K > kMostSize)
    return err(PF_EINVAL, "M must be 0 to 2^30, N and K 1 to 2^30 (got %d, %d, %d)", M, N, K);
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
  const long long dz_blocks = static_cast<long long>(w.col_blocks) * w.parts, blocks = dz_blocks + (dB ? M : 0);
  if (blocks > 0x7FFFFFFF) return err(PF_EINVAL, "more than 2^31 blocks");
  float *sums = dbias && w.parts == 1 ? dbias : partial;
  pf::launch_pdl(&pf::backward_operands, dim3(static_cast<unsigned>(blocks)), 256, 0, s, static_cast<const bf16 *>(dC), grad_codes,
                 dB ? a_scale : static_cast<const float *>(nullptr), M, N, static_cast<int>(dz_blocks), w.col_blocks, w.rows, dz, sums,
                 reinterpret_cast<const int8_t *>(a_codes), K, a);
  if (dbias && w.parts > 1)
    pf::launch_pdl(&pf::sum_row_blocks, dim3(blocks_of(N, 32)), 256, 0, s, static_cast<const float *>(partial), w.parts, N, dbias);
  typedef pf::EpilogueBf16<true> Divided;
  typedef pf::EpilogueBf16<false> Plain;
  const Product ga{M, K, N, dz, B, N, N}, gb{K, N, M, a, dz, K, N};
  bf16 *out_a = static_cast<bf16 *>(dA), *out_b = static_cast<bf16 *>(dB);
  if (dA && dB) return two_products<Divided, Plain>(*d, ga, {a_scale, out_a, K}, gb, {nullptr, out_b, N}, s, err);
  if (dA) return product<2, true, true, Plain>(*d, ga, {nullptr, out_a, K}, s, err);
  if (dB) return product<2, false, false, Plain>(*d, gb, {nullptr, out_b, N}, s, err);
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
  if (dst == PF_F32) dequantize_grad<float>(codes, count, X, s);
  else dequantize_grad<bf16>(codes, count, X, s);
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
  if (e == cudaSuccess && *err_word) {  // those alone: a kernel may have set another since
    clear_bits<<<1, 1>>>(d->status, *err_word);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? PF_OK : err(PF_ECUDA, "status read: %s", cudaGetErrorString(e));
}

int pf_ops8_selftest_wait_timeout(int device, unsigned long long timeout_ns, void *stream, char *err_text, size_t err_len) {
  const Err err{err_text, err_len};
  if (err_text && err_len) err_text[0] = '\0';
  if (timeout_ns == 0 || timeout_ns > pf::kSelftestMostNs)
    return err(PF_EINVAL, "timeout_ns must be 1 to %llu (got %llu)", pf::kSelftestMostNs, timeout_ns);
  Device *d;
  cudaStream_t s;
  int rc;
  if ((rc = device_of(device, err, &d))) return rc;
  DeviceGuard g(device);
  if ((rc = stream_of(device, stream, err, &s))) return rc;
  pf::selftest_wait_kernel<<<1, 32, 0, s>>>(d->status, timeout_ns);
  return launched(err);
}

}  // extern "C"

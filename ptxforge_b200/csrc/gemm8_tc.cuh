// gemm8_tc.cuh -- the products of the 8-bit operators on the 5th-generation tensor cores.
//
// Every one of them is  out[t][c] = f( sum_r T(t, r) W(r, c) )  with out row-major: t runs over tokens (for dB: over the
// input's columns), c over channels.  The tensor cores compute the transpose: UMMA rows are channels, UMMA columns
// tokens.  Then a TMEM lane is a channel, so
//   * a warp's store of one token is 32 neighbouring channels: whole sectors from registers, with no staging in shared
//     memory, no tensor map and no rule on out's alignment or row length;
//   * what belongs to a channel (its scale, its bias) sits in a register of its lane;
//   * few tokens make a narrow MMA (N = 16) instead of a mostly empty one, and little shared memory.
// Operands come by TMA in either order: K-major (the summed index contiguous) or MN-major, as they lie in memory; what a
// tile reaches past a matrix's edge is filled with zeros.  Element types: bf16 (fp32 sums) or int8 (int32 sums, exact).
//
//   gemm8_pair  256 channels x 256 tokens a CTA pair (.cta_group::2), persistent, two accumulators: tile i's epilogue
//               runs beside tile i+1's MMAs.  For products with enough tiles to fill the GPU.
//   gemm8_one   128 channels x 16..128 tokens a CTA, the sum split over a cluster of up to 8 CTAs whose accumulators are
//               added through distributed shared memory, in rank order.  For few tokens, where the bytes of W are
//               what counts, and for small products.
#pragma once

#include "gemm_tc.cuh"
#include "ops8_epilogue.cuh"

namespace pf {

// kElem: bytes of an element.  kWK: W lies as [c][r] (K-major), else as [r][c].  kTK: T lies as [t][r], else as [r][t].
// kTokens: tokens that this CTA loads.
template <int kElem, bool kWK, bool kTK, int kTokens, int kAtoms>
struct Operands {
  static constexpr int ELEM = kElem;
  static constexpr int TOKENS = kTokens;
  static constexpr int CHANNELS = 128;
  static constexpr int ATOM = 128 / kElem;        // elements of one 128-byte swizzle row
  static constexpr int BK = kAtoms * ATOM;        // summed index per stage
  static constexpr int UMMA_K = 32 / kElem;
  static constexpr int STEPS = BK / UMMA_K;       // MMAs per stage
  static constexpr int W_BYTES = kAtoms * CHANNELS * 128, T_BYTES = kAtoms * TOKENS * 128;
  static constexpr int STAGE_BYTES = W_BYTES + T_BYTES;
  static constexpr bool W_K = kWK, T_K = kTK;
  // TMA boxes: (inner, outer) elements
  static constexpr int W_BOX0 = ATOM, W_BOX1 = kWK ? CHANNELS : BK, T_BOX0 = ATOM, T_BOX1 = kTK ? TOKENS : BK;
  static_assert(kTK || TOKENS % ATOM == 0, "MN-major tokens come in whole 128-byte rows");
  static_assert(W_BOX1 <= 256 && T_BOX1 <= 256, "TMA box limit");

  template <bool kK, int kRows, class Load>
  static __device__ __forceinline__ void load(uint8_t *dst, int at, int kb, Load one) {
    if constexpr (kK) {
#pragma unroll
      for (int a = 0; a < kAtoms; ++a) one(dst + a * kRows * 128, kb * BK + a * ATOM, at);
    } else {
#pragma unroll
      for (int j = 0; j < kRows / ATOM; ++j) one(dst + j * BK * 128, at + j * ATOM, kb * BK);
    }
  }
  template <bool kK, int kRows>
  static __device__ __forceinline__ uint64_t desc(uint32_t addr, int step) {
    constexpr int PER_ATOM = ATOM / UMMA_K;
    if constexpr (kK)
      return smem_desc(addr + (step / PER_ATOM) * kRows * 128 + (step % PER_ATOM) * 32, 16, 1024, kSwizzle128B);
    else
      return smem_desc(addr + step * UMMA_K * 128, BK * 128, 1024, kSwizzle128B);
  }
  static constexpr uint32_t idesc(uint32_t M, uint32_t N) {
    // bf16: formats 1, fp32 sums (bits 4-5: 1); int8: signed formats 1, int32 sums (bits 4-5: 2)
    const uint32_t d = instr_desc(1u, 1u, kWK ? 0u : 1u, kTK ? 0u : 1u, M, N);
    return kElem == 2 ? d : (d & ~(3u << 4)) | (2u << 4);
  }
};

struct Gemm8Params {
  int channels, tokens;          // out's columns and rows
  int c_tiles, t_tiles, k_blocks;
  int group;                     // gemm8_pair: channel tiles that the raster walks before the next token tile
  int tiles;                     // gemm8_pair: the first so many of them
  int stages;                    // gemm8_one: pipeline depth, by the shared memory given
  unsigned *status;
  unsigned long long timeout_ns;
};

// ------------------------------------------------------------------------------------------------
// epilogues: one object a lane, for its channel.  Args::part: those of the product's part from channel c0, token t0 on.
// ------------------------------------------------------------------------------------------------
// Four neighbouring channels of a token, as the split sums come back (join_sums): `n` of them exist; `whole`: rows start
// on four-value boundaries, so that one store writes them.
__device__ __forceinline__ void store4(float *out, const float4 &y) { *reinterpret_cast<float4 *>(out) = y; }
__device__ __forceinline__ void store4(__nv_bfloat16 *out, const float4 &y) {
  *reinterpret_cast<uint2 *>(out) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}
template <class Out>
__device__ __forceinline__ void store_channels(Out *out, const float4 &y, int n, bool whole) {
  if (whole && n >= 4) {
    store4(out, y);
  } else {
    const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) out[j] = from_f32<Out>(v[j]);
  }
}
template <class Out>
__device__ __forceinline__ bool rows_of_four(const Out *out, long long ld) {
  return ld % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(Out)) == 0;
}
__device__ __forceinline__ float4 load_channels(const float *p, int n) {
  return make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
}

// A channel's scale as two factors, one of them 1: sum * first * (the token's scale) * last.  A scale below 1 goes first,
// any other last, so that no product on the way leaves fp32's range where the value itself does not (the two scales'
// own product may, and so may the sum times a large one).  Every kernel and every place in a tile takes this one order, so a
// token's values do not depend on what else is in the call.  It costs 0.4 % of 16384 x 14336 x 4096 (610 -> 612 us in bursts)
// and, where the epilogue is all, 3 % with GELU and 6 % without (8192^2 x 256: 70.1 -> 72.3, 53.2 -> 56.5) beside scales
// multiplied before the sum is there.
struct ChannelScale {
  float first, last;
  __device__ __forceinline__ explicit ChannelScale(float s) : first(fabsf(s) < 1.f ? s : 1.f), last(fabsf(s) < 1.f ? 1.f : s) {}
};

template <class Out>
struct EpilogueS8 {
  struct Args {
    const float *sa, *sb, *bias;  // bias may be null
    Out *out;
    long long ld;
    int gelu;
    Args part(int c0, int t0) const { return {sa + t0, sb + c0, bias ? bias + c0 : nullptr, out + t0 * ld + c0, ld, gelu}; }
  };
  static constexpr bool kTokenScalar = true;
  const Args &a;
  const int c;
  const bool inside;
  const ChannelScale sb;
  float bias;
  __device__ __forceinline__ EpilogueS8(const Args &args, int channel, int channels)
      : a(args), c(channel), inside(channel < channels), sb(channel < channels ? args.sb[channel] : 0.f) {
    bias = inside && a.bias ? a.bias[c] : 0.f;
  }
  static __device__ __forceinline__ float token(const Args &a, int t) { return a.sa[t]; }
  static __device__ __forceinline__ uint32_t add(uint32_t x, uint32_t y) { return x + y; }
  // Two tokens' sums and scalars -> their values.
  template <bool kGelu>
  __device__ __forceinline__ float2 value(uint32_t s0, uint32_t s1, float a0, float a1) const {
    const float2 sum = make_float2(static_cast<float>(static_cast<int>(s0)), static_cast<float>(static_cast<int>(s1)));
    const float2 x = __ffma2_rn(__fmul2_rn(__fmul2_rn(sum, both(sb.first)), make_float2(a0, a1)), both(sb.last), both(bias));
    return kGelu ? gelu_of(x) : x;
  }
  __device__ __forceinline__ void put(uint32_t sum, int t, float sa) const {
    const float2 y = a.gelu ? value<true>(sum, sum, sa, sa) : value<false>(sum, sum, sa, sa);
    if (inside) a.out[t * a.ld + c] = from_f32<Out>(y.x);
  }
  template <bool kGelu, int N>
  __device__ __forceinline__ void put_as(const uint32_t (&v)[N], int t0, const float *scalars) const {
    Out *out = a.out + t0 * a.ld + c;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 y = value<kGelu>(v[j], v[j + 1], scalars[j], scalars[j + 1]);
      if (inside) {
        out[j * a.ld] = from_f32<Out>(y.x);
        out[(j + 1) * a.ld] = from_f32<Out>(y.y);
      }
    }
  }
  template <int N>
  __device__ __forceinline__ void put_all(const uint32_t (&v)[N], int t0, const float *scalars) const {
    if (a.gelu) put_as<true>(v, t0, scalars);
    else put_as<false>(v, t0, scalars);
  }
  struct Row {
    const Args &a;
    const int c, n;
    const bool whole;
    float4 sb, bias;
    __device__ __forceinline__ Row(const Args &args, int c0, int channels)
        : a(args), c(c0), n(channels - c0), whole(rows_of_four(args.out, args.ld)) {
      sb = load_channels(a.sb + c, n);
      bias = a.bias ? load_channels(a.bias + c, n) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ void put(const uint32_t (&v)[4], int t, float sa) const {
      const auto two = [&](uint32_t v0, uint32_t v1, float s0, float s1, float b0, float b1) {
        const ChannelScale c0(s0), c1(s1);
        const float2 sum = make_float2(static_cast<float>(static_cast<int>(v0)), static_cast<float>(static_cast<int>(v1)));
        const float2 x = __ffma2_rn(__fmul2_rn(__fmul2_rn(sum, make_float2(c0.first, c1.first)), both(sa)),
                                    make_float2(c0.last, c1.last), make_float2(b0, b1));
        return a.gelu ? gelu_of(x) : x;
      };
      const float2 y0 = two(v[0], v[1], sb.x, sb.y, bias.x, bias.y), y1 = two(v[2], v[3], sb.z, sb.w, bias.z, bias.w);
      store_channels(a.out + t * a.ld + c, make_float4(y0.x, y0.y, y1.x, y1.y), n, whole);
    }
  };
};

struct EpilogueF32Sum {
  static __device__ __forceinline__ uint32_t add(uint32_t x, uint32_t y) {
    return __float_as_uint(__uint_as_float(x) + __uint_as_float(y));
  }
};

struct EpilogueCheckpoint : EpilogueF32Sum {
  struct Args {
    const float *bias;
    __nv_bfloat16 *out;
    uint8_t *codes;
    long long ld;
    Args part(int c0, int t0) const { return {bias + c0, out + t0 * ld + c0, codes + t0 * ld + c0, ld}; }
  };
  static constexpr bool kTokenScalar = false;
  const Args &a;
  const int c;
  const bool inside;
  float bias;
  __device__ __forceinline__ EpilogueCheckpoint(const Args &args, int channel, int channels)
      : a(args), c(channel), inside(channel < channels) {
    bias = inside ? a.bias[c] : 0.f;
  }
  static __device__ __forceinline__ float token(const Args &, int) { return 0.f; }
  __device__ __forceinline__ void put(uint32_t sum, int t, float) const {
    const float x = __uint_as_float(sum) + bias;
    const Gelu2 g = gelu_and_grad(make_float2(x, x));
    if (inside) {
      a.out[t * a.ld + c] = __float2bfloat16_rn(g.y.x);
      a.codes[t * a.ld + c] = static_cast<uint8_t>(grad_codes(g.d).x);
    }
  }
  template <int N>
  __device__ __forceinline__ void put_all(const uint32_t (&v)[N], int t0, const float *) const {
    const long long i = t0 * a.ld + c;
    __nv_bfloat16 *out = a.out + i;
    uint8_t *codes = a.codes + i;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const Gelu2 g = gelu_and_grad(__fadd2_rn(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), both(bias)));
      const uint2 code = grad_codes(g.d);
      if (inside) {
        out[j * a.ld] = __float2bfloat16_rn(g.y.x);
        out[(j + 1) * a.ld] = __float2bfloat16_rn(g.y.y);
        codes[j * a.ld] = static_cast<uint8_t>(code.x);
        codes[(j + 1) * a.ld] = static_cast<uint8_t>(code.y);
      }
    }
  }
  struct Row {  // channels come in eights here
    const Args &a;
    const int c;
    const bool inside;
    float4 bias;
    __device__ __forceinline__ Row(const Args &args, int c0, int channels) : a(args), c(c0), inside(c0 < channels) {
      bias = load_channels(a.bias + c, channels - c0);
    }
    __device__ __forceinline__ void put(const uint32_t (&v)[4], int t, float) const {
      const Gelu2 g0 = gelu_and_grad(make_float2(__uint_as_float(v[0]) + bias.x, __uint_as_float(v[1]) + bias.y));
      const Gelu2 g1 = gelu_and_grad(make_float2(__uint_as_float(v[2]) + bias.z, __uint_as_float(v[3]) + bias.w));
      const uint2 k0 = grad_codes(g0.d), k1 = grad_codes(g1.d);
      if (!inside) return;
      const long long i = t * a.ld + c;
      store4(a.out + i, make_float4(g0.y.x, g0.y.y, g1.y.x, g1.y.y));
      *reinterpret_cast<uint32_t *>(a.codes + i) =
          __byte_perm(__byte_perm(k0.x, k0.y, 0x0040), __byte_perm(k1.x, k1.y, 0x0040), 0x5410);
    }
  };
};

// kDivided: a token's row is divided by its m (split_scale of its input scale).
template <bool kDivided>
struct EpilogueBf16 : EpilogueF32Sum {
  struct Args {
    const float *token_scale;
    __nv_bfloat16 *out;
    long long ld;
    Args part(int c0, int t0) const { return {token_scale ? token_scale + t0 : nullptr, out + t0 * ld + c0, ld}; }
  };
  static constexpr bool kTokenScalar = kDivided;
  const Args &a;
  const int c;
  const bool inside;
  __device__ __forceinline__ EpilogueBf16(const Args &args, int channel, int channels)
      : a(args), c(channel), inside(channel < channels) {}
  static __device__ __forceinline__ float token(const Args &a, int t) {
    return kDivided ? __fdiv_rn(1.f, split_scale(a.token_scale[t]).m) : 1.f;
  }
  __device__ __forceinline__ void put(uint32_t sum, int t, float inv_m) const {
    if (inside) a.out[t * a.ld + c] = __float2bfloat16_rn(__uint_as_float(sum) * (kDivided ? inv_m : 1.f));
  }
  template <int N>
  __device__ __forceinline__ void put_all(const uint32_t (&v)[N], int t0, const float *scalars) const {
    __nv_bfloat16 *out = a.out + t0 * a.ld + c;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const __nv_bfloat16 y = __float2bfloat16_rn(__uint_as_float(v[j]) * (kDivided ? scalars[j] : 1.f));
      if (inside) out[j * a.ld] = y;
    }
  }
  struct Row {  // channels come in eights here
    const Args &a;
    const int c;
    const bool inside;
    __device__ __forceinline__ Row(const Args &args, int c0, int channels) : a(args), c(c0), inside(c0 < channels) {}
    __device__ __forceinline__ void put(const uint32_t (&v)[4], int t, float inv_m) const {
      const float f = kDivided ? inv_m : 1.f;
      if (inside)
        store4(a.out + t * a.ld + c, make_float4(__uint_as_float(v[0]) * f, __uint_as_float(v[1]) * f, __uint_as_float(v[2]) * f,
                                                 __uint_as_float(v[3]) * f));
    }
  };
};

// The scalars of tokens [t0, t0 + 32 n) into this warp's shared memory, from which a broadcast load brings four.
template <class Epi>
__device__ __forceinline__ void stage_scalars(const typename Epi::Args &args, int t0, int n, int tokens, int lane,
                                              float *scalars) {
  if constexpr (Epi::kTokenScalar) {
    __syncwarp();  // the last tile's were read
    for (int b = 0; b < n; ++b) {
      const int t = t0 + b * 32 + lane;
      scalars[b * 32 + lane] = t < tokens ? Epi::token(args, t) : 0.f;
    }
    __syncwarp();
  }
}

// N tokens from t0 on.  Whole blocks run without a branch a token, so that the arithmetic of many overlaps (with one, a
// tile of 256 x 256 took 27 us).
template <class Epi, int N>
__device__ __forceinline__ void put_block(const Epi &e, const uint32_t (&v)[N], int t0, int tokens, const float *scalars) {
  if (t0 + N <= tokens) {
    e.put_all(v, t0, scalars);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (t0 + j < tokens) e.put(v[j], t0 + j, Epi::kTokenScalar ? scalars[j] : 0.f);
  }
}

// ------------------------------------------------------------------------------------------------
// one CTA a tile, the sum split over a cluster
// ------------------------------------------------------------------------------------------------
constexpr int kOneThreads = 192;
constexpr int kOneMaxStages = 8;

// This CTA's share of the tokens: every CTA's sums, added in rank order.  They lie as [token][128 channels]; a warp takes a
// token, a lane four of its channels, so that what crosses between SMs are whole lines (as [channel][token], 16 bytes a
// lane, eight CTAs' sums of 128 x 128 took 50 us), and the sums of several tokens are on their way before the first
// addition.
template <int kTokens, int kSplits, class Epi>
__device__ __forceinline__ void join_sums(const typename Epi::Args &args, int c0, int channels, uint32_t base, uint32_t rank,
                                          int warp, int lane, int t0, int tokens, const float *scalars) {
  constexpr int SHARE = kTokens / kSplits, AHEAD = SHARE < 4 ? 1 : kSplits == 8 || SHARE < 16 ? 1 : kSplits == 4 ? 2 : 4;
  static_assert(AHEAD == 1 || SHARE % (4 * AHEAD) == 0, "the look-ahead stays in this CTA's share");
  const typename Epi::Row row(args, c0 + lane * 4, channels);
  const bool inside = c0 + lane * 4 < channels;
  const int mine = static_cast<int>(rank) * SHARE;
  uint32_t from[kSplits];
#pragma unroll
  for (int s = 0; s < kSplits; ++s) from[s] = mapa_shared(base + lane * 16, s);
#pragma unroll 1
  for (int t = mine + warp; t < mine + SHARE && t0 + t < tokens; t += 4 * AHEAD) {
    // Only sums that are stored below: the cluster's last barrier orders no memory, so what makes a remote load end before
    // its CTA may leave is that its value is used.
    uint32_t v[AHEAD][kSplits][4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (!inside || t0 + t + i * 4 >= tokens) continue;
#pragma unroll
      for (int s = 0; s < kSplits; ++s) ld_cluster4(from[s] + (t + i * 4) * 512, v[i][s]);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int at = t + i * 4;
      if (!inside || t0 + at >= tokens) continue;
#pragma unroll
      for (int s = 1; s < kSplits; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][0][j] = Epi::add(v[i][0][j], v[i][s][j]);
      row.put(v[i][0], t0 + at, Epi::kTokenScalar ? scalars[at] : 0.f);
    }
  }
}

template <class Op, class Epi>
__global__ void __launch_bounds__(kOneThreads, 4)
    gemm8_one(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmT, const Gemm8Params p,
              const typename Epi::Args args) {
  constexpr int TOKENS = Op::TOKENS;
  constexpr int TMEM_COLS = TOKENS < 32 ? 32 : TOKENS;
  constexpr uint32_t IDESC = Op::idesc(128, TOKENS);
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[kOneMaxStages], empty[kOneMaxStages], done;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  __shared__ __align__(16) float scalars[4][TOKENS < 32 ? 32 : TOKENS];
  volatile int *abort_flag = &abort_word;
  uint8_t *sW = smem, *sT = smem + p.stages * Op::W_BYTES;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
  const uint32_t rank = cluster_ctarank();
  const int c0 = static_cast<int>(blockIdx.x / splits) * 128, t0 = static_cast<int>(blockIdx.y) * TOKENS;
  const int tokens = min(p.tokens, t0 + TOKENS);
  // this CTA's share of the sum
  const int kb0 = static_cast<int>(static_cast<long long>(p.k_blocks) * rank / splits);
  const int kb1 = static_cast<int>(static_cast<long long>(p.k_blocks) * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmT);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_holder, TMEM_COLS);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  auto fail = [&](unsigned bit) {
    atomicOr(p.status, bit);
    *abort_flag = 1;
  };
  grid_launch_dependents();
  grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, p.timeout_ns, abort_flag)) {
          fail(kErrProducerWait);
          ok = false;
          break;
        }
        uint64_t *bar = &full[stage];
        mbar_arrive_expect_tx(bar, Op::STAGE_BYTES);
        Op::template load<Op::W_K, 128>(sW + stage * Op::W_BYTES, c0, kb, [&](uint8_t *dst, int x, int y) {
          tma_load_2d(dst, &tmW, bar, x, y);
        });
        Op::template load<Op::T_K, TOKENS>(sT + stage * Op::T_BYTES, t0, kb, [&](uint8_t *dst, int x, int y) {
          tma_load_2d(dst, &tmT, bar, x, y);
        });
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        // Loads in flight land before the CTA may exit (bounded).
        for (int s = 0; s < p.stages && s < issued; ++s) {
          const uint32_t ph = (s < stage) ? phase : (phase ^ 1u);
          volatile int no_abort = 0;
          if (!mbar_wait(&full[s], ph, p.timeout_ns, &no_abort)) atomicOr(p.status, kErrTeardownWait);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, p.timeout_ns, abort_flag)) {
          fail(kErrMmaWait);
          break;
        }
        tc_fence_after();
        const uint32_t w = smem_u32(sW + stage * Op::W_BYTES), t = smem_u32(sT + stage * Op::T_BYTES);
#pragma unroll
        for (int i = 0; i < Op::STEPS; ++i) {
          const uint64_t wd = Op::template desc<Op::W_K, 128>(w, i), td = Op::template desc<Op::T_K, TOKENS>(t, i);
          const uint32_t accumulate = (kb != kb0 || i != 0) ? 1u : 0u;
          if constexpr (Op::ELEM == 2) tc_mma_f16(tmem, wd, td, IDESC, accumulate);
          else tc_mma_i8(tmem, wd, td, IDESC, accumulate);
        }
        tc_commit(&empty[stage]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(&done);  // every MMA complete: the sums are in TMEM, and no stage is read any more
      volatile int no_abort = 0;
      if (!mbar_wait(&done, 0, p.timeout_ns, &no_abort)) atomicOr(p.status, kErrTeardownWait);
    }
  } else {
    const int q = warp & 3;
    const int c_local = q * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const Epi epi(args, c0 + c_local, p.channels);
    stage_scalars<Epi>(args, t0, (TOKENS + 31) / 32, tokens, lane, scalars[q]);
    const bool waited = mbar_wait(&done, 0, p.timeout_ns, abort_flag);
    if (!__all_sync(0xffffffffu, waited)) {
      if (lane == 0) fail(kErrEpilogueWait);
    } else {
      tc_fence_after();
      constexpr int N = TOKENS < 32 ? TOKENS : 32;
      uint32_t *mine = reinterpret_cast<uint32_t *>(smem) + c_local;  // [token][128 channels], where the stages were
#pragma unroll 1
      for (int b = 0; b < TOKENS / N; ++b) {
        if (t0 + b * N >= tokens) break;
        uint32_t v[N];
        tmem_ld<N>(t_row + b * N, v);
        tmem_ld_wait();
        if (splits == 1) {
          put_block(epi, v, t0 + b * N, tokens, scalars[q] + b * N);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) mine[(b * N + j) * 128] = v[j];
        }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();  // every CTA's sums are in its shared memory
    if (warp >= 2) {
      const uint32_t base = smem_u32(smem);
      const float *sc = scalars[warp & 3];
      if (splits == 2) join_sums<TOKENS, 2, Epi>(args, c0, p.channels, base, rank, warp - 2, lane, t0, tokens, sc);
      else if (splits == 4) join_sums<TOKENS, 4, Epi>(args, c0, p.channels, base, rank, warp - 2, lane, t0, tokens, sc);
      else join_sums<TOKENS, 8, Epi>(args, c0, p.channels, base, rank, warp - 2, lane, t0, tokens, sc);
    }
    __syncwarp();
    cluster_arrive_relaxed();
    cluster_wait();  // nobody leaves while its shared memory may be read
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------
// CTA pairs
// ------------------------------------------------------------------------------------------------
// Consecutive tiles walk down `group` channel tiles, then across the token tiles, so pairs that run at the same time
// share both operands' panels in L2.
__device__ __forceinline__ void pair_tile(int i, const Gemm8Params &p, int &ct, int &tt) {
  const int per_group = p.group * p.t_tiles;
  const int g = i / per_group, first = g * p.group;
  const int rows = min(p.c_tiles - first, p.group);
  const int r = i - g * per_group;
  ct = first + r % rows;
  tt = r / rows;
}

// A pair kernel walks the tiles of one product, or of two, one after the other: dA and dB of a layer keep the pairs busy
// together where either alone would leave a wave unfilled, and share the launch.
template <class Op, class Epi>
struct Job {
  typedef Op Operands;
  typedef Epi Epilogue;
  typedef typename Epi::Args Args;
  static constexpr bool kNone = false;
};
struct NoJob {
  struct Args {};
  static constexpr bool kNone = true;
};

template <class J, int kStages, int kEpiWarps>
struct PairConfig {
  typedef typename J::Operands Op;
  static constexpr int STAGES = kStages;
  static constexpr int EPI_WARPS = kEpiWarps;            // 8 or 16: 2 or 4 to a quarter of the TMEM lanes, which share its tokens
  static constexpr int EPI_BLOCKS = 32 / EPI_WARPS;      // blocks of 32 tokens a warp
  static constexpr int THREADS = 64 + EPI_WARPS * 32;
  static constexpr int NUM_BARS = 2 * STAGES + 4 + 1;
  static constexpr int SMEM_BYTES = 1024 + STAGES * Op::STAGE_BYTES + NUM_BARS * 8 + 16;
  static_assert(Op::TOKENS == 128, "each CTA of a pair supplies 128 tokens");
  static_assert(SMEM_BYTES <= 232448, "shared memory per block exceeds the sm_100 opt-in limit");
};

template <int kStages, int kEpiWarps, class J1, class J2>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairConfig<J1, kStages, kEpiWarps>::THREADS, 1)
    gemm8_pair(const __grid_constant__ CUtensorMap tmW1, const __grid_constant__ CUtensorMap tmT1,
               const __grid_constant__ CUtensorMap tmW2, const __grid_constant__ CUtensorMap tmT2, const Gemm8Params p1,
               const Gemm8Params p2, const typename J1::Args args1, const typename J2::Args args2) {
  using Cfg = PairConfig<J1, kStages, kEpiWarps>;
  constexpr int W_BYTES = Cfg::Op::W_BYTES, T_BYTES = Cfg::Op::T_BYTES, STAGE_BYTES = Cfg::Op::STAGE_BYTES;
  __shared__ __align__(16) float scalars[Cfg::EPI_WARPS][Cfg::EPI_BLOCKS * 32];
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sW = smem, *sT = smem + Cfg::STAGES * W_BYTES;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + Cfg::STAGES * STAGE_BYTES);  // leader: both CTAs' bytes landed
  uint64_t *empty = full + Cfg::STAGES;                                             // both: the stage was read
  uint64_t *tfull = empty + Cfg::STAGES;                                            // both: accumulator ready
  uint64_t *tempty = tfull + 2;                                                     // leader: accumulator drained
  uint64_t *drain = tempty + 2;                                                     // leader: all MMAs complete
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p1.tiles + (J2::kNone ? 0 : p2.tiles);
  // f(job, W's map, T's map, parameters, epilogue arguments, the job's tile) for tile i of the launch
  auto with_tile = [&](int i, auto f) {
    if constexpr (!J2::kNone) {
      static_assert(J2::Operands::W_BYTES == W_BYTES && J2::Operands::T_BYTES == T_BYTES, "the jobs share the stages");
      if (i >= p1.tiles) return f(J2{}, &tmW2, &tmT2, p2, args2, i - p1.tiles);
    }
    return f(J1{}, &tmW1, &tmT1, p1, args1, i);
  };

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW1);
    tma_prefetch_desc(&tmT1);
    if (!J2::kNone) {
      tma_prefetch_desc(&tmW2);
      tma_prefetch_desc(&tmT2);
    }
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * Cfg::EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, 512);
    tmem_relinquish_pair();
    tc_fence_before();
  }
  cluster_sync();  // both CTAs' barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  auto fail = [&](unsigned bit) {
    atomicOr(p1.status, bit);
    *abort_flag = 1;
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      auto produce = [&](auto job, const CUtensorMap *tmW, const CUtensorMap *tmT, const Gemm8Params &p, const auto &, int i) {
        using Op = typename decltype(job)::Operands;
        int ct, tt;
        pair_tile(i, p, ct, tt);
        const int c0 = ct * 256 + static_cast<int>(rank) * 128, t0 = tt * 256 + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, p.timeout_ns, abort_flag)) {
            fail(kErrProducerWait);
            return false;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * STAGE_BYTES);
          if (issued == 0) grid_dependency_wait();
          const uint32_t bar = pair_leader_addr(smem_u32(&full[stage]));
          Op::template load<Op::W_K, 128>(sW + stage * W_BYTES, c0, kb, [&](uint8_t *dst, int x, int y) {
            tma_load_2d_pair(dst, tmW, bar, x, y);
          });
          Op::template load<Op::T_K, 128>(sT + stage * T_BYTES, t0, kb, [&](uint8_t *dst, int x, int y) {
            tma_load_2d_pair(dst, tmT, bar, x, y);
          });
          ++issued;
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        return true;
      };
      bool ok = true;
      for (int i = pair; ok && i < tiles; i += pairs) ok = with_tile(i, produce);
      if (!ok && rank == 0) {
        // Loads in flight land before the pair may exit (bounded).
        for (int s = 0; s < Cfg::STAGES && s < issued; ++s) {
          const uint32_t ph = (s < stage) ? phase : (phase ^ 1u);
          volatile int no_abort = 0;
          if (!mbar_wait(&full[s], ph, p1.timeout_ns, &no_abort)) atomicOr(p1.status, kErrTeardownWait);
        }
      }
    }
    grid_launch_dependents();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      auto multiply = [&](auto job, const CUtensorMap *, const CUtensorMap *, const Gemm8Params &p, const auto &, int) {
        using Op = typename decltype(job)::Operands;
        constexpr uint32_t IDESC = Op::idesc(256, 256);
        if (!mbar_wait_cluster(&tempty[acc], acc_phase ^ 1u, p.timeout_ns, abort_flag)) {
          fail(kErrMmaWait);
          return false;
        }
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(acc * 256);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.timeout_ns, abort_flag)) {
            fail(kErrMmaWait);
            return false;
          }
          tc_fence_after();
          const uint32_t w = smem_u32(sW + stage * W_BYTES), t = smem_u32(sT + stage * T_BYTES);
#pragma unroll
          for (int k = 0; k < Op::STEPS; ++k) {
            const uint64_t wd = Op::template desc<Op::W_K, 128>(w, k), td = Op::template desc<Op::T_K, 128>(t, k);
            const uint32_t accumulate = (kb != 0 || k != 0) ? 1u : 0u;
            if constexpr (Op::ELEM == 2) tc_mma_f16_pair(d, wd, td, IDESC, accumulate);
            else tc_mma_i8_pair(d, wd, td, IDESC, accumulate);
          }
          tc_commit_pair_mc(&empty[stage], 0x3);
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        tc_commit_pair_mc(&tfull[acc], 0x3);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
        return true;
      };
      for (int i = pair; i < tiles; i += pairs)
        if (!with_tile(i, multiply)) break;
      tc_commit_pair(drain);
      volatile int no_abort = 0;
      if (!mbar_wait(drain, 0, p1.timeout_ns, &no_abort)) atomicOr(p1.status, kErrTeardownWait);
    }
    grid_launch_dependents();
  } else {
    grid_launch_dependents();
    grid_dependency_wait();
    const int q = warp & 3, first = ((warp - 2) >> 2) * Cfg::EPI_BLOCKS * 32;
    float *mine = scalars[warp - 2];
    int acc = 0;
    uint32_t acc_phase = 0;
    auto finish = [&](auto job, const CUtensorMap *, const CUtensorMap *, const Gemm8Params &p, const auto &args, int i) {
      using Epi = typename decltype(job)::Epilogue;
      int ct, tt;
      pair_tile(i, p, ct, tt);
      const int t0 = tt * 256 + first;
      // what belongs to the channel and the tokens is loaded while the accumulator fills
      const Epi epi(args, ct * 256 + static_cast<int>(rank) * 128 + q * 32 + lane, p.channels);
      stage_scalars<Epi>(args, t0, Cfg::EPI_BLOCKS, p.tokens, lane, mine);
      const bool waited = mbar_wait(&tfull[acc], acc_phase, p.timeout_ns, abort_flag);
      if (!__all_sync(0xffffffffu, waited)) {
        if (lane == 0) fail(kErrEpilogueWait);
        return false;
      }
      tc_fence_after();
      const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * 256 + first);
      // The next block's sums travel from TMEM while this block's values are computed.
      uint32_t v[2][32];
      tmem_ld_32x32b_x32(t_row, v[0]);
#pragma unroll
      for (int b = 0; b < Cfg::EPI_BLOCKS; ++b) {
        tmem_ld_wait();
        if (b + 1 < Cfg::EPI_BLOCKS) {
          tmem_ld_32x32b_x32(t_row + (b + 1) * 32, v[(b + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
        }
        if (t0 + b * 32 < p.tokens) put_block(epi, v[b & 1], t0 + b * 32, p.tokens, mine + b * 32);
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
      return true;
    };
    for (int i = pair; i < tiles; i += pairs)
      if (!with_tile(i, finish)) break;
  }
  // Neither CTA releases TMEM or exits while its peer may still address it (with a release: the last remote arrivals
  // on `tempty` land before the leader may leave).
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace pf

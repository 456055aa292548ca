// ops8_epilogue.cuh -- what the 8-bit operators do with a finished sum of a product.
//
//   gelu(x) = x p,  gelu'(x) = p + 2 u'(x) x p (1 - p),  p = 1 / (1 + exp(-2 u)),  u = k0 (x + k1 x^3)
//
// which is the tanh form (0.5 (1 + tanh u) = p) without the cancellation of 1 + tanh for negative x: exp2 and
// reciprocal in hardware leave a relative error of a few 2^-22, where tanh.approx's 2^-11 would move the 8-bit
// derivative by up to half a step.
#pragma once

#include "quant_s8.cuh"

namespace pf {

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x in [-12, 12]; a NaN stays one.
__device__ __forceinline__ float clamp12(float x) {
  float y;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC1400000;\n\tmin.NaN.f32 %0, t, 0f41400000;\n\t}" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kGeluK0 = 0.7978845608028654f, kGeluK1 = 0.044715f;
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Two values at a time: sm_100 multiplies and adds fp32 pairs in one instruction, each half rounded as alone.
// p of the formulas above; exp2 overflows to infinity for very negative x, whose reciprocal is 0.
__device__ __forceinline__ float2 gelu_p(float2 x, float2 x2) {
  constexpr float a = -2.f * kLog2E * kGeluK0, b = a * kGeluK1;
  const float2 e = __fmul2_rn(x, __ffma2_rn(both(b), x2, both(a)));
  const float2 q = __fadd2_rn(both(1.f), make_float2(exp2_approx(e.x), exp2_approx(e.y)));
  return make_float2(rcp_approx(q.x), rcp_approx(q.y));
}
__device__ __forceinline__ float2 gelu_of(float2 x) { return __fmul2_rn(x, gelu_p(x, __fmul2_rn(x, x))); }

// The GELU and its derivative.  Both use p at x clamped to [-12, 12], where it is 0 or 1 to fp32 already: an infinite x
// has the limit's derivative, not inf * 0.
struct Gelu2 {
  float2 y, d;
};
__device__ __forceinline__ Gelu2 gelu_and_grad(float2 x) {
  const float2 c = make_float2(clamp12(x.x), clamp12(x.y)), c2 = __fmul2_rn(c, c);
  const float2 p = gelu_p(c, c2);
  const float2 u2 = __fmul2_rn(c, __ffma2_rn(both(6.f * kGeluK0 * kGeluK1), c2, both(2.f * kGeluK0)));  // 2 u'(x) x
  const float2 pq = __ffma2_rn(make_float2(-p.x, -p.y), p, p);                                         // p (1 - p)
  return {__fmul2_rn(x, p), __ffma2_rn(u2, pq, p)};
}

// Codes of two derivatives in the low bytes: 200 d + 26 is added to 1.5 2^23, where a float's step is 1, so the rounding
// of the fused multiply-add is rint, and the low byte of its bits the code.  A NaN's bits are 0x7FFFFFFF: code 255.
__device__ __forceinline__ uint2 grad_codes(float2 d) {
  const float2 c = __ffma2_rn(d, both(kGradSteps), both(12582912.f + kGradZero));
  return make_uint2(__float_as_uint(c.x), __float_as_uint(c.y));
}

}  // namespace pf

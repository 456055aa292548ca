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

struct Gelu {
  float y, d;
};

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

constexpr float kGeluK0 = 0.7978845608028654f, kGeluK1 = 0.044715f;
constexpr float kLog2E = 1.4426950408889634f;

// p(x) of the formulas above.  exp2 overflows to infinity for very negative x, whose reciprocal is 0.
__device__ __forceinline__ float gelu_p(float x) {
  constexpr float a = -2.f * kLog2E * kGeluK0, b = a * kGeluK1;
  return rcp_approx(1.f + exp2_approx(x * fmaf(b, x * x, a)));
}
__device__ __forceinline__ float gelu_of(float x) { return x * gelu_p(x); }

// The derivative is taken at x clamped to [-12, 12], where it is 0 or 1 to fp32 already: an infinite x has the
// limit's derivative, not inf * 0.  A NaN stays one.
__device__ __forceinline__ Gelu gelu_and_grad(float x) {
  const float xc = x != x ? x : fminf(fmaxf(x, -12.f), 12.f);
  const float p = gelu_p(xc);
  const float du2 = fmaf(6.f * kGeluK0 * kGeluK1, xc * xc, 2.f * kGeluK0);
  const float d = fmaf(xc * du2, p * (1.f - p), p);
  return {xc == x ? x * p : gelu_of(x), d};
}

}  // namespace pf

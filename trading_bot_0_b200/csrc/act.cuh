// The step size's and the projection's softplus, from one exponential and a polynomial.
#pragma once
#include "umma.cuh"

namespace ssd {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// log(1 + e) for e in [0, 1]: e P(e) with P the least-maximum fit of log1p(e) / e of degree 8 (relative error 3e-8, 1.7e-7 as
// evaluated), so that small step sizes keep their digits where log(1 + e) would lose them.
__device__ __forceinline__ float log1p01(float e) {
  float p = 0.00523267664f;
  p = fmaf(p, e, -0.0295051682f);
  p = fmaf(p, e, 0.0782258369f);
  p = fmaf(p, e, -0.13663236f);
  p = fmaf(p, e, 0.191060022f);
  p = fmaf(p, e, -0.24842981f);
  p = fmaf(p, e, 0.333190967f);
  p = fmaf(p, e, -0.499994931f);
  p = fmaf(p, e, 0.99999997f);
  return p * e;
}
// exp(-|v|), the rounding of the argument made good where there is anything left of the result (t may be -inf, and is from |v| = 2.36e38
// on: the remainder is no number then; a NaN stays one)
__device__ __forceinline__ float exp_neg(float v) {
  const float x = -fabsf(v), t = x * LOG2E, r = fmaf(x, LOG2E, -t), e = umma::ex2(t);
  return t < -200.f ? e : fmaf(e, r * LN2, e);
}
__device__ __forceinline__ float softplusf_(float v) { return fmaxf(v, 0.f) + log1p01(exp_neg(v)); }

}  // namespace ssd

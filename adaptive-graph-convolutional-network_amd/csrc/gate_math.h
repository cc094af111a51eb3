// e^-x and 1 / (1 + e) for gates (sigmoid, tanh, silu) in fp32, on the hardware's exp2 and reciprocal.
#ifndef AGCN_GATE_MATH_H
#define AGCN_GATE_MATH_H
#include <hip/hip_runtime.h>

namespace agcn {
// e^-x for x >= 0, within a few 2^-24 of itself: the product with log2 e is carried in two parts.  (x beyond 128: e^-128 is below every
// normal number; a NaN stays one.)
__device__ __forceinline__ float exp_neg(float x) {
  x = x > 128.f ? -128.f : -x;
  const float hi = x * 1.44269504f, lo = fmaf(x, 1.925963033e-8f, fmaf(x, 1.44269504f, -hi));
  const float e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e, lo * 0.69314718f, e);
}
// 1 / (1 + e) for 0 <= e <= 1: the hardware's reciprocal and one Newton step
__device__ __forceinline__ float recip_1p(float e) {
  const float d = __builtin_amdgcn_rcpf(1.f + e);
  return fmaf(d, fmaf(-(1.f + e), d, 1.f), d);
}
}  // namespace agcn
#endif

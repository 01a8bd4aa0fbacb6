// The final-logit softcap as the head kernels' epilogues evaluate it.
#pragma once

#include "gs_internal.h"

namespace gs {

// cap tanh(x / cap) of kN values of each lane. Below 5/8 tanh q is
// q + q^3 P(q^2), P of degree 5 fitted over that range (relative error of the
// fit 2^-32; at most 0.70 ulp with its roundings); a wave whose values all lie
// there evaluates them side by side, where a tanhf a value, each behind its
// own branch, was one long chain (60 of 690 us at M 512, D 2048, V 262144).
// Their x / cap rounded to nearest takes two fused multiply-adds from
// r = 1 / cap rounded to nearest (Markstein: the remainder of q0 = x r is
// exact, and its share r completes the quotient). Every value takes the same
// formula in either branch. r = 0 (cap outside 2^+-60): always the division.
constexpr float kTanhSmall = 0.625f;
__device__ __forceinline__ float tanh_small(float q) {
  const float s = q * q;
  float p = 0x1.197b58p-9f;
  p = __builtin_fmaf(p, s, -0x1.0c213cp-7f);
  p = __builtin_fmaf(p, s, 0x1.6394d6p-6f);
  p = __builtin_fmaf(p, s, -0x1.b9ef7cp-5f);
  p = __builtin_fmaf(p, s, 0x1.11106cp-3f);
  p = __builtin_fmaf(p, s, -0x1.555554p-2f);
  return __builtin_fmaf(q * s, p, q);
}
__device__ __forceinline__ float reciprocal_of_cap(float cap) {
  return cap >= 0x1p-60f && cap <= 0x1p60f ? 1.0f / cap : 0.0f;
}
template <int kN>
__device__ __forceinline__ void lmhead_cap(float (&x)[kN], float cap, float r) {
  float q[kN];
  bool small = r != 0.0f;
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    const float q0 = x[e] * r;
    q[e] = __builtin_fmaf(__builtin_fmaf(-q0, cap, x[e]), r, q0);
    small = small && __builtin_fabsf(q[e]) < kTanhSmall;  // (false for a NaN)
  }
  if (__all(small)) {
#pragma unroll
    for (int e = 0; e < kN; ++e) x[e] = cap * tanh_small(q[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float v = x[e] / cap;
      x[e] = cap * (__builtin_fabsf(v) < kTanhSmall ? tanh_small(v) : tanhf(v));
    }
  }
}

}  // namespace gs

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

constexpr float kLog2e = 1.44269504088896341f;

// The cap, x -> cap tanh(x / cap). Below 5/8 of the cap tanh q = q (1 + s P(s)),
// s = q^2, P of degree 4 fitted over that range (relative error 2^-27); past it
// 1 - 2 / (e^2q + 1). Either is within 2e-7 of the cap.
__device__ constexpr float kCapP[5] = {-0x1.555532p-2f, 0x1.110726p-3f, -0x1.b83c58p-5f, 0x1.52268ep-6f, -0x1.75e194p-8f};
__device__ __forceinline__ float cap_series(float s) {
  float u = kCapP[4];
#pragma unroll
  for (int i = 3; i >= 0; --i) u = __builtin_fmaf(u, s, kCapP[i]);
  return __builtin_fmaf(u, s, 1.0f);
}
__device__ __forceinline__ float cap_far(float q) {
  return 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(q * (2.0f * kLog2e)) + 1.0f);
}
__device__ __forceinline__ float cap_any(float q) {  // tanh q
  return __builtin_fabsf(q) < kTanhSmall ? q * cap_series(q * q) : cap_far(q);
}

// The near part in x itself: cap tanh(x / cap) unit = x u(x^2), the powers of 1 /
// cap and the unit (1, or log2(e) for exponentials) in u's coefficients. `far`:
// where |x| has to stay below (0, never, for caps whose powers leave binary32's
// range).
struct CapSeries {
  float u[6], far;
  __device__ __forceinline__ CapSeries(float cap, float unit) {
    const float r = 1.0f / cap, r2 = r * r;
    float c = unit;
    u[0] = c;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      c *= r2;
      u[i + 1] = kCapP[i] * c;
    }
    far = cap >= 0x1p-6f && cap <= 0x1p10f ? kTanhSmall * cap : 0.0f;
  }
  __device__ __forceinline__ float operator()(float s) const {
    float v = u[5];
#pragma unroll
    for (int i = 4; i >= 0; --i) v = __builtin_fmaf(v, s, u[i]);
    return v;
  }
};

// The capped values of four logits: the series where |x| is below 5/8 of the cap
// (within 2 units of the last place), the division and tanhf past it. A value
// takes the same formula whatever its neighbours are.
__device__ __forceinline__ void cap_logits(float (&x)[4], float cap, const CapSeries& series) {
  bool near = true;
#pragma unroll
  for (int e = 0; e < 4; ++e) near = near && __builtin_fabsf(x[e]) < series.far;
  if (__all(near)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= series(x[e] * x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_fabsf(x[e]) < series.far ? x[e] * series(x[e] * x[e]) : cap * tanhf(x[e] / cap);
  }
}

}  // namespace gs

// Microscaled blocks: 32 values share one power of two (E8M0, bias 127, 255
// for a block that holds a NaN or an infinity) and are held in e2m1 (4 bits)
// or e4m3 (8 bits). The shared exponent is floor(log2 of the block's largest
// magnitude) less the element format's largest exponent (2 or 8), at least
// -127, so the largest magnitude lands in the format's top binade; what lies
// past its largest value there (6 or 448) becomes that value, everything else
// is rounded to nearest, ties to the even mantissa. Above the format's smallest
// normal value a rounding is off by at most 2^-4 (8 bits) or 2^-2 (4 bits) of the
// value; one that becomes the largest value, by up to 2^-3 (just below 512) or
// 2^-2 (just below 8): that is the choice of the formats.
#pragma once

#include "gs_internal.h"

namespace gs {

constexpr int kMxBlock = 32;

typedef uint32_t MxU32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t MxU32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any element's alignment (rows of odd strides)
typedef uint32_t MxU32x4Any __attribute__((ext_vector_type(4), aligned(2)));

// 8 values of a row as they lie in memory (bf16: 16 bytes), to be widened later.
template <bool kBf16>
struct Raw8 {
  uint32_t w[kBf16 ? 4 : 8];
  __device__ __forceinline__ void load(const void* p, int64_t e, int n) {
    if (kBf16) {
      const uint16_t* q = (const uint16_t*)p + e;
      if (n >= 8) {
        const MxU32x4Any u = *(const MxU32x4Any*)q;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = u[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = (2 * i < n ? (uint32_t)q[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)q[2 * i + 1] << 16 : 0u);
      }
    } else {
      const uint32_t* q = (const uint32_t*)p + e;
      typedef uint32_t U32x4Any __attribute__((ext_vector_type(4), aligned(4)));
      if (n >= 8) {
        const U32x4Any a = *(const U32x4Any*)q, b = *(const U32x4Any*)(q + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = a[i];
          w[kBf16 ? 0 : 4 + i] = b[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[kBf16 ? 0 : i] = i < n ? q[i] : 0u;
      }
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if (!kBf16) return __uint_as_float(w[i]);
    return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};

// 8 values of a row from element `e` on, `n` of them inside the row (zeros past it).
template <bool kBf16>
__device__ __forceinline__ void load_8(const void* p, int64_t e, int n, float (&v)[8]) {
  if (kBf16) {
    const uint16_t* q = (const uint16_t*)p + e;
    if (n >= 8) {
      const MxU32x4Any u = *(const MxU32x4Any*)q;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? __uint_as_float((uint32_t)q[i] << 16) : 0.0f;
    }
  } else {
    const float* q = (const float*)p + e;
    if (n >= 8) {
      typedef float F32x4Any __attribute__((ext_vector_type(4), aligned(4)));
      const F32x4Any a = *(const F32x4Any*)q, b = *(const F32x4Any*)(q + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? q[i] : 0.0f;
    }
  }
}

// Two floats as bf16, each rounded to nearest even (half a step, 2^-9 of the value's binade top).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));
  const Bf16x2 p = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, p);
}

template <bool kBf16>
__device__ __forceinline__ float rounded_to(float x) {
  return kBf16 ? (float)(__bf16)x : x;
}

template <bool kBf16>
__device__ __forceinline__ void store_8(void* p, int64_t e, int n, const float (&v)[8]) {
  if (kBf16) {
    uint16_t* q = (uint16_t*)p + e;
    const MxU32x4Any u = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    if (n >= 8) {
      *(MxU32x4Any*)q = u;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
    }
  } else {
    float* q = (float*)p + e;
    typedef float F32x4Any __attribute__((ext_vector_type(4), aligned(4)));
    if (n >= 8) {
      *(F32x4Any*)q = F32x4Any{v[0], v[1], v[2], v[3]};
      *(F32x4Any*)(q + 4) = F32x4Any{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = v[i];
    }
  }
}

// The scale code of a block from the bits of its largest magnitude: a NaN's
// bits are above an infinity's, so an integer maximum keeps either.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t amax_bits, int emax) {
  const int e = (int)(amax_bits >> 23);
  return e == 255 ? 255u : (uint32_t)(e > emax ? e - emax : 0);
}

// 2^(127 - code): the factor that brings a block's values into the element
// format's range (exact for every code below 255 of a finite block).
__device__ __forceinline__ float mx_inverse_scale(uint32_t code) { return __uint_as_float((254u - code) << 23); }
// 2^(code - 127), a subnormal for code 0, NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t code) {
  return code == 0 ? __uint_as_float(0x00400000u) : code == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(code << 23);
}

// The largest magnitude's bits over the four lanes that hold a block's 32
// values (8 each, lanes 4k .. 4k + 3).
__device__ __forceinline__ uint32_t mx_block_amax(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = op_max_u32(m, dpp_u32<kDppQuad1032, 0xF>(0u, m));
  return op_max_u32(m, dpp_u32<kDppQuad2301, 0xF>(0u, m));
}

// 8 values at the block's scale as e4m3 codes (a special block: NaN codes).
__device__ __forceinline__ MxU32x2 mx_codes_e4m3(const float (&v)[8], uint32_t code) {
  if (code == 255) return MxU32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
  const float s = mx_inverse_scale(code);
  int lo = 0, hi = 0;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __builtin_amdgcn_fmed3f(v[i] * s, -448.0f, 448.0f);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
  return MxU32x2{(uint32_t)lo, (uint32_t)hi};
}

// 8 values at the block's scale as e2m1 codes, the first in the low bits (a
// special block: zeros, its scale says NaN).
__device__ __forceinline__ uint32_t mx_codes_e2m1(const float (&v)[8], uint32_t code) {
  if (code == 255) return 0u;
  const float s = mx_inverse_scale(code);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __builtin_amdgcn_fmed3f(v[i] * s, -6.0f, 6.0f);
  uint32_t u = 0;
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[0], q[1], 1.0f, 0);
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[2], q[3], 1.0f, 1);
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[4], q[5], 1.0f, 2);
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[6], q[7], 1.0f, 3);
  return u;
}

}  // namespace gs

// Root-mean-square norm with the residual's addition, and its gradients.
//
//   h = x + residual                     (rounded to x's type: what later reads see)
//   y = h * r * (offset + w),  r = 1 / sqrt(mean(h^2) + eps)
//   dh = r (g - h r^2 mean(g h)) + dsummed,  g = dy (offset + w)
//   dw = sum over rows of dy h r
//
// Sums, r and the products are in binary32; y is rounded once, to x's type or
// to e4m3 blocks (gs_mx.h). h is rounded before the norm because the gradient
// and the next block read it so.
//
// A row is held in registers from its one read to its last write: 8 elements a
// thread and piece, so the memory traffic is each input and output once and
// the output may overwrite an input. Memory bound: 8192 x 2048 bf16 with a residual
// 23 us, 5.8 TB/s (a copy: 5.2); the gradient at 4099 x 3840 28 us, 4.5 TB/s and
// 0.5 more for the shares of dw, which take 4.5 us to join; small calls are the
// launches' (1 row of 2048: 2.8 us on the device).
#include "gs_mx.h"

namespace gs {
namespace {

constexpr int kNormThreads = 256;
constexpr int64_t kNormGrid = 1 << 20;  // workgroups a launch; they take more rows in turn

__device__ __forceinline__ uint32_t op_add_f32(uint32_t a, uint32_t b) {
  return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
__device__ __forceinline__ float wave_sum_f32(float x) {
  uint32_t v = __float_as_uint(x);
  GS_WAVE_REDUCE(uint32_t, dpp_u32, v, 0u, op_add_f32);
  return __uint_as_float(readlane_u32(v, 63));
}

// Sums of kCount values over kThreads threads (a wave, or the workgroup), the
// same for every thread and the same order on every call. lds: 4 kCount floats
// that the call before did not use.
template <int kThreads, int kCount>
__device__ __forceinline__ void row_sums(float (&v)[kCount], float* lds) {
#pragma unroll
  for (int c = 0; c < kCount; ++c) v[c] = wave_sum_f32(v[c]);
  if (kThreads == 64) return;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int c = 0; c < kCount; ++c) lds[c * 4 + wave] = v[c];
  }
  lds_barrier();
#pragma unroll
  for (int c = 0; c < kCount; ++c) v[c] = (lds[c * 4] + lds[c * 4 + 1]) + (lds[c * 4 + 2] + lds[c * 4 + 3]);
}

__device__ __forceinline__ void load_weight_8(const void* w, int bf16, int64_t e, int n, float offset, float (&v)[8]) {
  if (bf16) load_8<true>(w, e, n, v);
  else load_8<false>(w, e, n, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += offset;
}

// kThreads threads a row (64: four rows a workgroup), kN pieces of 8 elements a thread.
template <bool kBf16, int kThreads, int kN>
__global__ __launch_bounds__(kNormThreads) void rms_norm_kernel(NormArgs a) {
  __shared__ float lds[2][4];
  int turn = 0;
  const int t = threadIdx.x % kThreads;
  constexpr int kGroups = kNormThreads / kThreads;
  for (int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / kThreads; row < a.rows;
       row += (int64_t)gridDim.x * kGroups) {
    const char* x = (const char*)a.x + row * a.x_stride * (kBf16 ? 2 : 4);
    const char* res = a.residual ? (const char*)a.residual + row * a.residual_stride * (kBf16 ? 2 : 4) : nullptr;
    const int64_t out_at = row * a.width;
    float h[kN][8], w[kN][8];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int e = (i * kThreads + t) * 8, n = a.width - e;
      load_8<kBf16>(x, e, n, h[i]);
      if (res) {
        float r[8];
        load_8<kBf16>(res, e, n, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i][k] = rounded_to<kBf16>(h[i][k] + r[k]);
      }
      load_weight_8(a.weight, a.weight_bf16, e, n, a.offset, w[i]);
    }
    float ss[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s = __builtin_fmaf(h[i][k], h[i][k], s);
      ss[0] += s;
      if (a.summed) {
        const int e = (i * kThreads + t) * 8;
        store_8<kBf16>(a.summed, out_at + e, a.width - e, h[i]);
      }
    }
    row_sums<kThreads, 1>(ss, lds[turn]);
    turn ^= 1;
    const float r = 1.0f / sqrtf(ss[0] / (float)a.width + a.eps);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int e = (i * kThreads + t) * 8, n = a.width - e;
      float y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = h[i][k] * r * w[i][k];
      if (a.out) store_8<kBf16>(a.out, out_at + e, n, y);
      if (a.codes) {  // (the width is a multiple of 32: four neighbouring lanes hold a block, or none of it)
        const uint32_t code = mx_scale_code(mx_block_amax(y), 8);
        if (n > 0) {
          *(MxU32x2*)(a.codes + out_at + e) = mx_codes_e4m3(y, code);
          if ((t & 3) == 0) a.scales[(out_at + e) / kMxBlock] = (uint8_t)code;
        }
      }
    }
  }
}

// Each workgroup (each wave, kThreads 64) takes every n-th row, keeps its
// share of dw in registers and writes it once: `parts` shares in all, joined
// by norm_join_kernel in one order.
template <bool kBf16, int kThreads, int kN>
__global__ __launch_bounds__(kNormThreads) void rms_norm_grad_kernel(NormGradArgs a) {
  constexpr int kGroups = kNormThreads / kThreads, kSize = kBf16 ? 2 : 4;
  __shared__ float lds[2][8];
  // the weights, which wait apart from the rows' values here (a wait for one
  // load covers all that were issued before it); later the waves' shares
  __shared__ __attribute__((aligned(16))) float weights[kThreads * kN * 8];
  int turn = 0;
  const int t = threadIdx.x % kThreads, group = threadIdx.x / kThreads;
  float dw[kN][8];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = 0.0f;
  }
  // The next row's values are on their way while a row is worked on, as far as
  // the registers reach: otherwise each row waits for its own.
  constexpr bool kAhead = kN <= (kBf16 ? 4 : 2);
  const int64_t first = (int64_t)blockIdx.x * kGroups + group, step = (int64_t)gridDim.x * kGroups;
  Raw8<kBf16> h[kN], g[kN], d[kN];
  auto load = [&](int64_t row, Raw8<kBf16>(&h)[kN], Raw8<kBf16>(&g)[kN], Raw8<kBf16>(&d)[kN]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int e = (i * kThreads + t) * 8, n = a.width - e;
      h[i].load((const char*)a.h + row * a.h_stride * kSize, e, n);
      g[i].load((const char*)a.dy + row * a.dy_stride * kSize, e, n);
      if (a.dsummed) d[i].load((const char*)a.dsummed + row * a.dsummed_stride * kSize, e, n);
    }
  };
  if (first < a.rows) load(first, h, g, d);
  for (int c = threadIdx.x * 8; c < kThreads * kN * 8; c += kNormThreads * 8) {
    float w[8];
    load_weight_8(a.weight, a.weight_bf16, c, a.width - c, a.offset, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) weights[c + k] = w[k];
  }
  lds_barrier();
  for (int64_t row = first; row < a.rows; row += step) {
    Raw8<kBf16> h1[kN], g1[kN], d1[kN];
    if (kAhead && row + step < a.rows) load(row + step, h1, g1, d1);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float* w = &weights[(i * kThreads + t) * 8];
      float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s0 = __builtin_fmaf(h[i][k], h[i][k], s0);
        s1 = __builtin_fmaf(g[i][k] * w[k], h[i][k], s1);
      }
      s[0] += s0;
      s[1] += s1;
    }
    row_sums<kThreads, 2>(s, lds[turn]);
    turn ^= 1;
    const float r = 1.0f / sqrtf(s[0] / (float)a.width + a.eps);
    const float c = r * r * (s[1] / (float)a.width);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int e = (i * kThreads + t) * 8, n = a.width - e;
      if (a.dx) {
        const float* w = &weights[e];
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = r * (g[i][k] * w[k] - h[i][k] * c);
          if (a.dsummed) v[k] += d[i][k];
        }
        store_8<kBf16>(a.dx, row * a.width + e, n, v);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) dw[i][k] = __builtin_fmaf(g[i][k], h[i][k] * r, dw[i][k]);
    }
    if (kAhead) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        h[i] = h1[i];
        g[i] = g1[i];
        d[i] = d1[i];
      }
    } else if (row + step < a.rows) {
      load(row + step, h, g, d);
    }
  }
  if (!a.parts) return;
  if (kGroups > 1) {
    // the waves' shares one after another
    float* joined = weights;
    __syncthreads();
    for (int w = 0; w < kGroups; ++w) {
      if (group == w) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float* p = &joined[(i * kThreads + t) * 8 + k];
            *p = w == 0 ? dw[i][k] : *p + dw[i][k];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.width; c += kNormThreads) a.parts[(int64_t)blockIdx.x * a.width + c] = joined[c];
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int e = (i * kThreads + t) * 8;
      store_8<false>(a.parts, (int64_t)blockIdx.x * a.width + e, a.width - e, dw[i]);
    }
  }
}

// dw[c] = sum over the shares: 32 columns a workgroup, 32 slices of shares.
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* __restrict__ parts, int n_parts, int width,
                                                         float* __restrict__ dw) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, slice = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float s = 0.0f;
  if (col < width) {
#pragma unroll 8
    for (int p = slice; p < n_parts; p += 32) s += parts[(int64_t)p * width + col];
  }
  sums[slice][c] = s;
  __syncthreads();
  if (slice == 0 && col < width) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) total += sums[i][c];
    dw[col] = total;
  }
}

__global__ __launch_bounds__(256) void fill_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

template <bool kBf16>
void norm_forward(const NormArgs& a, hipStream_t s) {
  const bool wave = norm_wave_rows(a.rows, a.width);
  const int threads = wave ? 64 : 256, n = (a.width + threads * 8 - 1) / (threads * 8);
  const int64_t groups = wave ? ((int64_t)a.rows + 3) / 4 : a.rows;
  const dim3 grid((unsigned)(groups < kNormGrid ? groups : kNormGrid)), block(kNormThreads);
  switch ((wave ? 100 : 0) + n) {
#define GS_CASE(c, th, n_)                                                     \
  case c:                                                                      \
    rms_norm_kernel<kBf16, th, n_><<<grid, block, 0, s>>>(a);                  \
    break;
    GS_CASE(101, 64, 1) GS_CASE(102, 64, 2) GS_CASE(103, 64, 3) GS_CASE(104, 64, 4)
    GS_CASE(1, 256, 1) GS_CASE(2, 256, 2) GS_CASE(3, 256, 3) GS_CASE(4, 256, 4)
    GS_CASE(5, 256, 5) GS_CASE(6, 256, 6) GS_CASE(7, 256, 7) GS_CASE(8, 256, 8)
#undef GS_CASE
  }
}

template <bool kBf16>
void norm_backward(const NormGradArgs& a, hipStream_t s) {
  const bool wave = norm_wave_rows(a.rows, a.width);
  const int threads = wave ? 64 : 256, n = (a.width + threads * 8 - 1) / (threads * 8);
  const dim3 grid((unsigned)norm_parts(a.rows, a.width)), block(kNormThreads);
  switch ((wave ? 100 : 0) + n) {
#define GS_CASE(c, th, n_)                                                     \
  case c:                                                                      \
    rms_norm_grad_kernel<kBf16, th, n_><<<grid, block, 0, s>>>(a);             \
    break;
    GS_CASE(101, 64, 1) GS_CASE(102, 64, 2) GS_CASE(103, 64, 3) GS_CASE(104, 64, 4)
    GS_CASE(1, 256, 1) GS_CASE(2, 256, 2) GS_CASE(3, 256, 3) GS_CASE(4, 256, 4)
    GS_CASE(5, 256, 5) GS_CASE(6, 256, 6) GS_CASE(7, 256, 7) GS_CASE(8, 256, 8)
#undef GS_CASE
  }
}

}  // namespace

// Many narrow rows: a wave a row (no barrier). Few, or wide: a workgroup a row
// (the forward pass of 8192 rows of 2048: 28.4 us, and 30.4 with a wave a row; the
// gradient follows it, unmeasured the other way).
bool norm_wave_rows(int32_t rows, int32_t width) { return rows >= 2048 && width <= 1024; }

// Workgroups of the gradient's kernel: as many shares of dw. About 768, three a
// compute unit of this card (4099 rows of 3840, the one size it was chosen at: 37.7 us,
// with 512 41.6, with 1024 45.1), and as many rows for each as can be alike.
int32_t norm_parts(int32_t rows, int32_t width) {
  const int32_t groups = norm_wave_rows(rows, width) ? rows / 4 + (rows % 4 != 0) : rows;
  const int32_t each = groups < 1152 ? 1 : groups / 768 + (groups % 768 >= 384);
  return groups / each + (groups % each != 0);
}

void launch_rms_norm(const NormArgs& a, bool bf16, hipStream_t s) {
  if (bf16) norm_forward<true>(a, s);
  else norm_forward<false>(a, s);
}

void launch_rms_norm_grad(const NormGradArgs& a, bool bf16, float* dweight, hipStream_t s) {
  if (bf16) norm_backward<true>(a, s);
  else norm_backward<false>(a, s);
  if (a.parts)
    norm_join_kernel<<<dim3((unsigned)((a.width + 31) / 32)), dim3(1024), 0, s>>>(
        a.parts, norm_parts(a.rows, a.width), a.width, dweight);
}

void launch_fill_zero(void* p, int64_t bytes, hipStream_t s) {
  const int64_t n = bytes / 2, blocks = (n + 255) / 256;
  fill_zero_kernel<<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s>>>((uint16_t*)p, n);
}

}  // namespace gs

// Microscaled blocks (gs_mx.h): quantisation, reading back, and the lm_head
// over e2m1 weights and e4m3 hidden states.
#include "gs_cap.h"
#include "gs_mx.h"

namespace gs {
namespace {

// ------------------------------------------------- values <-> codes
// One thread 8 values, four threads a block. Memory bound: a value is read
// once and its code and scale written once.
constexpr int kMxThreads = 256;

template <bool kBf16, bool kFp4>
__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(const void* __restrict__ x, int64_t n_groups,
                                                                 int32_t row_groups, int64_t row_stride,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales) {
  const int64_t at = (int64_t)blockIdx.x * kMxThreads + threadIdx.x;  // group of 8 values
  if (at >= n_groups) return;  // (a multiple of 4: whole blocks stay or go)
  int64_t e = at * 8;
  if (row_stride != (int64_t)row_groups * 8) {
    const int64_t row = at / row_groups;
    e = row * row_stride + (at - row * row_groups) * 8;
  }
  float v[8];
  load_8<kBf16>(x, e, 8, v);
  const uint32_t code = mx_scale_code(mx_block_amax(v), kFp4 ? 2 : 8);
  if (kFp4) ((uint32_t*)codes)[at] = mx_codes_e2m1(v, code);
  else ((MxU32x2*)codes)[at] = mx_codes_e4m3(v, code);
  if ((threadIdx.x & 3) == 0) scales[at >> 2] = (uint8_t)code;
}

template <bool kBf16, bool kFp4>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales,
                                                                   int64_t n_groups, void* __restrict__ out) {
  typedef float F32x2 __attribute__((ext_vector_type(2)));
  const int64_t at = (int64_t)blockIdx.x * kMxThreads + threadIdx.x;
  if (at >= n_groups) return;
  const float s = mx_scale(scales[at >> 2]);
  F32x2 p[4];
  if (kFp4) {
    const uint32_t u = ((const uint32_t*)codes)[at];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 3);
  } else {
    const MxU32x2 u = ((const MxU32x2*)codes)[at];
    p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)u.x, false);
    p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)u.x, true);
    p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)u.y, false);
    p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)u.y, true);
  }
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = p[i].x * s;
    v[2 * i + 1] = p[i].y * s;
  }
  store_8<kBf16>(out, at * 8, 8, v);
}

// ------------------------------------------------- the 4-bit head
// logits[m][v] = cap(sum over blocks of 2^(sh + sw) sum_k h[m][k] w[v][k]) on
// v_mfma_scale_f32_16x16x128_f8f6f4 (the scales are its operands), tiles of
// 256 vocabulary rows by kCols hidden rows, 8 waves, 256 columns of K a stage.
//
// K order: the instruction multiplies four blocks of 32 at a time, one a group
// of 16 lanes. Step s (of two) of a stage takes blocks s, 2 + s, 4 + s, 6 + s,
// so the two blocks of a lane group lie side by side: 32 bytes of a row of W,
// and one 2-byte load of their scales, picked by the instruction's selector.
// The 8-bit operand's lane (j, g) holds the half g & 1 of the hardware blocks
// g / 2 and 2 + g / 2.
constexpr int kHeadThreads = 512;
constexpr int kHeadRows = 256;   // vocabulary rows a tile
constexpr int kHeadK = 256;      // columns a stage
constexpr int kHeadStride = kHeadRows + 4;  // LDS floats per staged output row

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* LdsPtr;

template <int kCols>
struct HeadTile {
  static constexpr int kWavesV = kCols == 128 ? 4 : 8;
  static constexpr int kWavesM = 8 / kWavesV;
  static constexpr int kRT = 16 / kWavesV;            // 16-row tiles of W a wave
  static constexpr int kCT = kCols / 16 / kWavesM;    // 16-row tiles of H a wave
  static constexpr int kStages = kCols == 128 ? 2 : 3;
  static constexpr int kW = kHeadRows * 128;          // bytes of a stage: codes of W,
  static constexpr int kH = kCols * 256;              // of H,
  static constexpr int kWS = kHeadRows * 16;          // scales of W (a dword holds a pair),
  static constexpr int kHS = kCols * 16;              // of H
  static constexpr int kStage = kW + kH + kWS + kHS;
  static constexpr int kFetches = 4 + kCols / 32 + 3; // memory instructions of a wave and stage
  static constexpr int kHeadLds = kStages * kStage + 256;  // and where waves without scales of H put theirs
};

struct HeadOffsets {
  uint32_t w[4], h[4], ws[2], hs;     // this lane's byte offsets in a stage's rows
  uint32_t w_tail, h_tail[2], s_tail; // kBufferOutOfRange where the last stage has no such columns
};

template <int kCols, typename Rsrc>
__device__ __forceinline__ void head_fetch(char* lds, char* spare, int wave, Rsrc wr, Rsrc hr, Rsrc wsr, Rsrc hsr,
                                           const HeadOffsets& o, uint32_t k, bool tail, bool none) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef HeadTile<kCols> T;
  const uint32_t off = none ? kBufferOutOfRange : 0u;
  const uint32_t wt = off | (tail ? o.w_tail : 0u), st = off | (tail ? o.s_tail : 0u);
  const uint32_t ht[2] = {off | (tail ? o.h_tail[0] : 0u), off | (tail ? o.h_tail[1] : 0u)};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (LdsPtr)(lds + 4096 * wave + 1024 * i), 16, o.w[i] | wt, k * 128, 0, 0);
  char* h = lds + T::kW;
#pragma unroll
  for (int i = 0; i < kCols / 32; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(hr, (LdsPtr)(h + 32 * kCols * wave + 1024 * i), 16, o.h[i] | ht[i & 1],
                                             k * 256, 0, 0);
  char* ws = h + T::kH;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (LdsPtr)(ws + 512 * wave + 256 * i), 2, o.ws[i] | st, k * 8, 0, 0);
  char* hs = 16 * wave < kCols ? ws + T::kWS + 256 * wave : spare;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(hsr, (LdsPtr)hs, 2, o.hs | st, k * 8, 0, 0);
#endif
}

// One stage: the next fetches go out, then two steps of 128 columns.
template <int kCols, typename Rsrc>
__device__ __forceinline__ void head_block(const char* __restrict__ cur, char* __restrict__ next, char* spare, int wave,
                                           int wv, int wm, int j, int g, Rsrc wr, Rsrc hr, Rsrc wsr, Rsrc hsr,
                                           const HeadOffsets& o, uint32_t k, bool tail, bool none,
                                           f32x4 (&acc)[HeadTile<kCols>::kRT][HeadTile<kCols>::kCT]) {
  typedef HeadTile<kCols> T;
  head_fetch<kCols>(next, spare, wave, wr, hr, wsr, hsr, o, k, tail, none);
  const char* w = cur + (16 * T::kRT * wv + j) * 128;
  const char* h = cur + T::kW + (16 * T::kCT * wm + j) * 256;
  const int* ws = (const int*)(cur + T::kW + T::kH) + (16 * T::kRT * wv + j) * 4 + g;
  const int* hs = (const int*)(cur + T::kW + T::kH + T::kWS) + (16 * T::kCT * wm + j) * 4 + g;
  int sw[T::kRT], sh[T::kCT];
#pragma unroll
  for (int a = 0; a < T::kRT; ++a) sw[a] = ws[64 * a];
#pragma unroll
  for (int b = 0; b < T::kCT; ++b) sh[b] = hs[64 * b];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    i32x8 x[T::kRT], y[T::kCT];
#pragma unroll
    for (int a = 0; a < T::kRT; ++a) {
      const i32x4 c = *(const i32x4*)(w + 2048 * a + (((2 * g + s) ^ (j & 7)) * 16));
      x[a] = __builtin_shufflevector(c, c, 0, 1, 2, 3, -1, -1, -1, -1);
    }
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) {
      const int c = ((4 * (g >> 1) + 2 * s + (g & 1)) ^ (j & 7)) * 16;
      const i32x4 lo = *(const i32x4*)(h + 4096 * b + c), hi = *(const i32x4*)(h + 4096 * b + c + 128);
      y[b] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
      for (int b = 0; b < T::kCT; ++b) {
        if (s == 0) acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[a], y[b], acc[a][b], 4, 0, 0, sw[a], 0, sh[b]);
        else acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[a], y[b], acc[a][b], 4, 0, 1, sw[a], 1, sh[b]);
      }
    }
  }
}

template <int kCols>
__global__ __launch_bounds__(kHeadThreads, 2) void mx_head_kernel(
    const uint8_t* __restrict__ H, const uint8_t* __restrict__ HS, const uint8_t* __restrict__ W,
    const uint8_t* __restrict__ WS, int M, int D, int V, int m_blocks, int wide, float cap, float* __restrict__ out) {
  typedef HeadTile<kCols> T;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // consecutive workgroups go to the XCDs in turn: an XCD takes the row
  // blocks of one tile of W one after another
  const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
  const int vt = (local / m_blocks) * 8 + xcd;
  const int64_t v0 = (int64_t)vt * kHeadRows, m0 = (int64_t)(local % m_blocks) * kCols;
  if (v0 >= V) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, g = lane >> 4, wv = wave % T::kWavesV, wm = wave / T::kWavesV;
  const int v_rows = V - v0 < kHeadRows ? (int)(V - v0) : kHeadRows;
  const int m_rows = M - m0 < kCols ? (int)(M - m0) : kCols;
  const int ds = D / 32;
  // rows past V or M read zeros (and scales of 2^-127)
  const __amdgpu_buffer_rsrc_t wr =
      __builtin_amdgcn_make_buffer_rsrc((void*)(W + (size_t)v0 * (D / 2)), (short)0, v_rows * (D / 2), kBufferWord3);
  const __amdgpu_buffer_rsrc_t hr =
      __builtin_amdgcn_make_buffer_rsrc((void*)(H + (size_t)m0 * D), (short)0, m_rows * D, kBufferWord3);
  const __amdgpu_buffer_rsrc_t wsr =
      __builtin_amdgcn_make_buffer_rsrc((void*)(WS + (size_t)v0 * ds), (short)0, v_rows * ds, kBufferWord3);
  const __amdgpu_buffer_rsrc_t hsr =
      __builtin_amdgcn_make_buffer_rsrc((void*)(HS + (size_t)m0 * ds), (short)0, m_rows * ds, kBufferWord3);
  // Fetched rows: 16-byte chunk c of row r lands at chunk c ^ (r & 7), so that
  // the lanes of an operand read that go together hit different banks.
  HeadOffsets o;
  const int nk = (D + kHeadK - 1) / kHeadK, last_k = D - (nk - 1) * kHeadK;  // columns of the last stage
  {
    const int r = lane >> 3, c = (lane & 7) ^ r;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.w[i] = (uint32_t)((32 * wave + 8 * i + r) * (D / 2) + 16 * c);
    o.w_tail = 32 * c < last_k ? 0u : kBufferOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (kCols / 8) * wave + 4 * i + (lane >> 4), c = (lane & 15) ^ (row & 7);
    o.h[i] = (uint32_t)(row * D + 16 * c);
    if (i < 2) o.h_tail[i] = 16 * c < last_k ? 0u : kBufferOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) o.ws[i] = (uint32_t)(((2 * wave + i) * 16 + (lane >> 2)) * ds + 2 * (lane & 3));
  o.hs = 16 * wave < kCols ? (uint32_t)((16 * wave + (lane >> 2)) * ds + 2 * (lane & 3)) : kBufferOutOfRange;
  o.s_tail = 64 * (lane & 3) < last_k ? 0u : kBufferOutOfRange;

  f32x4 acc[T::kRT][T::kCT];
#pragma unroll
  for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  char* spare = lds + T::kStages * T::kStage;
  // tiles start at different columns: their reads spread over the memory channels
  const int first = vt % nk;
  auto at = [&](int kb) __attribute__((always_inline)) {
    const int k = (kb < nk ? kb : 0) + first;
    return k < nk ? k : k - nk;
  };
  auto partial = [&](int k) __attribute__((always_inline)) { return k == nk - 1 && last_k < kHeadK; };
#pragma unroll
  for (int u = 0; u < T::kStages - 1; ++u)
    head_fetch<kCols>(lds + u * T::kStage, spare, wave, wr, hr, wsr, hsr, o, (uint32_t)at(u), partial(at(u)), u >= nk);
  for (int kb = 0; kb < nk; kb += T::kStages) {
#pragma unroll
    for (int u = 0; u < T::kStages; ++u) {
      if (kb + u < nk) {
        // the stage has landed for every wave, and every wave has read the one before
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((T::kStages - 2) * T::kFetches) : "memory");
        const int n = kb + u + T::kStages - 1, k = at(n);
        head_block<kCols>(lds + u * T::kStage, lds + (u + T::kStages - 1) % T::kStages * T::kStage, spare, wave, wv, wm, j,
                          g, wr, hr, wsr, hsr, o, (uint32_t)k, partial(k), n >= nk, acc);
      }
    }
  }
  // nothing is in flight to or from LDS before the outputs take its place
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // the cap, then the tile through LDS, so that rows go out in pieces of 1 KB
  // (lane (j, g) holds column j of H's rows, rows 4 g + e of W's)
  float* stage = (float*)lds;
  const float rcap = reciprocal_of_cap(cap);
#pragma unroll
  for (int b = 0; b < T::kCT; ++b) {
#pragma unroll
    for (int a = 0; a < T::kRT; ++a) {
      float x[4] = {acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
      if (cap > 0.0f) lmhead_cap<4>(x, cap, rcap);
      *(f32x4*)&stage[(16 * (T::kCT * wm + b) + j) * kHeadStride + 16 * (T::kRT * wv + a) + 4 * g] =
          f32x4{x[0], x[1], x[2], x[3]};
    }
  }
  __syncthreads();
  float* p = out + (size_t)m0 * V + v0;
  if (wide) {  // V % 4 == 0 and 16-byte aligned logits: a piece lies within its row
    for (int q = tid; q < m_rows * (kHeadRows / 4); q += kHeadThreads) {
      const int row = q / (kHeadRows / 4), c = 4 * (q % (kHeadRows / 4));
      if (c < v_rows)
        __builtin_nontemporal_store(*(const f32x4*)&stage[row * kHeadStride + c], (f32x4*)&p[(size_t)row * V + c]);
    }
  } else {
    for (int q = tid; q < m_rows * kHeadRows; q += kHeadThreads) {
      const int row = q / kHeadRows, c = q % kHeadRows;
      if (c < v_rows) __builtin_nontemporal_store(stage[row * kHeadStride + c], &p[(size_t)row * V + c]);
    }
  }
}

template <int kCols>
void head_launch(const uint8_t* H, const uint8_t* HS, const uint8_t* W, const uint8_t* WS, int32_t m, int32_t width,
                 int32_t vocab, float cap, float* out, hipStream_t s, LaunchEvents ev) {
  typedef HeadTile<kCols> T;
  constexpr int kOut = kCols * kHeadStride * 4;
  constexpr int kBytes = T::kHeadLds > kOut ? T::kHeadLds : kOut;
  static_assert(kBytes <= 160 * 1024, "LDS of a compute unit");
  const int m_blocks = (m + kCols - 1) / kCols, v_tiles = (vocab + kHeadRows - 1) / kHeadRows;
  const dim3 grid((unsigned)((v_tiles + 7) / 8 * 8 * m_blocks)), block(kHeadThreads);
  const int wide = vocab % 4 == 0 && ((uintptr_t)out & 15) == 0;
  hipExtLaunchKernelGGL((mx_head_kernel<kCols>), grid, block, kBytes, s, ev.start, ev.stop, 0, H, HS, W, WS, m, width,
                        vocab, m_blocks, wide, cap, out);
}

}  // namespace

void launch_mx_quantize(const void* x, bool bf16, int32_t format, int64_t rows, int32_t width, int64_t row_stride,
                        uint8_t* codes, uint8_t* scales, hipStream_t s) {
  const int64_t groups = rows * (width / 8);
  const dim3 grid((unsigned)((groups + kMxThreads - 1) / kMxThreads)), block(kMxThreads);
  if (rows == 1) row_stride = width;
#define GS_CASE(b, f) mx_quantize_kernel<b, f><<<grid, block, 0, s>>>(x, groups, width / 8, row_stride, codes, scales)
  if (format == GS_MX_E2M1) {
    if (bf16) GS_CASE(true, true);
    else GS_CASE(false, true);
  } else {
    if (bf16) GS_CASE(true, false);
    else GS_CASE(false, false);
  }
#undef GS_CASE
}

void launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int32_t format, int64_t rows, int32_t width,
                          bool bf16, void* out, hipStream_t s) {
  const int64_t groups = rows * (width / 8);
  const dim3 grid((unsigned)((groups + kMxThreads - 1) / kMxThreads)), block(kMxThreads);
#define GS_CASE(b, f) mx_dequantize_kernel<b, f><<<grid, block, 0, s>>>(codes, scales, groups, out)
  if (format == GS_MX_E2M1) {
    if (bf16) GS_CASE(true, true);
    else GS_CASE(false, true);
  } else {
    if (bf16) GS_CASE(true, false);
    else GS_CASE(false, false);
  }
#undef GS_CASE
}

void launch_mx_lmhead(const uint8_t* hidden, const uint8_t* hidden_scales, const uint8_t* weight,
                      const uint8_t* weight_scales, int32_t m, int32_t width, int32_t vocab, float softcap, float* out,
                      hipStream_t s, LaunchEvents ev) {
  if (m <= 32) head_launch<32>(hidden, hidden_scales, weight, weight_scales, m, width, vocab, softcap, out, s, ev);
  else if (m <= 64) head_launch<64>(hidden, hidden_scales, weight, weight_scales, m, width, vocab, softcap, out, s, ev);
  else head_launch<128>(hidden, hidden_scales, weight, weight_scales, m, width, vocab, softcap, out, s, ev);
}

}  // namespace gs

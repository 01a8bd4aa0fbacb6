// Softmax cross entropy of the head's logits, and its gradients, without the
// logits in memory:
//   z = cap(H W^T),  lse[m] = log sum_v exp z[m][v],  loss[m] = lse[m] - z[m][t[m]]
//   g[m][v] = dloss[m] / most (exp(z[m][v] - lse[m]) - [v = t[m]]) (1 - (z[m][v] / cap)^2)
//   dH = most g W,  dW = most g^T H,  most = max |dloss|
//
// Four products on v_mfma_f32_16x16x32_bf16 with one main loop (tiles of 256
// rows by kCols columns, 8 waves, 64 of the summed index a stage, operands by
// the memory pipe straight into LDS):
//   kStats   W x H, the epilogue leaves a (max, sum) per hidden row and tile;
//   kGrad    W x H again, a piece of the vocabulary, the epilogue writes g in
//            bf16 (the matrix cores read 16 bits: half a step of 2^-8 a value, the
//            sums are binary32). The largest |dloss| stays out of g: where every
//            row has the same, as in a mean, a row's largest value, at the target,
//            is then near -1, which bf16 holds, and not a product whose rounding
//            all rows share (dW's error at M 4096 was 1.7 times its own rounding's);
//   kHidden  W^T x g, summed over the piece, in shares of its vocabulary rows;
//   kWeight  H^T x g^T, summed over the hidden rows.
// kHidden and kWeight sum over an operand's rows: those tiles lie in LDS as
// they do in memory and are transposed by the LDS reads (ds_read_b64_tr_b16).
#include <algorithm>

#include "gs_cap.h"
#include "gs_mx.h"

namespace gs {
namespace {

enum Pass { kStats, kGrad, kHidden, kWeight };

constexpr int kRows = 256;  // rows of a tile (vocabulary rows; columns of K in kHidden and kWeight)
constexpr int kBlock = 64;  // of the summed index a stage
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLowest = -1.0e38f;  // a maximum over nothing; times log2(e) still finite

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* LdsPtr;
typedef __attribute__((address_space(3))) i16x4* LdsTrPtr;

struct LossArgs {
  const uint16_t* W;   // the piece's first row
  const uint16_t* H;
  uint16_t* G;         // [M][g_stride]
  const int32_t* targets;
  const float* lse;
  const float* dloss;
  const float* most;   // the largest |dloss| of the scored rows
  float2* stats;       // kStats: [v_tiles][M]
  float* part;         // kHidden: [splits][M][D]
  uint16_t* dW;        // kWeight: the piece's first row
  float cap;
  int32_t M, D, V;     // V: vocabulary rows of the piece
  int32_t v_base;      // the piece's first vocabulary row
  int32_t vocab;
  int32_t g_stride;    // a multiple of 256, at least V
  int32_t row_tiles, col_tiles, splits, split_rows;  // split_rows: vocabulary rows a share, a multiple of 64
  int32_t accumulate;  // kHidden: add to the shares of the pieces before
};

struct Column {
  int32_t target;  // negative: not scored
  float ll;        // -lse log2(e)
  float share;     // dloss over the largest |dloss|
};

template <Pass kPass, int kCols>
struct Tile {
  static constexpr bool kTrA = kPass == kHidden || kPass == kWeight, kTrB = kPass == kWeight;
  // 256 columns are bound by the matrix cores: 4 waves of 128 x 128, one a SIMD
  // with the registers of two, read an LDS byte for the fewest products. Fewer
  // columns are bound by memory: 8 waves, and more stages under way.
  static constexpr bool kWide = kCols == 256;
  static constexpr int kWaves = kWide ? 4 : 8, kThreads = 64 * kWaves;
  static constexpr int kWavesR = kWide ? 2 : kCols == 128 ? 4 : 8;
  static constexpr int kWavesC = kWaves / kWavesR;
  static constexpr int kRT = 16 / kWavesR;          // 16-row tiles a wave
  static constexpr int kCT = kCols / 16 / kWavesC;  // 16-column tiles a wave
  static constexpr int kStages = kWide ? 2 : 3;
  static constexpr int kA = kRows * kBlock * 2, kB = kCols * kBlock * 2;
  static constexpr int kStage = kA + kB;
  static constexpr int kFetchA = 32 / kWaves, kFetchB = kCols / 8 / kWaves;  // wave instructions of 1 KB
  static constexpr int kFetches = kFetchA + kFetchB;
  static constexpr int kOutStride = 256 + 8;        // 16-bit values a staged output row
  static constexpr int kOut = kPass == kGrad || kPass == kWeight ? kCols * kOutStride * 2 : 0;
  static constexpr int kOperands = kWide ? 5 * kA : kStages * kStage;  // (kWide: kA == kB)
  static constexpr int kColumns = kPass == kGrad ? kCols * (int)sizeof(Column) : 0;
  static constexpr int kLds = kOperands > kOut + kColumns ? kOperands : kOut + kColumns;
  static_assert(kLds <= 160 * 1024, "LDS of a compute unit");
};

// The position of 16-byte chunk pairs in a transposed tile's row: the 8 rows
// that a half wave reads together (4 of each of two lane groups) take 8
// different pairs of the banks.
__device__ __forceinline__ int pair_swizzle(int row) { return (row & 3) | ((row >> 1) & 4); }

// A stage's fetches of one operand: kN wave instructions of 1 KB.
template <int kN, typename Rsrc>
__device__ __forceinline__ void loss_fetch(Rsrc r, char* lds, const uint32_t (&off)[kN], uint32_t k) {
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
  for (int i = 0; i < kN; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)(lds + 1024 * i), 16, off[i], k, 0, 0);
#endif
}

// Operand tile t's values of the summed index 32 s + 8 g .. + 7 for lane (j, g).
template <bool kTr>
__device__ __forceinline__ bf16x8 loss_operand(const char* p, int t, int s, uint32_t pos0, uint32_t pos1) {
  if (!kTr) return *(const bf16x8*)(p + 2048 * t + (s ? pos1 : pos0));
#ifdef __HIP_DEVICE_COMPILE__
  // pos0: this lane's row and place in a pair, pos1: its swizzle
  const char* q = p + s * 16384 + pos0 + ((32 * (uint32_t)t) ^ pos1);
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTrPtr)q);
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTrPtr)(q + 2048));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
  return bf16x8{};
#endif
}

// One stage of the narrow tiles: the next fetches go out, then two steps of 32.
template <Pass kPass, int kCols, typename Rsrc>
__device__ __forceinline__ void loss_block(const char* __restrict__ a, const char* __restrict__ b,
                                           char* __restrict__ a_next, char* __restrict__ b_next, Rsrc ar, Rsrc br,
                                           const uint32_t (&a_off)[Tile<kPass, kCols>::kFetchA],
                                           const uint32_t (&b_off)[Tile<kPass, kCols>::kFetchB], uint32_t ak,
                                           uint32_t bk, int a_tile, int b_tile, const uint32_t (&a_pos)[2],
                                           const uint32_t (&b_pos)[2],
                                           f32x4 (&acc)[Tile<kPass, kCols>::kRT][Tile<kPass, kCols>::kCT]) {
  typedef Tile<kPass, kCols> T;
  loss_fetch<T::kFetchA>(ar, a_next, a_off, ak);
  loss_fetch<T::kFetchB>(br, b_next, b_off, bk);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    bf16x8 x[T::kRT], y[T::kCT];
#pragma unroll
    for (int i = 0; i < T::kRT; ++i) x[i] = loss_operand<T::kTrA>(a, a_tile + i, s, a_pos[0], a_pos[1]);
#pragma unroll
    for (int i = 0; i < T::kCT; ++i) y[i] = loss_operand<T::kTrB>(b, b_tile + i, s, b_pos[0], b_pos[1]);
#pragma unroll
    for (int i = 0; i < T::kRT; ++i) {
#pragma unroll
      for (int c = 0; c < T::kCT; ++c)
        acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y[c], acc[i][c], 0, 0, 0);
    }
  }
}

// Half a stage of the wide tile: 64 products of the operands in registers and,
// in a fixed order between them, the reads of the next half's operands from `a`
// and `b` (the columns' first: every product of the next half's first eighth
// needs them) and the fetches of one operand's tile of a later stage (kSlots of
// the 16 places for them). Left to the compiler, the fetches go out in one run
// that the matrix core waits for (dH's product at M 4096, D 2048, 32768
// vocabulary rows took 490 us).
template <Pass kPass, int kSlots, typename Rsrc>
__device__ __forceinline__ void loss_half(const char* __restrict__ a, const char* __restrict__ b,
                                          char* __restrict__ next, Rsrc rsrc, const uint32_t (&off)[8], uint32_t k,
                                          int s, int a_tile, int b_tile, const uint32_t (&a_pos)[2],
                                          const uint32_t (&b_pos)[2], const bf16x8 (&x)[8], const bf16x8 (&y)[8],
                                          bf16x8 (&x_next)[8], bf16x8 (&y_next)[8], f32x4 (&acc)[8][8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
#ifdef __HIP_DEVICE_COMPILE__
      typedef Tile<kPass, 256> T;
      if (h < 2) {
        const int t = 2 * (i & 3) + h;
        if (i < 4) y_next[t] = loss_operand<T::kTrB>(b, b_tile + t, s, b_pos[0], b_pos[1]);
        else x_next[t] = loss_operand<T::kTrA>(a, a_tile + t, s, a_pos[0], a_pos[1]);
      } else {
        const int slot = 2 * i + h - 2, n = slot * 8 / kSlots;
        if (n < 8 && slot * 8 % kSlots == 0)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsPtr)(next + 1024 * n), 16, off[n], k, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
#endif
      acc[i][2 * h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y[2 * h], acc[i][2 * h], 0, 0, 0);
      acc[i][2 * h + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y[2 * h + 1], acc[i][2 * h + 1], 0, 0, 0);
#ifdef __HIP_DEVICE_COMPILE__
      __builtin_amdgcn_sched_barrier(0);
#endif
    }
  }
}

// The cap, x -> cap tanh(x / cap). Below 5/8 of the cap tanh q = q (1 + s P(s)),
// s = q^2, P of degree 4 fitted over that range (relative error 2^-27); past it
// 1 - 2 / (e^2q + 1). Either is within 2e-7 of the cap.
__device__ __forceinline__ float cap_series(float s) {
  float u = -0x1.75e194p-8f;
  u = __builtin_fmaf(u, s, 0x1.52268ep-6f);
  u = __builtin_fmaf(u, s, -0x1.b83c58p-5f);
  u = __builtin_fmaf(u, s, 0x1.110726p-3f);
  u = __builtin_fmaf(u, s, -0x1.555532p-2f);
  return __builtin_fmaf(u, s, 1.0f);
}
__device__ __forceinline__ float cap_far(float q) {
  return 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(q * (2.0f * kLog2e)) + 1.0f);
}

// The smallest and the largest of a lane's values of one column.
template <int kRT, int kCT>
__device__ __forceinline__ void column_range(const f32x4 (&acc)[kRT][kCT], int b, float& lo, float& hi) {
  lo = __builtin_inff();
  hi = -__builtin_inff();
#pragma unroll
  for (int a = 0; a < kRT; ++a) {
    const f32x4 x = acc[a][b];
    hi = __builtin_fmaxf(__builtin_fmaxf(hi, x[0]), x[1]);
    hi = __builtin_fmaxf(__builtin_fmaxf(hi, x[2]), x[3]);
    lo = __builtin_fminf(__builtin_fminf(lo, x[0]), x[1]);
    lo = __builtin_fminf(__builtin_fminf(lo, x[2]), x[3]);
  }
}

// A (max, sum of exponentials over it) pair with another's.
__device__ __forceinline__ void join_sums(float& mx, float& sum, float om, float os) {
  const float nm = __builtin_fmaxf(mx, om);
  sum = sum * __builtin_amdgcn_exp2f((mx - nm) * kLog2e) + os * __builtin_amdgcn_exp2f((om - nm) * kLog2e);
  mx = nm;
}

template <Pass kPass, int kCols, bool kCap>
__global__ __launch_bounds__((Tile<kPass, kCols>::kThreads), (Tile<kPass, kCols>::kWide ? 1 : 2)) void loss_kernel(
    LossArgs p) {
  typedef Tile<kPass, kCols> T;
  __shared__ __attribute__((aligned(16))) char lds[T::kLds];
  // An XCD (consecutive workgroups go to them in turn) takes a run of adjacent
  // tiles, so its workgroups share their operands' lines in its L2: four row
  // tiles by all column tiles (kStats, kGrad), all row tiles by a run of
  // column tiles (kHidden, kWeight).
  const int total = p.row_tiles * p.col_tiles * p.splits;
  int id = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  if (id >= total) return;
  int rt, ct, split = 0;
  if (kPass == kStats || kPass == kGrad) {
    const int group = id / (4 * p.col_tiles) * 4;
    const int in = p.row_tiles - group < 4 ? p.row_tiles - group : 4;
    id -= group * p.col_tiles;
    rt = group + id % in;
    ct = id / in;
  } else {
    rt = id % p.row_tiles;
    id /= p.row_tiles;
    ct = id % p.col_tiles;
    split = id / p.col_tiles;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, g = lane >> 4, wr = wave % T::kWavesR, wc = wave / T::kWavesR;
  const int M = p.M, D = p.D, V = p.V;
  const int r0 = rt * kRows, c0 = ct * kCols;

  // kGrad: what the epilogue needs of column tid, read now and kept
  Column column{-1, 0.0f, 0.0f};
  if (kPass == kGrad && tid < kCols && c0 + tid < M) {
    const int t = p.targets[c0 + tid];
    const float most = *p.most;
    column.target = t < p.vocab ? t : -1;
    column.ll = -p.lse[c0 + tid] * kLog2e;
    column.share = most > 0.0f ? p.dloss[c0 + tid] / most : most;
  }

  // operands: where their first row lies, how many rows there are, their stride
  const int sum0 = kPass == kHidden ? split * p.split_rows : 0;  // first of the summed index
  int sums = kPass == kHidden ? (V - sum0 < p.split_rows ? V - sum0 : p.split_rows) : kPass == kWeight ? M : D;
  if (sums < 0) sums = 0;  // a share past the piece's last row: zeros
  const uint16_t *A, *B;
  int a_stride, b_stride, a_bytes, b_bytes;
  if (kPass == kStats || kPass == kGrad) {
    const int ra = V - r0 < kRows ? V - r0 : kRows, rb = M - c0 < kCols ? M - c0 : kCols;
    A = p.W + (size_t)r0 * D;
    B = p.H + (size_t)c0 * D;
    a_stride = b_stride = D;
    a_bytes = ra * D * 2;
    b_bytes = rb * D * 2;
  } else if (kPass == kHidden) {
    const int rb = M - c0 < kCols ? M - c0 : kCols;
    A = p.W + (size_t)sum0 * D + r0;
    a_stride = D;
    a_bytes = (sums * D - r0) * 2;
    B = p.G + (size_t)c0 * p.g_stride + sum0;
    b_stride = p.g_stride;
    b_bytes = (rb * p.g_stride - sum0) * 2;
    if (sums == 0) a_bytes = b_bytes = 0;
  } else {
    A = p.H + r0;
    a_stride = D;
    a_bytes = (M * D - r0) * 2;
    B = p.G + c0;
    b_stride = p.g_stride;
    b_bytes = (M * p.g_stride - c0) * 2;
  }
  const __amdgpu_buffer_rsrc_t ar = __builtin_amdgcn_make_buffer_rsrc((void*)A, (short)0, a_bytes, kBufferWord3);
  const __amdgpu_buffer_rsrc_t br = __builtin_amdgcn_make_buffer_rsrc((void*)B, (short)0, b_bytes, kBufferWord3);

  // fetch offsets and read positions. Rows of 64 (128 bytes): 16-byte chunk c of
  // row r lands at chunk c ^ (r & 7). Transposed tiles: rows of 256 (512 bytes).
  uint32_t a_off[T::kFetchA], b_off[T::kFetchB], a_pos[2], b_pos[2];
  const uint32_t nat0 = (uint32_t)(j * 128 + ((g ^ (j & 7)) * 16)), nat1 = (uint32_t)(j * 128 + (((4 + g) ^ (j & 7)) * 16));
  const uint32_t tr0 = (uint32_t)((8 * g + (j >> 2)) * 512 + (j & 3) * 8), tr1 = (uint32_t)(((j >> 2) | ((g & 1) << 2)) * 32);
  // row of this lane in fetch i of a transposed tile (the same for both operands, where both are)
  auto turned_row = [&](int i) __attribute__((always_inline)) { return 64 / T::kWaves * wave + 2 * i + (lane >> 5); };
  auto natural = [&](int row, int stride) __attribute__((always_inline)) {
    return (uint32_t)(row * stride * 2 + ((lane & 7) ^ (lane >> 3)) * 16);
  };
  auto turned = [&](int i, int stride, int cols) __attribute__((always_inline)) {
    const int row = turned_row(i), c = (((lane & 31) >> 1) ^ pair_swizzle(row)) * 2 + (lane & 1);
    return 8 * c < cols ? (uint32_t)(row * stride * 2 + c * 16) : kBufferOutOfRange;
  };
#pragma unroll
  for (int i = 0; i < T::kFetchA; ++i)
    a_off[i] = T::kTrA ? turned(i, a_stride, D - r0) : natural(kRows / T::kWaves * wave + 8 * i + (lane >> 3), a_stride);
#pragma unroll
  for (int i = 0; i < T::kFetchB; ++i)
    b_off[i] = T::kTrB ? turned(i, b_stride, 256) : natural(kCols / T::kWaves * wave + 8 * i + (lane >> 3), b_stride);
  a_pos[0] = T::kTrA ? tr0 : nat0;
  a_pos[1] = T::kTrA ? tr1 : nat1;
  b_pos[0] = T::kTrB ? tr0 : nat0;
  b_pos[1] = T::kTrB ? tr1 : nat1;

  f32x4 acc[T::kRT][T::kCT];
#pragma unroll
  for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int nk = (sums + kBlock - 1) / kBlock;
  // W's rows are read at other columns on other XCDs, which spreads them over the memory channels
  const int first = kPass == kStats || kPass == kGrad ? (int)(blockIdx.x & 7) * nk / 8 : 0;
  auto at = [&](int kb) __attribute__((always_inline)) {
    const int k = (kb < nk ? kb : 0) + first;  // (within the operands also where nothing is fetched)
    return (uint32_t)(k < nk ? k : k - nk);
  };
  const uint32_t a_step = T::kTrA ? (uint32_t)(kBlock * a_stride * 2) : kBlock * 2;
  const uint32_t b_step = T::kTrB ? (uint32_t)(kBlock * b_stride * 2) : kBlock * 2;
  // A stage past the last is fetched as nothing (zeros); in the last stage of a
  // sum over rows, rows past it are too.
  auto offsets_a = [&](int kb, uint32_t (&ao)[T::kFetchA]) __attribute__((always_inline)) {
    const uint32_t none = kb < nk ? 0u : kBufferOutOfRange;
    const int rows = sums - (int)at(kb) * kBlock;
#pragma unroll
    for (int i = 0; i < T::kFetchA; ++i) ao[i] = a_off[i] | (T::kTrA && turned_row(i) >= rows ? kBufferOutOfRange : none);
  };
  auto offsets_b = [&](int kb, uint32_t (&bo)[T::kFetchB]) __attribute__((always_inline)) {
    const uint32_t none = kb < nk ? 0u : kBufferOutOfRange;
    const int rows = sums - (int)at(kb) * kBlock;
#pragma unroll
    for (int i = 0; i < T::kFetchB; ++i) bo[i] = b_off[i] | (T::kTrB && turned_row(i) >= rows ? kBufferOutOfRange : none);
  };
  const int a_dst = T::kA / T::kWaves * wave, b_dst = T::kB / T::kWaves * wave;
  const int a_tile = T::kRT * wr, b_tile = T::kCT * wc;
  auto fetch = [&](int kb, char* a, char* b) __attribute__((always_inline)) {
    uint32_t ao[T::kFetchA], bo[T::kFetchB];
    offsets_a(kb, ao);
    offsets_b(kb, bo);
    loss_fetch<T::kFetchA>(ar, a + a_dst, ao, at(kb) * a_step);
    loss_fetch<T::kFetchB>(br, b + b_dst, bo, at(kb) * b_step);
  };
  if constexpr (T::kWide) {
    // The stages' tiles (A, B, A, B, ...) take five places in turn. A stage's
    // operands are in registers half a stage before its last products, so from
    // the middle of stage k on its two places are free: B of stage k + 2 is
    // fetched into the one in the second half (early in it), A of stage k + 3
    // into the other in the next stage's first half, and both have landed by the
    // middle of the stage before theirs. (All fetches in the second half, into
    // two whole buffers, took 3% more.)
    bf16x8 x0[8], y0[8], x1[8], y1[8];
    fetch(0, lds, lds + T::kA);
    fetch(1, lds + 2 * T::kA, lds + 3 * T::kA);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(T::kFetches) : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x0[i] = loss_operand<T::kTrA>(lds, a_tile + i, 0, a_pos[0], a_pos[1]);
      y0[i] = loss_operand<T::kTrB>(lds + T::kA, b_tile + i, 0, b_pos[0], b_pos[1]);
    }
    for (int kb = 0; kb < nk; kb += 5) {
#pragma unroll
      for (int u = 0; u < 5; ++u) {
        if (kb + u < nk) {
          const char *a = lds + 2 * u % 5 * T::kA, *b = lds + (2 * u + 1) % 5 * T::kA;
          const char *a1 = lds + (2 * u + 2) % 5 * T::kA, *b1 = lds + (2 * u + 3) % 5 * T::kA;
          char *a2 = lds + (2 * u + 4) % 5 * T::kA, *b2 = lds + 2 * u % 5 * T::kA;
          const int n = kb + u + 2;
          uint32_t off[8];
          offsets_a(n, off);
          loss_half<kPass, 16>(a, b, a2 + a_dst, ar, off, at(n) * a_step, 1, a_tile, b_tile, a_pos, b_pos, x0, y0, x1,
                               y1, acc);
          // the next stage has landed for every wave, and every wave has read this one
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(T::kFetchA) : "memory");
          offsets_b(n, off);
          loss_half<kPass, 8>(a1, b1, b2 + b_dst, br, off, at(n) * b_step, 0, a_tile, b_tile, a_pos, b_pos, x1, y1, x0,
                              y0, acc);
        }
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < T::kStages - 1; ++u) fetch(u, lds + u * T::kStage, lds + u * T::kStage + T::kA);
    for (int kb = 0; kb < nk; kb += T::kStages) {
#pragma unroll
      for (int u = 0; u < T::kStages; ++u) {
        if (kb + u < nk) {
          // the stage has landed for every wave, and every wave has read the one before
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((T::kStages - 2) * T::kFetches) : "memory");
          const int n = kb + u + T::kStages - 1;
          char* next = lds + (u + T::kStages - 1) % T::kStages * T::kStage;
          const char* cur = lds + u * T::kStage;
          uint32_t ao[T::kFetchA], bo[T::kFetchB];
          offsets_a(n, ao);
          offsets_b(n, bo);
          loss_block<kPass, kCols>(cur, cur + T::kA, next + a_dst, next + T::kA + b_dst, ar, br, ao, bo, at(n) * a_step,
                                   at(n) * b_step, a_tile, b_tile, a_pos, b_pos, acc);
        }
      }
    }
  }
  // nothing is in flight to or from LDS before the epilogue uses it
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  if constexpr (kPass == kGrad) {
    // the columns' values behind the staged outputs
    if (tid < kCols) ((Column*)(lds + T::kOut))[tid] = column;
    __syncthreads();
  }
  // lane (j, g) holds rows 16 a + 4 g + e and column 16 b + j of its wave's tile
  const int row0 = 16 * T::kRT * wr + 4 * g, col0 = 16 * T::kCT * wc + j;
  if constexpr (kPass == kStats) {
    const float rcap = kCap ? 1.0f / p.cap : 0.0f, rcap2 = rcap * rcap, far = kTanhSmall * p.cap;
    const bool tail = V - r0 < kRows;  // (uniform) rows past the vocabulary count nothing
    float2* sums_of = (float2*)lds;    // [kWavesR][kCols]
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) {
      if (tail) {
#pragma unroll
        for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r0 + row0 + 16 * a + e >= V) acc[a][b][e] = -__builtin_inff();
        }
      }
      float lo, mx, sum = 0.0f;
      column_range(acc, b, lo, mx);
      if (!kCap) {
        mx = __builtin_fmaxf(mx, kLowest);
        const float ml = -mx * kLog2e;
#pragma unroll
        for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[a][b][e], kLog2e, ml));
        }
      } else {
        const bool near = lo > -far && mx < far;  // (false with a NaN about, or a masked row)
        mx = p.cap * cap_far(mx * rcap);          // tanh keeps the order
        const float ml = -mx * kLog2e;
        if (__all(near)) {
#pragma unroll
          for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = acc[a][b][e], s = x * (x * rcap2);
              sum += __builtin_amdgcn_exp2f(__builtin_fmaf(x * kLog2e, cap_series(s), ml));
            }
          }
        } else {
#pragma unroll
          for (int a = 0; a < T::kRT; ++a) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = acc[a][b][e], q = x * rcap;
              const float z = __builtin_fabsf(q) < kTanhSmall ? x * cap_series(q * q) : p.cap * cap_far(q);
              const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, ml));
              sum += tail && r0 + row0 + 16 * a + e >= V ? 0.0f : v;
            }
          }
        }
      }
      // the four lane groups of a column
#pragma unroll
      for (int d = 16; d < 64; d <<= 1) join_sums(mx, sum, __shfl_xor(mx, d), __shfl_xor(sum, d));
      if (g == 0) sums_of[wr * kCols + col0 + 16 * b] = make_float2(mx, sum);
    }
    __syncthreads();
    if (tid < kCols && c0 + tid < M) {
      float2 s = sums_of[tid];
#pragma unroll
      for (int w = 1; w < T::kWavesR; ++w) {
        const float2 o = sums_of[w * kCols + tid];
        join_sums(s.x, s.y, o.x, o.y);
      }
      p.stats[(size_t)rt * M + c0 + tid] = s;
    }
  } else if constexpr (kPass == kGrad) {
    const float rcap = kCap ? 1.0f / p.cap : 0.0f, rcap2 = rcap * rcap, far = kTanhSmall * p.cap;
    uint16_t* stage = (uint16_t*)lds;
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) {
      const int col = col0 + 16 * b;
      const Column c = ((const Column*)(lds + T::kOut))[col];
      const bool scored = c.target >= 0;
      const float ll = c.ll, share = c.share;
      const int hit = c.target - p.v_base - r0 - row0;  // the target's place among this lane's rows
      const bool any_hit = __any(scored && hit >= 0 && hit < 16 * T::kRT);
      bool near = true;
      if (kCap) {
        float lo, hi;
        column_range(acc, b, lo, hi);
        near = __all(lo > -far && hi < far);
      }
#pragma unroll
      for (int a = 0; a < T::kRT; ++a) {
        float v[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc[a][b][e];
          w[e] = 1.0f;
          if (!kCap) {
            v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, ll));
          } else if (near) {
            const float s = x * (x * rcap2), u = cap_series(s);
            v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x * kLog2e, u, ll));
            w[e] = __builtin_fmaf(-s, u * u, 1.0f);
          } else {
            const float q = x * rcap;
            const float t = __builtin_fabsf(q) < kTanhSmall ? q * cap_series(q * q) : cap_far(q);
            v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p.cap * t, kLog2e, ll));
            w[e] = __builtin_fmaf(-t, t, 1.0f);
          }
        }
        if (any_hit) {  // (uniform)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hit == 16 * a + e) v[e] -= 1.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= kCap ? w[e] * share : share;
        if (V - r0 < kRows) {  // (uniform) zeros past the vocabulary
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r0 + row0 + 16 * a + e >= V) v[e] = 0.0f;
        }
        // a row that is not scored has no gradient, whatever its hidden state holds
        const MxU32x2 o = {scored ? pack_bf16(v[0], v[1]) : 0u, scored ? pack_bf16(v[2], v[3]) : 0u};
        *(MxU32x2*)&stage[col * T::kOutStride + row0 + 16 * a] = o;
      }
    }
    __syncthreads();
    // rows of 512 bytes of g
#pragma unroll 4
    for (int q = tid; q < kCols * 32; q += T::kThreads) {
      const int m = q >> 5, c = (q & 31) * 8;
      if (c0 + m < M)
        *(MxU32x4*)&p.G[(size_t)(c0 + m) * p.g_stride + r0 + c] = *(const MxU32x4*)&stage[m * T::kOutStride + c];
    }
  } else if constexpr (kPass == kHidden) {
    float* part = p.part + (size_t)split * M * D;
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) {
      const int m = c0 + col0 + 16 * b;
#pragma unroll
      for (int a = 0; a < T::kRT; ++a) {
        const int k = r0 + row0 + 16 * a;
        if (m < M && k < D) {
          f32x4* o = (f32x4*)&part[(size_t)m * D + k];
          f32x4 v = acc[a][b];
          if (p.accumulate) v += *o;
          *o = v;
        }
      }
    }
  } else {
    uint16_t* stage = (uint16_t*)lds;
    const float most = *p.most;
#pragma unroll
    for (int b = 0; b < T::kCT; ++b) {
#pragma unroll
      for (int a = 0; a < T::kRT; ++a) {
        const f32x4 v = acc[a][b] * most;
        *(MxU32x2*)&stage[(col0 + 16 * b) * T::kOutStride + row0 + 16 * a] =
            MxU32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int q = tid; q < kCols * 32; q += T::kThreads) {
      const int v = q >> 5, c = (q & 31) * 8;
      if (c0 + v < V && r0 + c < D)
        *(MxU32x4*)&p.dW[(size_t)(c0 + v) * D + r0 + c] = *(const MxU32x4*)&stage[v * T::kOutStride + c];
    }
  }
}

// lse and loss of 8 rows a workgroup: the tiles' (max, sum) joined in one
// order, and the target's logit as one dot product.
constexpr int kJoinRows = 8;
__global__ __launch_bounds__(256) void loss_join_kernel(const float2* __restrict__ stats, int n_tiles,
                                                        const uint16_t* __restrict__ H, const uint16_t* __restrict__ W,
                                                        const int32_t* __restrict__ targets, int M, int D, int V,
                                                        float cap, float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ float2 slices[32][kJoinRows];
  __shared__ float lse_of[kJoinRows];
  const int tid = threadIdx.x, i = tid & (kJoinRows - 1), slice = tid / kJoinRows;
  const int m0 = (int)blockIdx.x * kJoinRows;
  float2 s = make_float2(kLowest, 0.0f);
  if (m0 + i < M) {
#pragma unroll 4
    for (int t = slice; t < n_tiles; t += 32) {
      const float2 o = stats[(size_t)t * M + m0 + i];
      join_sums(s.x, s.y, o.x, o.y);
    }
  }
  slices[slice][i] = s;
  __syncthreads();
  if (slice == 0 && m0 + i < M) {
    for (int t = 1; t < 32; ++t) {
      const float2 o = slices[t][i];
      join_sums(s.x, s.y, o.x, o.y);
    }
    const float l = s.x + logf(s.y);
    lse_of[i] = l;
    lse[m0 + i] = l;
  }
  __syncthreads();
  const int lane = tid & 63, wave = tid >> 6;
  for (int r = wave; r < kJoinRows && m0 + r < M; r += 4) {
    const int64_t t = targets[m0 + r];
    if (t < 0 || t >= V) {
      if (lane == 0) loss[m0 + r] = 0.0f;
      continue;
    }
    float z = 0.0f;
    for (int c = lane * 8; c < D; c += 512) {
      float x[8], y[8];
      load_8<true>(H, (int64_t)(m0 + r) * D + c, 8, x);
      load_8<true>(W, t * D + c, 8, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) z = __builtin_fmaf(x[e], y[e], z);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) z += __shfl_xor(z, d);
    if (cap > 0.0f) z = cap * tanhf(z / cap);
    if (lane == 0) loss[m0 + r] = lse_of[r] - z;
  }
}

// The largest |dloss| of the scored rows (a NaN stays one: its bits are above
// every number's).
__global__ __launch_bounds__(1024) void loss_scale_kernel(const float* __restrict__ dloss,
                                                          const int32_t* __restrict__ targets, int M, int V,
                                                          float* __restrict__ most) {
  __shared__ uint32_t wave_most[16];
  uint32_t b = 0;
  for (int m = threadIdx.x; m < M; m += 1024) {
    const int t = targets[m];
    const uint32_t d = t >= 0 && t < V ? __float_as_uint(dloss[m]) & 0x7fffffffu : 0u;
    b = d > b ? d : b;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)b, d);
    b = o > b ? o : b;
  }
  if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = b;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) b = wave_most[i] > b ? wave_most[i] : b;
    *most = __uint_as_float(b);
  }
}

// H with zeros in the rows that are not scored, for dW's product: their g is
// zero, but zero times what a padded row may hold need not be.
__global__ __launch_bounds__(256) void loss_rows_kernel(const uint16_t* __restrict__ H,
                                                        const int32_t* __restrict__ targets, int V, int D, int64_t n,
                                                        uint16_t* __restrict__ out) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= n) return;
  const int t = targets[e / D];
  const MxU32x4 z = {0, 0, 0, 0};
  *(MxU32x4*)&out[e] = t >= 0 && t < V ? *(const MxU32x4*)&H[e] : z;
}

// dH = most times the shares, added in order and rounded once; zeros in the rows
// that are not scored.
__global__ __launch_bounds__(256) void loss_hidden_kernel(const float* __restrict__ part, int splits, int64_t n,
                                                          const int32_t* __restrict__ targets,
                                                          const float* __restrict__ most, int V, int D,
                                                          uint16_t* __restrict__ dH) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= n) return;
  const int t = targets[e / D];
  float v[8];
  load_8<false>(part, e, 8, v);
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    float o[8];
    load_8<false>(part, s * n + e, 8, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += o[i];
  }
  const float f = *most;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = t >= 0 && t < V ? v[i] * f : 0.0f;
  store_8<true>(dH, e, 8, v);
}

template <Pass kPass, bool kCap>
void loss_launch_capped(const LossArgs& p, int cols, hipStream_t s) {
  const int total = p.row_tiles * p.col_tiles * p.splits;
  const dim3 grid((unsigned)((total + 7) / 8 * 8));
  if constexpr (kPass != kWeight) {
    if (cols == 64) {
      loss_kernel<kPass, 64, kCap><<<grid, dim3(Tile<kPass, 64>::kThreads), 0, s>>>(p);
      return;
    }
    if (cols == 128) {
      loss_kernel<kPass, 128, kCap><<<grid, dim3(Tile<kPass, 128>::kThreads), 0, s>>>(p);
      return;
    }
  }
  loss_kernel<kPass, 256, kCap><<<grid, dim3(Tile<kPass, 256>::kThreads), 0, s>>>(p);
}

template <Pass kPass>
void loss_launch(const LossArgs& p, int cols, hipStream_t s) {
  if constexpr (kPass == kStats || kPass == kGrad) {
    if (p.cap > 0.0f) {
      loss_launch_capped<kPass, true>(p, cols, s);
      return;
    }
  }
  loss_launch_capped<kPass, false>(p, cols, s);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

LossPlan loss_plan(int32_t rows, int32_t width, int32_t vocab, int32_t cu_count) {
  LossPlan q{};
  q.cols = rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  q.v_tiles = (vocab + kRows - 1) / kRows;
  // a piece: at most 256 MB of g, and its offsets (and W's) within 31 bits
  int64_t piece = ((int64_t)256 << 20) / ((int64_t)rows * 2);
  piece = std::min<int64_t>(piece, ((int64_t)1 << 30) / width - 256);
  piece = std::max<int64_t>(256, piece / 256 * 256);
  q.piece = (int32_t)std::min<int64_t>(piece, (int64_t)q.v_tiles * 256);
  const int tiles = (width + kRows - 1) / kRows * ((rows + q.cols - 1) / q.cols);
  const int cus = cu_count > 0 ? cu_count : 256;
  q.splits = std::max(1, std::min(cus / tiles, q.piece / 256));
  q.stats_bytes = up256((size_t)q.v_tiles * rows * sizeof(float2));
  q.g_bytes = up256((size_t)rows * q.piece * 2);
  q.h_bytes = up256((size_t)rows * width * 2);
  q.part_bytes = up256((size_t)q.splits * rows * width * 4);
  return q;
}

void launch_lmhead_loss(const uint16_t* hidden, const uint16_t* weight, const int32_t* targets, int32_t rows,
                        int32_t width, int32_t vocab, float softcap, const LossPlan& plan, uint8_t* work, float* loss,
                        float* lse, hipStream_t s) {
  LossArgs p{};
  p.W = weight;
  p.H = hidden;
  p.stats = (float2*)work;
  p.cap = softcap;
  p.M = rows;
  p.D = width;
  p.V = vocab;
  p.row_tiles = plan.v_tiles;
  p.col_tiles = (rows + plan.cols - 1) / plan.cols;
  p.splits = 1;
  loss_launch<kStats>(p, plan.cols, s);
  loss_join_kernel<<<dim3((unsigned)((rows + kJoinRows - 1) / kJoinRows)), dim3(256), 0, s>>>(
      p.stats, plan.v_tiles, hidden, weight, targets, rows, width, vocab, softcap, loss, lse);
}

void launch_lmhead_loss_grad(const uint16_t* hidden, const uint16_t* weight, const int32_t* targets, const float* lse,
                             const float* dloss, int32_t rows, int32_t width, int32_t vocab, float softcap,
                             const LossPlan& plan, uint8_t* work, uint16_t* dhidden, uint16_t* dweight, hipStream_t s) {
  const int64_t n = (int64_t)rows * width;
  const dim3 per8((unsigned)((n / 8 + 255) / 256)), block(256);
  uint16_t* scored = (uint16_t*)(work + plan.g_bytes);
  float* part = (float*)(work + plan.g_bytes + plan.h_bytes);
  float* most = (float*)(work + plan.g_bytes + plan.h_bytes + plan.part_bytes);
  loss_scale_kernel<<<dim3(1), dim3(1024), 0, s>>>(dloss, targets, rows, vocab, most);
  if (dweight) loss_rows_kernel<<<per8, block, 0, s>>>(hidden, targets, vocab, width, n, scored);
  const int k_tiles = (width + kRows - 1) / kRows;
  int splits = 1;
  for (int32_t v = 0; v < vocab; v += plan.piece) {
    LossArgs p{};
    p.W = weight + (size_t)v * width;
    p.H = hidden;
    p.G = (uint16_t*)work;
    p.targets = targets;
    p.lse = lse;
    p.dloss = dloss;
    p.most = most;
    p.part = part;
    p.cap = softcap;
    p.M = rows;
    p.D = width;
    p.V = std::min(plan.piece, vocab - v);
    p.v_base = v;
    p.vocab = vocab;
    p.g_stride = (p.V + 255) / 256 * 256;
    p.row_tiles = p.g_stride / 256;
    p.col_tiles = (rows + plan.cols - 1) / plan.cols;
    p.splits = 1;
    loss_launch<kGrad>(p, plan.cols, s);
    if (dhidden) {
      // every piece fills the same shares: the last, shorter one in shorter runs
      p.row_tiles = k_tiles;
      if (v == 0) splits = std::min(plan.splits, p.g_stride / 256);
      p.splits = splits;
      p.split_rows = ((p.V + splits - 1) / splits + kBlock - 1) / kBlock * kBlock;
      p.accumulate = v > 0;
      loss_launch<kHidden>(p, plan.cols, s);
    }
    if (dweight) {
      p.H = scored;
      p.dW = dweight + (size_t)v * width;
      p.row_tiles = k_tiles;
      p.col_tiles = p.g_stride / 256;
      p.splits = 1;
      loss_launch<kWeight>(p, 256, s);
    }
  }
  if (dhidden) loss_hidden_kernel<<<per8, block, 0, s>>>(part, splits, n, targets, most, vocab, width, dhidden);
}

}  // namespace gs

// Softmax cross entropy of the head's logits, and its gradients, without the
// logits in memory:
//   z = cap(H W^T),  lse[m] = log sum_v exp z[m][v],  loss[m] = lse[m] - z[m][t[m]]
//   g[m][v] = dloss[m] / most (exp(z[m][v] - lse[m]) - [v = t[m]]) (1 - (z[m][v] / cap)^2)
//   dH = most g W,  dW = most g^T H,  most = max |dloss| of the finite ones
//
// Four products on v_mfma_f32_16x16x32_bf16 with one main loop: tiles of 256
// rows by kCols columns, 4 waves of 128 by kCols / 2, one a SIMD with the
// registers of two (an LDS byte is read for the fewest products so), 64 of the
// summed index a stage, operands by the memory pipe straight into LDS. A
// workgroup takes tile after tile and fetches the next one's first stages while
// it finishes the last.
//   kStats   W x H, the epilogue leaves a (max, sum) per hidden row and tile;
//   kGrad    W x H again, a piece of the vocabulary, the epilogue writes g in
//            bf16 (the matrix cores read 16 bits: half a step of 2^-8 a value, the
//            sums are binary32). The largest |dloss| stays out of g: where every
//            row has the same, as in a mean, a row's largest value, at the target,
//            is then near -1, which bf16 holds, and not a product whose rounding
//            all rows share (dW's error at M 4096 was 1.7 times its own rounding's;
//            so it is 1.95e-3 of its norm, and dH's 1.94e-3, where the roundings of the
//            results to bf16 alone make 1.66e-3);
//   kHidden  W^T x g, summed over the piece, in shares of its vocabulary rows;
//   kWeight  H^T x g^T, summed over the hidden rows.
// kHidden and kWeight sum over an operand's rows: those tiles lie in LDS as
// they do in memory and are transposed by the LDS reads (ds_read_b64_tr_b16).
//
// Few rows are bound by W's bytes (100 x 2048 x 151643: kStats 117 us for 621 MB,
// 5.3 TB/s), many by the matrix cores: at 4096 x 2048 x 262144 kStats 3.5 ms at best (1.25
// PFLOP/s, the cores busy for 63 %; 3.7 over a run), and for a piece of 32768 vocabulary rows kGrad
// 529 us (52 %), kHidden 409 and kWeight 411 (1.34 PFLOP/s, 69 %; a library product
// of that size reaches 1.46). The rest is the epilogues', which one wave a SIMD has
// nothing to run beside; two of half the tile would read LDS twice as often.
#include <algorithm>

#include "gs_cap.h"
#include "gs_mx.h"

namespace gs {
namespace {

enum Pass { kStats, kGrad, kHidden, kWeight };

constexpr int kLossThreads = 256;
constexpr int kRows = 256;  // rows of a tile (vocabulary rows; columns of K in kHidden and kWeight)
constexpr int kBlock = 64;  // of the summed index a stage
constexpr int kFewRows = 128;  // columns of a tile up to which the forward pass waits for W's bytes
constexpr float kLowest = -1.0e38f;  // a maximum over nothing; times log2(e) still finite

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* LdsPtr;
typedef __attribute__((address_space(3))) i16x4* LdsTrPtr;

// What kGrad needs of a hidden row.
struct Column {
  int32_t target;  // negative: not scored
  float ll;        // -lse log2(e)
  float share;     // dloss over the largest finite |dloss|
  float none;
};

struct LossArgs {
  const uint16_t* W;      // the piece's first row
  const uint16_t* H;
  uint16_t* G;            // [M][g_stride]
  const Column* columns;  // [M]
  const float* most;      // the largest finite |dloss| of the scored rows, 1 if that is 0
  float2* stats;          // kStats: [row_tiles][M]
  int tile_rows;          // kStats: rows of W a tile
  float* part;            // kHidden: [splits][M][D]
  uint16_t* dW;           // kWeight: the piece's first row
  float cap;
  int32_t M, D, V;        // V: vocabulary rows of the piece
  int32_t v_base;         // the piece's first vocabulary row
  int32_t g_stride;       // a multiple of 256, at least V
  int32_t row_tiles, col_tiles, splits, split_rows;  // split_rows: vocabulary rows a share, a multiple of 64
  int32_t accumulate;     // kHidden: add to the shares of the pieces before
};

template <Pass kPass, int kCols>
struct Tile {
  static constexpr bool kTrA = kPass == kHidden || kPass == kWeight, kTrB = kPass == kWeight;
  static constexpr int kCT = kCols / 32;     // 16-column tiles a wave (two waves abreast)
  static constexpr int kA = kRows * kBlock * 2, kB = kCols * kBlock * 2;
  static constexpr int kFetchB = kCT;        // wave instructions of 1 KB (8 for the rows)
  // Wide tiles: the stages' tiles (A, B, A, B, ...) take five places of 32 KB in
  // turn, two stages ahead. Narrow ones: whole stages in three places, three ahead.
  static constexpr bool kFive = kCols >= 192;
  static constexpr int kPlace = kFive ? kA : kA + kB;
  static constexpr int kScratch = 4096;      // a (max, sum) a row half and column, or the columns' values
  static constexpr int kOperands = kFive ? 5 * kA : 3 * kPlace;
  static constexpr int kLds = kFive ? kOperands : kOperands + kScratch;
  // fetches after the next stage's own when that one has to have landed
  static constexpr int kAhead = kFive ? 8 : 8 + kFetchB;
  // stores of a tile's epilogue, always issued, that may still be under way then
  static constexpr int kStores = kPass == kStats ? 0 : kPass == kHidden ? 8 * kCT : 4 * kCT;
  static constexpr int kAheadStores = kAhead + kStores < 63 ? kAhead + kStores : 63;
  static_assert(kLds <= 160 * 1024, "LDS of a compute unit");
};

// The position of 16-byte chunk pairs in a transposed tile's row: the 8 rows
// that a half wave reads together (4 of each of two lane groups) take 8
// different pairs of the banks.
__device__ __forceinline__ int pair_swizzle(int row) { return (row & 3) | ((row >> 1) & 4); }

// Operand tile t's values of the summed index 32 s + 8 g .. + 7 for lane (j, g),
// from the wave's first tile. Rows of 64: pos is the lane's row and chunk.
// Transposed: its row and place in a pair, turn the pair's swizzle.
template <bool kTr>
__device__ __forceinline__ bf16x8 loss_operand(const char* p, int t, int s, uint32_t pos, uint32_t turn) {
  if (!kTr) return *(const bf16x8*)(p + pos + 2048 * t);
#ifdef __HIP_DEVICE_COMPILE__
  const char* q = p + pos + ((32 * (uint32_t)t) ^ turn) + s * 16384;
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTrPtr)q);
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTrPtr)(q + 2048));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
  return bf16x8{};
#endif
}

// Waits until at most kAhead memory instructions of this wave are under way
// (kAheadStores if `stored`) and for every wave. The choice is in the assembly:
// a branch around it would have the compiler keep two copies of the stage, with
// the sums in other registers.
template <int kAhead, int kAheadStores>
__device__ __forceinline__ void landed(int stored) {
  asm volatile(
      "s_cmp_lg_u32 %0, 0\n\t"
      "s_cbranch_scc1 .Lstored%=\n\t"
      "s_waitcnt vmcnt(%1)\n\t"
      ".Lstored%=:\n\t"
      "s_waitcnt vmcnt(%2) lgkmcnt(0)\n\t"
      "s_barrier" ::"s"(stored),
      "n"(kAhead), "n"(kAheadStores)
      : "memory", "scc");
}

// Nothing moves across: an epilogue handles one 16-column tile after another (the
// scheduler would read many of them into registers that the products hold).
__device__ __forceinline__ void order() {
#ifdef __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// acc += x y, the sums in the accumulation registers and in place: with the
// builtin the compiler moves the 256 of them about between stages. A tile's sums
// are read no sooner than sums_ready() after the last of these: the compiler puts
// no waits around assembly. None is needed before one, as its operands come from
// LDS by reads that are waited for, and from no vector instruction (the built code
// is tested for it; two states in front of every product cost 3.5 % of a training
// step).
__device__ __forceinline__ void add_products(f32x4& acc, const bf16x8& x, const bf16x8& y) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
#endif
}
__device__ __forceinline__ void sums_ready() {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// Where a lane reads an operand's half s, and the transposed tiles' swizzle.
struct ReadPos {
  uint32_t half[2], turn;
};

// What the order below leaves to the compiler: address arithmetic, which fits
// into the products' shadow.
[[maybe_unused]] constexpr int kOrder = 0x6;  // (vector and scalar ALU instructions may cross)

// Half a stage: the products of the operands in registers and, in a fixed order
// between them, the reads of the next half's operands and kNA + kNB fetches. Left
// to the compiler, the fetches go out in one run that the matrix core waits for.
// The columns' operands come first (all of them are needed for the next half's
// first products), a row tile's as soon as its products are out, into its place.
template <Pass kPass, int kCols, int kNA, int kNB, typename Rsrc>
__device__ __forceinline__ void loss_half(const char* __restrict__ a, const char* __restrict__ b, int s,
                                          const ReadPos& a_pos, const ReadPos& b_pos, char* __restrict__ a_next,
                                          char* __restrict__ b_next, Rsrc ar, Rsrc br, const uint32_t (&a_off)[8],
                                          const uint32_t (&b_off)[Tile<kPass, kCols>::kFetchB], uint32_t ak, uint32_t bk,
                                          bf16x8 (&x)[8], const bf16x8 (&y)[kCols / 32], bf16x8 (&y_next)[kCols / 32],
                                          f32x4 (&acc)[8][kCols / 32]) {
  constexpr int kCT = kCols / 32, kSlots = 4 * kCT;
#pragma unroll
  for (int t = 0; t <= kSlots; ++t) {
#ifdef __HIP_DEVICE_COMPILE__
    typedef Tile<kPass, kCols> T;
    // (B of a wide tile is needed a whole stage later: its fetches go out early)
    constexpr int kN = kNA + kNB, kSpread = kN && !kNA ? kSlots / 2 : kSlots;
#pragma unroll
    for (int i = 0; i < kCT; ++i)
      if (t == 3 * i) y_next[i] = loss_operand<T::kTrB>(b, i, s, b_pos.half[s], b_pos.turn);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (t == ((i + 1) * kCT + 1) / 2 + (i < 7 ? 1 : 0)) x[i] = loss_operand<T::kTrA>(a, i, s, a_pos.half[s], a_pos.turn);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (t != i * kSpread / (kN ? kN : 1)) continue;
      if (i < kNA) __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, (LdsPtr)(a_next + 1024 * i), 16, a_off[i], ak, 0, 0);
      else __builtin_amdgcn_raw_ptr_buffer_load_lds(br, (LdsPtr)(b_next + 1024 * (i - kNA)), 16, b_off[i - kNA], bk, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(kOrder);
#endif
    if (t == kSlots) break;
#pragma unroll
    for (int h = 2 * t; h < 2 * t + 2; ++h)
      add_products(acc[h / kCT][h % kCT], x[h / kCT], y[h % kCT]);
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_sched_barrier(kOrder);
#endif
  }
}

// Rows 4 g .. + 3 of tiles a (first) and a + 1 in two words each, exchanged
// between neighbouring lane groups: 8 rows of tile a + (g & 1) in one lane.
__device__ __forceinline__ MxU32x4 eight_rows(MxU32x2 first, MxU32x2 second) {
#ifdef __HIP_DEVICE_COMPILE__
  const auto x = __builtin_amdgcn_permlane16_swap(first.x, second.x, false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(first.y, second.y, false, false);
  return MxU32x4{x[0], y[0], x[1], y[1]};
#else
  return MxU32x4{first.x, first.y, second.x, second.y};
#endif
}

// This wave's 64 of a tile's columns (16 bytes each) into LDS, one wave
// instruction; columns past M read zeros.
__device__ __forceinline__ void loss_columns(const LossArgs& p, int c0, int wave, int lane, char* lds) {
#ifdef __HIP_DEVICE_COMPILE__
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)p.columns, (short)0, p.M * 16, kBufferWord3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)(lds + 1024 * wave), 16, (uint32_t)((c0 + 64 * wave + lane) * 16), 0, 0, 0);
#endif
}

// A (max, sum of exponentials over it) pair with another's.
__device__ __forceinline__ void join_sums(float& mx, float& sum, float om, float os) {
  const float nm = __builtin_fmaxf(mx, om);
  sum = sum * __builtin_amdgcn_exp2f((mx - nm) * kLog2e) + os * __builtin_amdgcn_exp2f((om - nm) * kLog2e);
  mx = nm;
}

template <Pass kPass, int kCols, bool kCap>
__global__ __launch_bounds__(kLossThreads, 1) void loss_kernel(LossArgs p) {
  typedef Tile<kPass, kCols> T;
  constexpr int kCT = T::kCT;
  __shared__ __attribute__((aligned(16))) char lds[T::kLds];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, g = lane >> 4, wr = wave & 1, wc = wave >> 1;
  const int M = p.M, D = p.D, V = p.V;

  // An XCD (consecutive workgroups go to them in turn) takes a run of adjacent
  // tiles, so its workgroups share their operands' lines in its L2: four row
  // tiles by all column tiles (kStats, kGrad), all row tiles by a run of
  // column tiles (kHidden, kWeight).
  const int total = p.row_tiles * p.col_tiles * p.splits;
  const int run = (total + 7) / 8, step = (int)(gridDim.x >> 3);
  int id = (int)(blockIdx.x & 7) * run + (int)(blockIdx.x >> 3);
  const int id_end = ((int)(blockIdx.x & 7) + 1) * run < total ? ((int)(blockIdx.x & 7) + 1) * run : total;
  if (id >= id_end) return;
  struct Place {
    int r0, c0, split;
  };
  auto locate = [&](int id) __attribute__((always_inline)) {
    int rt, ct, split = 0;
    if (kPass == kStats || kPass == kGrad) {
      const int group = id / (4 * p.col_tiles) * 4;
      const int in = p.row_tiles - group < 4 ? p.row_tiles - group : 4;
      id -= group * p.col_tiles;
      ct = id / in;
      rt = group + id - ct * in;
    } else {
      const int q = id / p.row_tiles;
      rt = id - q * p.row_tiles;
      split = q / p.col_tiles;
      ct = q - split * p.col_tiles;
    }
    return Place{rt * (kPass == kStats ? p.tile_rows : kRows), ct * kCols, split};
  };
  auto sums_of_split = [&](int split) __attribute__((always_inline)) {
    if (kPass != kHidden) return kPass == kWeight ? M : D;
    const int n = V - split * p.split_rows;
    return n < 0 ? 0 : n < p.split_rows ? n : p.split_rows;  // (0: a share past the piece's last row, zeros)
  };
  auto stages_of = [&](int sums) __attribute__((always_inline)) { return sums > kBlock ? (sums + kBlock - 1) / kBlock : 1; };

  // ---- fetches: where this lane's 16 bytes of each wave instruction come from
  const int a_stride = D, b_stride = kPass == kStats || kPass == kGrad ? D : p.g_stride;
  const uint32_t a_step = T::kTrA ? (uint32_t)(kBlock * a_stride * 2) : kBlock * 2;
  const uint32_t b_step = T::kTrB ? (uint32_t)(kBlock * b_stride * 2) : kBlock * 2;
  // Rows of 64 (128 bytes): 16-byte chunk c of row r lands at chunk c ^ (r & 7).
  // Transposed tiles: rows of 256 (512 bytes), pairs of chunks swizzled.
  auto turned_row = [&](int i) __attribute__((always_inline)) { return 16 * wave + 2 * i + (lane >> 5); };
  auto turned_chunk = [&](int i) __attribute__((always_inline)) {
    return (((lane & 31) >> 1) ^ pair_swizzle(turned_row(i))) * 2 + (lane & 1);
  };
  auto natural = [&](int row, int stride) __attribute__((always_inline)) {
    return (uint32_t)(row * stride * 2 + ((lane & 7) ^ (lane >> 3)) * 16);
  };
  uint32_t a_off[8], b_off[T::kFetchB];
#pragma unroll
  for (int i = 0; i < 8; ++i) a_off[i] = T::kTrA ? 0u : natural(64 * wave + 8 * i + (lane >> 3), a_stride);
#pragma unroll
  for (int i = 0; i < T::kFetchB; ++i)
    b_off[i] = T::kTrB ? (uint32_t)(turned_row(i) * b_stride * 2 + turned_chunk(i) * 16)
                       : natural(kCols / 4 * wave + 8 * i + (lane >> 3), b_stride);
  // W's rows are read at other columns on other XCDs, which spreads them over the memory channels
  const int first = kPass == kStats || kPass == kGrad ? (int)(blockIdx.x & 7) * (D / kBlock) / 8 : 0;
  // the tile and the stage that are fetched next
  __amdgpu_buffer_rsrc_t ar, br;
  int f_id = id, f_left = 0, f_nk = 0, f_k = 0, f_sums = 0;
  uint32_t f_ak = 0, f_bk = 0;
  // (The resources end with the last summed row, and the offset of a stage counts
  // in their bounds check: rows past it are read as zeros.)
  auto fetch_tile = [&]() __attribute__((always_inline)) {
    int t = f_id;
    asm volatile("" : "+s"(t));  // (nothing of this is computed ahead of the branch here)
    const uint16_t *A = p.W, *B = p.H;
    int a_bytes = 0, b_bytes = 0;  // past the last tile: nothing is read
    f_sums = 0;
    f_nk = f_left = 1;
    f_k = 0;
    if (t < id_end) {
      const Place q = locate(t);
      f_sums = sums_of_split(q.split);
      f_nk = f_left = stages_of(f_sums);
      f_k = first;
      if (kPass == kStats || kPass == kGrad) {
        A = p.W + (size_t)q.r0 * D;
        B = p.H + (size_t)q.c0 * D;
        const int most = kPass == kStats ? p.tile_rows : kRows;
        a_bytes = (V - q.r0 < most ? V - q.r0 : most) * D * 2;
        b_bytes = (M - q.c0 < kCols ? M - q.c0 : kCols) * D * 2;
      } else if (f_sums > 0) {
        const int sum0 = kPass == kHidden ? q.split * p.split_rows : 0;
        if (kPass == kHidden) {
          A = p.W + (size_t)sum0 * D + q.r0;
          B = p.G + (size_t)q.c0 * p.g_stride + sum0;
          b_bytes = ((M - q.c0 < kCols ? M - q.c0 : kCols) * p.g_stride - sum0) * 2;
        } else {
          A = p.H + q.r0;
          B = p.G + q.c0;
          b_bytes = (M * p.g_stride - q.c0) * 2;
        }
        a_bytes = (f_sums * D - q.r0) * 2;
      }
      if (T::kTrA) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          a_off[i] = 8 * turned_chunk(i) < D - q.r0 ? (uint32_t)(turned_row(i) * a_stride * 2 + turned_chunk(i) * 16)
                                                    : kBufferOutOfRange;
      }
    }
    ar = __builtin_amdgcn_make_buffer_rsrc((void*)A, (short)0, a_bytes, kBufferWord3);
    br = __builtin_amdgcn_make_buffer_rsrc((void*)B, (short)0, b_bytes, kBufferWord3);
    f_ak = (uint32_t)f_k * a_step;
    f_bk = (uint32_t)f_k * b_step;
  };
  auto fetch_next = [&]() __attribute__((always_inline)) {
    if (--f_left == 0) {
      f_id = f_id < id_end ? f_id + step : f_id;
      fetch_tile();
    } else {
      const bool wrap = ++f_k == f_nk;
      f_k = wrap ? 0 : f_k;
      f_ak = wrap ? 0u : f_ak + a_step;
      f_bk = wrap ? 0u : f_bk + b_step;
    }
  };
  const int a_dst = T::kA / 4 * wave, b_dst = T::kB / 4 * wave;

  // ---- reads: lane (j, g) holds the summed index 8 g .. + 7 of a half for row (column) j of a tile
  ReadPos a_pos, b_pos;
  {
    const uint32_t nat0 = (uint32_t)(j * 128 + ((g ^ (j & 7)) * 16)), nat1 = (uint32_t)(j * 128 + (((4 + g) ^ (j & 7)) * 16));
    const uint32_t tr = (uint32_t)((8 * g + (j >> 2)) * 512 + (j & 3) * 8), turn = (uint32_t)(((j >> 2) | ((g & 1) << 2)) * 32);
    a_pos.half[0] = T::kTrA ? tr + 256 * wr : nat0 + 16384 * wr;  // (a wave's tiles start at a multiple of 8)
    a_pos.half[1] = T::kTrA ? tr + 256 * wr : nat1 + 16384 * wr;
    a_pos.turn = turn;
    b_pos.half[0] = T::kTrB ? tr + 256 * wc : nat0 + 2048 * kCT * wc;
    b_pos.half[1] = T::kTrB ? tr + 256 * wc : nat1 + 2048 * kCT * wc;
    b_pos.turn = turn;
  }

  // ---- the first stages
  fetch_tile();
#pragma unroll
  for (int u = 0; u < (T::kFive ? 2 : 3); ++u) {
    [[maybe_unused]] char* a = lds + (T::kFive ? 2 * u * T::kA : u * T::kPlace);
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int i = 0; i < 8; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, (LdsPtr)(a + a_dst + 1024 * i), 16, a_off[i], f_ak, 0, 0);
#pragma unroll
    for (int i = 0; i < T::kFetchB; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(br, (LdsPtr)(a + T::kA + b_dst + 1024 * i), 16, b_off[i], f_bk, 0, 0);
#endif
    fetch_next();
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((T::kFive ? 1 : 2) * (8 + T::kFetchB)) : "memory");

  // ---- tile after tile
  // the ring: where a stage's operands and the next ones lie (bytes into lds)
  int ring[T::kFive ? 5 : 3];
#pragma unroll
  for (int i = 0; i < (T::kFive ? 5 : 3); ++i) ring[i] = i * T::kPlace;
  int stored = 0;  // a tile has just been stored
  for (; id < id_end; id += step) {
    f32x4 acc[8][kCT];
#pragma unroll
    for (int a = 0; a < 8; ++a) {
#pragma unroll
      for (int b = 0; b < kCT; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bf16x8 x[8], y0[kCT], y1[kCT];
    {
      const char *a = lds + ring[0], *b = lds + (T::kFive ? ring[1] : ring[0] + T::kA);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = loss_operand<T::kTrA>(a, i, 0, a_pos.half[0], a_pos.turn);
#pragma unroll
      for (int i = 0; i < kCT; ++i) y0[i] = loss_operand<T::kTrB>(b, i, 0, b_pos.half[0], b_pos.turn);
    }
    const Place here = locate(id);
    const int nk = stages_of(sums_of_split(here.split));
    char* scratch = lds + T::kOperands;
    for (int kb = 0; kb < nk; ++kb) {
      const bool last = kb + 1 == nk;
      if constexpr (T::kFive) {
        // places: this stage's A and B, the next one's, and a free one, which takes
        // A of the stage after; its B takes this A's place from the middle on
        char *a = lds + ring[0], *b = lds + ring[1], *a1 = lds + ring[2], *b1 = lds + ring[3], *a2 = lds + ring[4];
        scratch = b;  // read by the middle of the stage, and not yet taken again
        loss_half<kPass, kCols, 8, 0>(a, b, 1, a_pos, b_pos, a2 + a_dst, nullptr, ar, br, a_off, b_off, f_ak, f_bk, x, y0, y1, acc);
        // the next stage has landed for every wave, and every wave has read this one
        landed<T::kAhead, T::kAheadStores>(stored);
        if (kPass == kGrad && last) loss_columns(p, here.c0, wave, lane, scratch);
        loss_half<kPass, kCols, 0, T::kFetchB>(a1, b1, 0, a_pos, b_pos, nullptr, a + b_dst, ar, br, a_off, b_off, f_ak, f_bk,
                                               x, y1, y0, acc);
        const int r0 = ring[0], r1 = ring[1];
        ring[0] = ring[2];
        ring[1] = ring[3];
        ring[2] = ring[4];
        ring[3] = r0;
        ring[4] = r1;
      } else {
        char *cur = lds + ring[0], *next = lds + ring[1];
        loss_half<kPass, kCols, 0, 0>(cur, cur + T::kA, 1, a_pos, b_pos, nullptr, nullptr, ar, br, a_off, b_off, 0, 0, x, y0,
                                      y1, acc);
        landed<T::kAhead, T::kAheadStores>(stored);
        if (kPass == kGrad && last) loss_columns(p, here.c0, wave, lane, scratch);
        loss_half<kPass, kCols, 8, T::kFetchB>(next, next + T::kA, 0, a_pos, b_pos, cur + a_dst, cur + T::kA + b_dst, ar, br,
                                               a_off, b_off, f_ak, f_bk, x, y1, y0, acc);
        const int r0 = ring[0];
        ring[0] = ring[1];
        ring[1] = ring[2];
        ring[2] = r0;
      }
      fetch_next();
      asm volatile("s_mov_b32 %0, 0" : "=s"(stored));  // (a constant from here on would have the first stage peeled)
    }

    sums_ready();
    // ---- the tile is done: lane (j, g) holds rows 16 a + 4 g + e and column 16 b + j of its wave's part
    const int r0 = here.r0, c0 = here.c0;
    int l = lane;
    asm volatile("" : "+v"(l));  // (what follows is computed here, not kept in registers over the products)
    const int ej = l & 15, eg = l >> 4;
    const int row0 = 128 * wr + 4 * eg, col0 = 16 * kCT * wc + ej;
    const int row8 = 128 * wr + 16 * (eg & 1) + 4 * (eg & 2);  // after an exchange: 8 rows from 16 a + this on, a even
    const bool tail = V - r0 < kRows;  // (uniform; kGrad) the tile ends past the vocabulary
    if constexpr (kPass == kStats) {
      // the wave's rows, counted from row0: those past them count nothing; whole blocks of 16 are left out where
      // tiles may be smaller (elsewhere the branches cost more, 4 % of 300 or 2048 rows)
      const int rows = (V - r0 < p.tile_rows ? V - r0 : p.tile_rows) - 128 * wr;
      constexpr bool kSkip = kCols <= kFewRows;
      const CapSeries series(p.cap, kLog2e);
      float2* sums_of = (float2*)scratch;  // [2][kCols]
#pragma unroll
      for (int b = 0; b < kCT; ++b) {
        order();
        if (kSkip ? (rows & 15) != 0 : tail) {  // (the vocabulary's last tile)
#pragma unroll
          for (int a = 0; a < 8; ++a) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * a + 4 * eg + e >= rows) acc[a][b][e] = -__builtin_inff();
          }
        }
        float lo = __builtin_inff(), mx = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          if (kSkip && 16 * a >= rows) continue;  // (uniform, here and below)
          const f32x4 x = acc[a][b];
          mx = __builtin_fmaxf(__builtin_fmaxf(mx, x[0]), x[1]);
          mx = __builtin_fmaxf(__builtin_fmaxf(mx, x[2]), x[3]);
          if (kCap) {
            lo = __builtin_fminf(__builtin_fminf(lo, x[0]), x[1]);
            lo = __builtin_fminf(__builtin_fminf(lo, x[2]), x[3]);
          }
        }
        if (!kCap) {
          mx = __builtin_fmaxf(mx, kLowest);
          const float ml = -mx * kLog2e;
#pragma unroll
          for (int a = 0; a < 8; ++a) {
            if (kSkip && 16 * a >= rows) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[a][b][e], kLog2e, ml));
          }
        } else {
          const bool near = lo > -series.far && mx < series.far;  // (false with a masked row; a NaN stays one either way)
          mx = p.cap * cap_any(mx / p.cap);                       // tanh keeps the order; as near as the terms are
          const float ml = -mx * kLog2e;
          if (__all(near)) {
#pragma unroll
            for (int a = 0; a < 8; ++a) {
              if (kSkip && 16 * a >= rows) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = acc[a][b][e];
                sum += __builtin_amdgcn_exp2f(__builtin_fmaf(x, series(x * x), ml));
              }
            }
          } else {
#pragma unroll
            for (int a = 0; a < 8; ++a) {
              if (kSkip && 16 * a >= rows) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(p.cap * cap_any(acc[a][b][e] / p.cap), kLog2e, ml));
                sum += (kSkip || tail) && 16 * a + 4 * eg + e >= rows ? 0.0f : v;
              }
            }
          }
        }
        // the four lane groups of a column
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) join_sums(mx, sum, __shfl_xor(mx, d), __shfl_xor(sum, d));
        if (eg == 0) sums_of[wr * kCols + col0 + 16 * b] = make_float2(mx, sum);
      }
      lds_barrier();
      if (tid < kCols && c0 + tid < M) {
        float2 s = sums_of[tid];
        const float2 o = sums_of[kCols + tid];
        join_sums(s.x, s.y, o.x, o.y);
        p.stats[(size_t)(r0 / p.tile_rows) * M + c0 + tid] = s;
      }
      lds_barrier();  // read before a fetch takes the place
    } else if constexpr (kPass == kGrad) {
      const CapSeries series(p.cap, kLog2e);
      const float per_cap2 = 1.0f / (p.cap * kLog2e) / (p.cap * kLog2e);  // (finite where the series is taken)
      // the columns' values have landed for every wave; the next tile's fetches may be under way
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(T::kFive ? T::kFetchB : 8 + T::kFetchB) : "memory");
      const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.G + (size_t)c0 * p.g_stride), (short)0, (M - c0 < kCols ? M - c0 : kCols) * p.g_stride * 2, kBufferWord3);
#pragma unroll
      for (int b = 0; b < kCT; ++b) {
        order();
        const int col = col0 + 16 * b;
        const Column c = ((const Column*)scratch)[col];
        const bool scored = c.target >= 0;
        const int hit = c.target - p.v_base - r0 - row0;  // the target's place among this lane's rows
        const bool any_hit = __any(scored && hit >= 0 && hit < 128);
        bool near = true;
        if (kCap) {
          float most = 0.0f;
#pragma unroll
          for (int a = 0; a < 8; ++a) {
            const f32x4 x = acc[a][b];
            most = __builtin_fmaxf(__builtin_fmaxf(most, __builtin_fabsf(x[0])), __builtin_fabsf(x[1]));
            most = __builtin_fmaxf(__builtin_fmaxf(most, __builtin_fabsf(x[2])), __builtin_fabsf(x[3]));
          }
          near = __all(most < series.far);
        }
        // With a cap: y = z log2(e) by the series, else (uniform) 2 z / cap, in x's place; both of its uses
        // hold their range for any finite cap (z log2(e) over the cap's square would not).
        const float y_log2 = near ? 1.0f : p.cap * (0.5f * kLog2e);
        const float y_slope = near ? -per_cap2 * c.share : -0.25f * c.share;
        if (kCap && !near) {
#pragma unroll
          for (int a = 0; a < 8; ++a) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][b][e] = 2.0f * cap_any(acc[a][b][e] / p.cap);
          }
        }
        MxU32x2 w[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          float v[4], slope[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = acc[a][b][e];
            if (!kCap) {
              v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, c.ll));
              slope[e] = c.share;
            } else {
              // the probability, and share (1 - (z / cap)^2)
              const float y = near ? x * series(x * x) : x;
              v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(y, y_log2, c.ll));
              slope[e] = __builtin_fmaf(y * y, y_slope, c.share);
            }
          }
          if (any_hit) {  // (uniform)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hit == 16 * a + e) v[e] -= 1.0f;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= slope[e];
          if (tail) {  // zeros past the vocabulary
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (r0 + row0 + 16 * a + e >= V) v[e] = 0.0f;
          }
          // a row that is not scored has no gradient, whatever its hidden state holds
          w[a] = MxU32x2{scored ? pack_bf16(v[0], v[1]) : 0u, scored ? pack_bf16(v[2], v[3]) : 0u};
        }
#pragma unroll
        for (int a = 0; a < 8; a += 2)
          __builtin_amdgcn_raw_buffer_store_b128(eight_rows(w[a], w[a + 1]), out,
                                                 (uint32_t)((col * p.g_stride + r0 + row8 + 16 * a) * 2), 0, 0);
      }
      lds_barrier();  // the columns' values are read before a fetch takes the place
    } else if constexpr (kPass == kHidden) {
      const int rows = M - c0 < kCols ? M - c0 : kCols;
      const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.part + ((size_t)here.split * M + c0) * D), (short)0, rows * D * 4, kBufferWord3);
#pragma unroll
      for (int b = 0; b < kCT; ++b) {
        order();
        uint32_t o[8];
        f32x4 v[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          const int k = r0 + row0 + 16 * a;
          o[a] = k < D ? (uint32_t)(((col0 + 16 * b) * D + k) * 4) : kBufferOutOfRange;
          v[a] = acc[a][b];
          if (p.accumulate) v[a] += __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(out, o[a], 0, 0));
        }
#pragma unroll
        for (int a = 0; a < 8; ++a) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(MxU32x4, v[a]), out, o[a], 0, 0);
      }
    } else {
      const float most = *p.most;
      const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.dW + (size_t)c0 * D), (short)0, (V - c0 < kCols ? V - c0 : kCols) * D * 2, kBufferWord3);
#pragma unroll
      for (int b = 0; b < kCT; ++b) {
        order();
#pragma unroll
        for (int a = 0; a < 8; a += 2) {
          const f32x4 v = acc[a][b] * most, u = acc[a + 1][b] * most;
          const int k = r0 + row8 + 16 * a;
          __builtin_amdgcn_raw_buffer_store_b128(
              eight_rows(MxU32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])},
                         MxU32x2{pack_bf16(u[0], u[1]), pack_bf16(u[2], u[3])}),
              out, k < D ? (uint32_t)(((col0 + 16 * b) * D + k) * 2) : kBufferOutOfRange, 0, 0);
        }
      }
    }
    stored = 1;
  }
  // no fetch is under way to LDS that the next workgroup may get
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// lse and loss, four rows a workgroup: each wave takes one row's target logit, a
// dot product; 64 threads a row join the tiles' (max, sum), then one another's,
// in one order. All latency: few rows a workgroup, and the loads of several tiles
// under way (100 rows of 593 tiles: 6.4 us, 11 with eight rows a workgroup).
constexpr int kJoinRows = 4, kJoinThreads = 256, kJoinAhead = 8;
__global__ __launch_bounds__(kJoinThreads) void loss_join_kernel(const float2* __restrict__ stats, int n_tiles,
                                                                 const uint16_t* __restrict__ H,
                                                                 const uint16_t* __restrict__ W,
                                                                 const int32_t* __restrict__ targets, int M, int D,
                                                                 int V, float cap, float* __restrict__ loss,
                                                                 float* __restrict__ lse) {
  __shared__ float2 of_wave[4][kJoinRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m0 = (int)blockIdx.x * kJoinRows;
  // the wave's own row
  const int own = m0 + wave;
  const int64_t t = own < M ? targets[own] : -1;
  const bool scored = t >= 0 && t < V;
  float z = 0.0f;
  if (scored) {
    for (int c = lane * 8; c < D; c += 512) {
      float x[8], y[8];
      load_8<true>(H, (int64_t)own * D + c, 8, x);
      load_8<true>(W, t * D + c, 8, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) z = __builtin_fmaf(x[e], y[e], z);
    }
  }
  // the rows' tiles
  const int i = tid & (kJoinRows - 1);
  float mx = kLowest, sum = 0.0f;
  if (m0 + i < M) {
#pragma unroll kJoinAhead
    for (int tile = tid / kJoinRows; tile < n_tiles; tile += kJoinThreads / kJoinRows) {
      const float2 o = stats[(size_t)tile * M + m0 + i];
      join_sums(mx, sum, o.x, o.y);
    }
  }
#pragma unroll
  for (int d = kJoinRows; d < 64; d <<= 1) join_sums(mx, sum, __shfl_xor(mx, d), __shfl_xor(sum, d));
  if (lane < kJoinRows) of_wave[wave][lane] = make_float2(mx, sum);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) z += __shfl_xor(z, d);
  __syncthreads();
  if (lane == 0 && own < M) {
    float2 s = of_wave[0][wave];
#pragma unroll
    for (int w = 1; w < 4; ++w) join_sums(s.x, s.y, of_wave[w][wave].x, of_wave[w][wave].y);
    const float l = s.x + logf(s.y);
    if (cap > 0.0f) z = cap * tanhf(z / cap);
    lse[own] = l;
    // (z's sum is in another order than the one in l: at a certain target the difference may come out below 0)
    const float d = l - z;
    loss[own] = !scored || d < 0.0f ? 0.0f : d;  // (a NaN stays one)
  }
}

// The first workgroup: the largest finite |dloss| of the scored rows (1 where it is
// 0: an infinity or a NaN is then the share of its own row, and no other row meets
// it), and then every row's values for kGrad. The
// others (for dW): H with zeros in the rows that are not scored; their g is zero,
// but zero times what a padded row may hold need not be. (One launch less: 1 us of 164 at 300 x 704 x 50257.)
constexpr int kColumnThreads = 1024;
__global__ __launch_bounds__(kColumnThreads) void loss_columns_kernel(
    const float* __restrict__ dloss, const int32_t* __restrict__ targets, const float* __restrict__ lse,
    const uint16_t* __restrict__ H, int M, int V, int D, int64_t n, float* __restrict__ most,
    Column* __restrict__ columns, uint16_t* __restrict__ scored) {
  if (blockIdx.x > 0) {
    const int64_t e = ((int64_t)(blockIdx.x - 1) * kColumnThreads + threadIdx.x) * 8;
    if (e >= n) return;
    const int t = targets[e / D];
    const MxU32x4 z = {0, 0, 0, 0};
    *(MxU32x4*)&scored[e] = t >= 0 && t < V ? *(const MxU32x4*)&H[e] : z;
    return;
  }
  __shared__ uint32_t wave_most[kColumnThreads / 64];
  uint32_t b = 0;
  for (int m = threadIdx.x; m < M; m += kColumnThreads) {
    const int t = targets[m];
    const uint32_t d = t >= 0 && t < V ? __float_as_uint(dloss[m]) & 0x7fffffffu : 0u;
    b = d > b && d < 0x7f800000u ? d : b;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)b, d);
    b = o > b ? o : b;
  }
  if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = b;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kColumnThreads / 64; ++i) b = wave_most[i] > b ? wave_most[i] : b;
  const float top = b ? __uint_as_float(b) : 1.0f;
  if (threadIdx.x == 0) *most = top;
  for (int m = threadIdx.x; m < M; m += kColumnThreads) {
    const int t = targets[m];
    columns[m] = Column{t < V ? t : -1, -lse[m] * kLog2e, dloss[m] / top, 0.0f};
  }
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

template <Pass kPass, int kCols>
void loss_launch_cols(const LossArgs& p, int cus, hipStream_t s) {
  const int total = p.row_tiles * p.col_tiles * p.splits;
  const dim3 grid((unsigned)std::min((total + 7) / 8 * 8, std::max(8, cus / 8 * 8))), block(kLossThreads);
  if constexpr (kPass == kStats || kPass == kGrad) {
    if (p.cap > 0.0f) {
      loss_kernel<kPass, kCols, true><<<grid, block, 0, s>>>(p);
      return;
    }
  }
  loss_kernel<kPass, kCols, false><<<grid, block, 0, s>>>(p);
}

template <Pass kPass>
void loss_launch(const LossArgs& p, int cols, int cus, hipStream_t s) {
  if constexpr (kPass == kWeight) {
    loss_launch_cols<kPass, 256>(p, cus, s);
  } else {
    switch (cols) {
      case 64: loss_launch_cols<kPass, 64>(p, cus, s); break;
      case 128: loss_launch_cols<kPass, 128>(p, cus, s); break;
      case 160: loss_launch_cols<kPass, 160>(p, cus, s); break;
      case 192: loss_launch_cols<kPass, 192>(p, cus, s); break;
      default: loss_launch_cols<kPass, 256>(p, cus, s);
    }
  }
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

LossPlan loss_plan(int32_t rows, int32_t width, int32_t vocab, int32_t cu_count) {
  LossPlan q{};
  const int cus = cu_count > 0 ? cu_count : 256;
  q.cus = cus;
  q.v_tiles = (vocab + kRows - 1) / kRows;
  // The columns of a tile: a stage takes the matrix cores 8 cycles a column, the
  // LDS 768 and 3 a column (its reads by four waves and its writes), an epilogue
  // about 80 a column; the tiles go out in rounds of a workgroup a compute unit.
  int64_t least = INT64_MAX;
  for (const int c : {256, 192, 160, 128, 64}) {
    const int64_t tiles = (int64_t)q.v_tiles * ((rows + c - 1) / c);
    const int64_t cost = (tiles + cus - 1) / cus * ((int64_t)(width / kBlock) * std::max(8 * c, 768 + 3 * c) + 80 * c);
    if (cost < least) {
      least = cost;
      q.cols = c;
    }
  }
  // The forward pass of few rows waits for W's bytes, and its last round of tiles is
  // as long as the others: tiles as small as the same number of rounds takes (a call
  // at 100 x 2048 x 151643 128 us, 139 with tiles of 256; at 128 x 1536 x 200000 141
  // and 153). Not within one round (17 x 704 x 32768: 21.9 us, and 20.6 with 256).
  q.stat_rows = kRows;
  const int64_t col_tiles = (rows + q.cols - 1) / q.cols, rounds = (q.v_tiles * col_tiles + cus - 1) / cus;
  if (q.cols <= kFewRows && rounds > 1) {
    const int64_t places = rounds * cus / col_tiles;  // at least v_tiles
    q.stat_rows = (int32_t)(((vocab + places - 1) / places + 15) / 16 * 16);
  }
  q.stat_tiles = (vocab + q.stat_rows - 1) / q.stat_rows;
  // a piece: at most 256 MB of g, and its offsets (and W's) within 31 bits
  int64_t piece = ((int64_t)256 << 20) / ((int64_t)rows * 2);
  piece = std::min<int64_t>(piece, ((int64_t)1 << 30) / width - 256);
  piece = std::max<int64_t>(256, piece / 256 * 256);
  q.piece = (int32_t)std::min<int64_t>(piece, (int64_t)q.v_tiles * 256);
  const int tiles = (width + kRows - 1) / kRows * ((rows + q.cols - 1) / q.cols);
  q.splits = std::max(1, std::min(cus / tiles, q.piece / 256));
  q.stats_bytes = up256((size_t)q.stat_tiles * rows * sizeof(float2));
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
  p.tile_rows = plan.stat_rows;
  p.row_tiles = plan.stat_tiles;
  p.col_tiles = (rows + plan.cols - 1) / plan.cols;
  p.splits = 1;
  loss_launch<kStats>(p, plan.cols, plan.cus, s);
  loss_join_kernel<<<dim3((unsigned)((rows + kJoinRows - 1) / kJoinRows)), dim3(kJoinThreads), 0, s>>>(
      p.stats, plan.stat_tiles, hidden, weight, targets, rows, width, vocab, softcap, loss, lse);
}

void launch_lmhead_loss_grad(const uint16_t* hidden, const uint16_t* weight, const int32_t* targets, const float* lse,
                             const float* dloss, int32_t rows, int32_t width, int32_t vocab, float softcap,
                             const LossPlan& plan, uint8_t* work, uint16_t* dhidden, uint16_t* dweight, hipStream_t s) {
  const int64_t n = (int64_t)rows * width;
  const dim3 per8((unsigned)((n / 8 + 255) / 256)), block(256);
  uint16_t* scored = (uint16_t*)(work + plan.g_bytes);
  float* part = (float*)(work + plan.g_bytes + plan.h_bytes);
  float* most = (float*)(work + plan.g_bytes + plan.h_bytes + plan.part_bytes);
  Column* columns = (Column*)(most + 64);
  const int64_t row_blocks = dweight ? (n / 8 + kColumnThreads - 1) / kColumnThreads : 0;
  loss_columns_kernel<<<dim3((unsigned)(1 + row_blocks)), dim3(kColumnThreads), 0, s>>>(
      dloss, targets, lse, hidden, rows, vocab, width, n, most, columns, scored);
  const int k_tiles = (width + kRows - 1) / kRows;
  int splits = 1;
  for (int32_t v = 0; v < vocab; v += plan.piece) {
    LossArgs p{};
    p.W = weight + (size_t)v * width;
    p.H = hidden;
    p.G = (uint16_t*)work;
    p.columns = columns;
    p.most = most;
    p.part = part;
    p.cap = softcap;
    p.M = rows;
    p.D = width;
    p.V = std::min(plan.piece, vocab - v);
    p.v_base = v;
    p.g_stride = (p.V + 255) / 256 * 256;
    p.row_tiles = p.g_stride / 256;
    p.col_tiles = (rows + plan.cols - 1) / plan.cols;
    p.splits = 1;
    loss_launch<kGrad>(p, plan.cols, plan.cus, s);
    if (dhidden) {
      // every piece fills the same shares: the last, shorter one in shorter runs
      p.row_tiles = k_tiles;
      if (v == 0) splits = std::min(plan.splits, p.g_stride / 256);
      p.splits = splits;
      p.split_rows = ((p.V + splits - 1) / splits + kBlock - 1) / kBlock * kBlock;
      p.accumulate = v > 0;
      loss_launch<kHidden>(p, plan.cols, plan.cus, s);
    }
    if (dweight) {
      p.H = scored;
      p.dW = dweight + (size_t)v * width;
      p.row_tiles = k_tiles;
      p.col_tiles = p.g_stride / 256;
      p.splits = 1;
      loss_launch<kWeight>(p, 256, plan.cus, s);
    }
  }
  if (dhidden) loss_hidden_kernel<<<per8, block, 0, s>>>(part, splits, n, targets, most, vocab, width, dhidden);
}

}  // namespace gs

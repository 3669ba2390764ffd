// MXFP4 x MXFP4 on tiles staged through LDS, for products that fill the CUs with them
// (l2c_matmul_mxfp4, l2c_mx4gemm.hip, which also holds the operands' layout and what
// happens past the end of K).
//
//  * v_mfma_scale_f32_32x32x64_f8f6f4 in format E2M1: lane (r, h) = (l % 32, l / 32)
//    supplies one 32-value block of row r, 16 bytes, and its scale byte.
//  * A workgroup of 8 waves computes a tile of 2 MI x 2 NI blocks of 32 x 32; its waves
//    are 2 x 2 sub-tiles of MI x NI such blocks, twice: the two groups take half of
//    every step's k each, and their sums are added at the end through LDS. Waves of the
//    two groups share a SIMD, so one reads fragments while the other multiplies, and a
//    wave's sub-tile is twice as large as with eight, which saves a quarter of the LDS
//    reads (256 x 128: 96 KB in 1024 cycles of MFMA a step).
//  * A step is 256 k: 128 bytes a row, a whole cache line. LDS DMA (16 B a lane) fills
//    STAGES stages, all but one under way while a step is multiplied. The 16-byte
//    blocks of a row are stored XOR-swizzled by the row.
//  * Which block of a step a lane multiplies when is free, as long as X and W agree:
//    half h of group g takes blocks 4 h + 2 g and 4 h + 2 g + 1, whose scale bytes are
//    neighbours in the word that both MFMAs take their byte from.
//  * Scales: every eight steps lane l of the workgroup loads the 64 scale bytes of row l of
//    the tile (any alignment), and stores 16 of them to LDS every second step, where the
//    waves read two words a fragment. Each load costs a cache line, however little of it
//    is used: loaded by each wave for itself, two bytes a lane and fragment, they took as
//    much of L2 as the codes (1024 x 16384 x 8192 158 us), 16 bytes a row every two steps
//    a third (82 us).
//  * Rows past the operands re-read the last row, steps past the end the last block, scales
//    past the last whole step the ones before: every access is inside the operands.
//    K >= 512.
//  * 1024 x 16384 x 8192 takes 77 to 82 us, 3.5 PFLOP/s, with the matrix cores busy 0.46 of
//    the time. Copies of the kernel with parts left out take 65.5 us with staging alone
//    and 56 with the products, or the products and the fragments' reads, alone; so staging is the
//    longer part, and they overlap only in part. Staging brings 805 MB at 12 TB/s, of which 143
//    MB miss L2, and takes no longer a step where rows are no power of two apart (lengths of 15872 and
//    16640: 66.8 and 68.4 us). The clock is 1.84 GHz, with the products alone 1.90, with staging
//    alone 2.35. 256 x 4096 x 11008 on 128 x 128: 16.9, staging alone 13.4, products alone 11.7.
#include <type_traits>

#include "l2c_common.h"
#include "l2c_mx4gemm.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef __attribute__((address_space(3))) void lds_ptr;

constexpr int kE2M1 = 4;
constexpr int kThreads = 512;
constexpr int kRow = 128;  // code bytes of a row and step
constexpr int kQueue = 4;  // pairs of steps whose scales a lane loads at once

using First = std::integral_constant<int, 0>;
using Second = std::integral_constant<int, 1>;

// A block's codes as an MFMA operand, of which E2M1 uses half.
__device__ __forceinline__ i32x8 wide(u32x4 v) {
  i32x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = static_cast<int>(v[e]);
  return w;
}

// The column of a row's block b is b ^ swizzle(row): 16 lanes of ds_read_b128 that are
// served together then meet every bank once (by row % 8 half the cycles were conflicts).
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned char *dst, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr *)dst, 16, voffset, soffset, 0, 0);
}

template <int MI, int NI, int STAGES>
struct Tile {
  static constexpr int kStages = STAGES;
  static constexpr int kBM = 64 * MI, kBN = 64 * NI;
  static constexpr int kStage = (kBM + kBN) * kRow;
  static constexpr int kDma = (kBM + kBN) / 64;  // a wave's DMAs of 8 rows a step
  static constexpr int kScales = kStages * kStage;  // 16 scale bytes a row of the tile
  static constexpr int kExchange = 8 * MI * NI * 512 * 4;
  static constexpr int kLds = kScales + 16 * (kBM + kBN) > kExchange ? kScales + 16 * (kBM + kBN) : kExchange;
  static_assert(kBM + kBN <= kThreads, "a lane loads the scales of one row");
};

template <int MI, int NI, int STAGES>
__global__ __launch_bounds__(kThreads) void mxfp4_tile_kernel(float *__restrict__ out, const uint8_t *__restrict__ X,
                                                              const uint8_t *__restrict__ Xs,
                                                              const uint8_t *__restrict__ W,
                                                              const uint8_t *__restrict__ Ws, int M, int N,
                                                              int blocks) {
  using T = Tile<MI, NI, STAGES>;
  constexpr int kStages = STAGES;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[T::kLds];
  const int tile = l2c::xcd_tile(blockIdx.x, gridDim.x);
  const int mtiles = (M + T::kBM - 1) / T::kBM;
  const int m0 = tile % mtiles * T::kBM, n0 = tile / mtiles * T::kBN;
  const int mrows = min(T::kBM, M - m0), nrows = min(T::kBN, N - n0);
  const int lane = threadIdx.x % L2C_WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int g = wave >> 2, p = wave & 3, wm = p & 1, wn = p >> 1;
  const int r = lane % 32, h = lane / 32;
  const int pitch = 16 * blocks;
  const int full = blocks / 8, rest = blocks % 8, steps = full + (rest != 0);
  const __amdgpu_buffer_rsrc_t rx =
      l2c::buffer_rsrc(X + static_cast<size_t>(m0) * pitch, static_cast<uint32_t>(mrows) * pitch);
  const __amdgpu_buffer_rsrc_t rw =
      l2c::buffer_rsrc(W + static_cast<size_t>(n0) * pitch, static_cast<uint32_t>(nrows) * pitch);
  // DMA i of a wave fills rows 8 (8 i + wave) + lane / 8 of the tile's X then W rows, column
  // lane % 8 with block column ^ swizzle(row). Rows of X are whole multiples of 64.
  const int dblock = (lane % 8) ^ swizzle(8 * wave + lane / 8);
  int source[T::kDma];
#pragma unroll
  for (int i = 0; i < T::kDma; ++i) {
    const int row = 8 * (8 * i + wave) + lane / 8;
    source[i] = i < MI ? min(row, mrows - 1) * pitch : min(row - T::kBM, nrows - 1) * pitch;
  }
  const int sblock = 4 * h + 2 * g;
  // The lane's row of scales, and where it goes; lanes past the tile's rows load its last.
  const int srow = min(static_cast<int>(threadIdx.x), T::kBM + T::kBN - 1);
  const uint8_t *const scales =
      srow < T::kBM ? Xs + static_cast<size_t>(m0 + min(srow, mrows - 1)) * blocks
                    : Ws + static_cast<size_t>(n0 + min(srow - T::kBM, nrows - 1)) * blocks;
  u32x4 queue[kQueue];  // of pair u in queue[u % kQueue]
  auto load_scales = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kQueue; ++k)
      queue[k] = *reinterpret_cast<const u32x4_any *>(scales + min(16 * (u + k), 8 * full - 16));
  };
  auto store_scales = [&](u32x4 words) __attribute__((always_inline)) {
    *reinterpret_cast<u32x4 *>(lds + T::kScales + 16 * srow) = words;
  };
  // Of each fragment's row, the word of the lane's blocks in both steps; group 1's are in
  // its upper half.
  struct Scales {
    unsigned x[MI][2], w[NI][2];
  };
  auto read_scales = [&](Scales &s, int k) __attribute__((always_inline)) {  // of fragment k
    const int row = k < NI ? T::kBM + 32 * (NI * wn + k) + r : 32 * (MI * wm + k - NI) + r;
    const unsigned *word = reinterpret_cast<const unsigned *>(lds + T::kScales + 16 * row + 4 * h);
#pragma unroll
    for (int p = 0; p < 2; ++p) (k < NI ? s.w[k][p] : s.x[k - NI][p]) = word[2 * p];
  };
  // The last step's blocks past the end are the last one.
  auto dma = [&](int stage, int t, int i) __attribute__((always_inline)) {
    const int block = 16 * (t < full ? dblock : min(dblock, rest - 1));
    dma16(i < MI ? rx : rw, lds + stage * T::kStage + (8 * i + wave) * 1024, source[i] + block, kRow * t);
  };
  auto dma_step = [&](int stage, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T::kDma; ++i) dma(stage, t, i);
  };
  // All but the DMAs of this wave's newest steps have landed and its LDS accesses are done;
  // then the workgroup's barrier. Nothing is scheduled across it. (The loads of scales
  // come ahead of the DMAs; wherever they are, they make the wait stricter.)
  auto sync = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kStages - 2) * T::kDma) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  u32x4 fa[2][MI], fb[2][NI];
  const int ra = (32 * MI * wm + r) * kRow, rb = (T::kBM + 32 * NI * wn + r) * kRow;
  constexpr int kReads = MI + NI;  // fragments of half a step, W's first
  auto read = [&](int stage, int c, int k) __attribute__((always_inline)) {
    const unsigned char *base = lds + stage * T::kStage + 16 * ((sblock + c) ^ swizzle(r));
    if (k < NI) fb[c][k] = *reinterpret_cast<const u32x4 *>(base + rb + 32 * kRow * k);
    else fa[c][k - NI] = *reinterpret_cast<const u32x4 *>(base + ra + 32 * kRow * (k - NI));
  };
  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
  auto multiply = [&](auto half, auto parity, int k, const Scales &s) __attribute__((always_inline)) {
    constexpr int c = decltype(half)::value, p = decltype(parity)::value;
    const int i = k / NI, j = k % NI;
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(fa[c][i]), wide(fb[c][j]), acc[i][j], kE2M1,
                                                                 kE2M1, c, s.x[i][p], c, s.w[j][p]);
  };
  // Step t, in stage `at`: the products of its first half, among them the reads of its
  // second half's fragments; then, with all waves past their reads of the stage, the
  // second half's, among them step t + STAGES's DMAs into the stage and the reads of step t + 1's
  // first half. One of each a product: a wave issues in order, and six DMAs in a row hold
  // up what follows them. Steps go in pairs: the second of pair u stores the scales of pair
  // u + 2 once all waves have read those of u + 1, as they do in its first.
  const int last = steps - 1;
  int at = 0;
  Scales now, next;
  auto step = [&](int t, auto parity, u32x4 words) __attribute__((always_inline)) {
    constexpr bool kOdd = decltype(parity)::value == 1;
    constexpr int kProducts = MI * NI, kRounds = kProducts > kReads ? kProducts : kReads;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (k < kProducts) multiply(First{}, parity, k, now);
      if (k < kReads) read(at, 1, k);
      __builtin_amdgcn_sched_barrier(0);
    }
    sync();
    if constexpr (kOdd) {
      store_scales(words);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int after = at == kStages - 1 ? 0 : at + 1;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (k < kProducts) multiply(Second{}, parity, k, now);
      if (k < T::kDma) dma(at, min(t + kStages, last), k);
      if (k < kReads) read(after, 0, k);
      if (!kOdd && k < kReads) read_scales(next, k);
      __builtin_amdgcn_sched_barrier(0);
    }
    at = after;
  };
  auto settle = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int i = 0; i < MI; ++i) now.x[i][p] = next.x[i][p] >> (16 * g);
#pragma unroll
      for (int j = 0; j < NI; ++j) now.w[j][p] = next.w[j][p] >> (16 * g);
    }
  };
  // The scales of the blocks past the last whole step, of which some are the last again.
  unsigned tail[kReads] = {};
  if (rest) {
    const int b0 = 8 * full + min(sblock, rest - 1), b1 = 8 * full + min(sblock + 1, rest - 1);
#pragma unroll
    for (int k = 0; k < kReads; ++k) {
      const uint8_t *s = k < MI ? Xs + static_cast<size_t>(m0 + min(32 * (MI * wm + k) + r, mrows - 1)) * blocks
                                : Ws + static_cast<size_t>(n0 + min(32 * (NI * wn + k - MI) + r, nrows - 1)) * blocks;
      tail[k] = s[b0] | s[b1] << 8;
    }
  }
  load_scales(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int s = 0; s < kStages; ++s) dma_step(s, min(s, last));
  __builtin_amdgcn_sched_barrier(0);
  store_scales(queue[0]);
#pragma unroll
  for (int k = 0; k < kQueue; ++k) asm volatile("" : "+v"(queue[k]));  // loaded here, not where they are used
#pragma unroll
  for (int k = 0; k < kReads; ++k) asm volatile("" : "+v"(tail[k]));
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kStages - 1) * T::kDma) : "memory");
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    read(0, 0, k);
    read_scales(next, k);
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // all have read pair 0's scales
  settle();
  store_scales(queue[1]);
  int t = 0;
  auto pair = [&](u32x4 words) __attribute__((always_inline)) {
    step(t, First{}, words);
    step(t + 1, Second{}, words);
    settle();
    t += 2;
  };
  // Four pairs without a branch, past which the compiler would move the products.
  static_assert(kQueue == 4, "pairs of an iteration");
  while (t + 2 * kQueue <= full) {
    pair(queue[2]);
    pair(queue[3]);
    load_scales(t / 2 + 2);
    pair(queue[0]);
    pair(queue[1]);
  }
  while (t + 2 <= full) {  // three at most: their scales are there
    pair(queue[2]);
    queue[2] = queue[3];
  }
  if (t < full) step(t, Second{}, queue[2]);  // its scales end the row, as a pair's second step's do
  if (rest) {  // the first half's fragments are read or on their way
#pragma unroll
    for (int k = 0; k < kReads; ++k) read(at, 1, k);
#pragma unroll
    for (int i = 0; i < MI; ++i) now.x[i][0] = tail[i];
#pragma unroll
    for (int j = 0; j < NI; ++j) now.w[j][0] = tail[MI + j];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < MI; ++i)
        if (sblock + c >= rest) fa[c][i] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < MI * NI; ++k) {
      multiply(First{}, First{}, k, now);
      multiply(Second{}, First{}, k, now);
    }
  }

  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  // The two groups' sums: each wave keeps half of its values and gets the other group's.
  float *const mine = reinterpret_cast<float *>(lds) + (2 * p + g) * (MI * NI * 512) + lane;
  float *const theirs = reinterpret_cast<float *>(lds) + (2 * p + 1 - g) * (MI * NI * 512) + lane;
  auto send = [&](auto half) __attribute__((always_inline)) {
    constexpr int first = 8 * decltype(half)::value;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int v = 0; v < 8; ++v) theirs[((i * NI + j) * 8 + v) * L2C_WAVE] = acc[i][j][first + v];
  };
  auto finish = [&](auto half) __attribute__((always_inline)) {
    constexpr int first = 8 * decltype(half)::value;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = 32 * (NI * wn + j) + r;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          const int m = 32 * (MI * wm + i) + 8 * ((first + v) / 4) + 4 * h + v % 4;
          const float sum = acc[i][j][first + v] + mine[((i * NI + j) * 8 + v) * L2C_WAVE];
          if (m < mrows && n < nrows) out[static_cast<size_t>(m0 + m) * N + n0 + n] = sum;
        }
    }
  };
  if (g == 0) send(Second{});
  else send(First{});
  __syncthreads();
  if (g == 0) finish(First{});
  else finish(Second{});
}

template <int MI, int NI, int STAGES>
constexpr l2c::Mx4Tile tile(double launch, double per_tile, double per_k) {
  using T = Tile<MI, NI, STAGES>;
  return {mxfp4_tile_kernel<MI, NI, STAGES>, T::kBM, T::kBN, kThreads, 16, launch, per_tile, per_k};
}

}  // namespace

const l2c::Mx4Tile l2c::mx4_lds_tiles[kMx4LdsTiles] = {
    tile<1, 1, 4>(2515, 1150, 1.166), tile<1, 2, 4>(498, 3560, 1.731), tile<2, 2, 4>(0, 5454, 2.199),
    tile<2, 3, 3>(0, 6769, 2.769), tile<4, 2, 3>(1317, 7368, 2.907)};

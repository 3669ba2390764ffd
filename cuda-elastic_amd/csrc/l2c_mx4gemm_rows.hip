// MXFP4 x MXFP4 on tiles of 16 x 16 straight from memory, for a few batch rows and for short
// K (l2c_matmul_mxfp4, l2c_mx4gemm.hip, which also holds the operands' layout and what
// happens past the end of K).
//
//  * v_mfma_scale_f32_16x16x128_f8f6f4 in format E2M1: lane (r, q) = (l % 16, l / 16)
//    supplies row r's block q, 16 bytes, and its scale byte; value v of lane l of the
//    result is C[4 (l / 16) + v][l % 16]. A fragment is one 16-byte load a lane: nothing is
//    gained by staging what a wave uses once, and tiles so small have the most waves to
//    wait for memory.
//  * The four waves of a workgroup take 512-deep groups of k in turn (group i on wave i % 4)
//    and load the next while they multiply, so that one row of weights is read in pieces of
//    256 contiguous bytes, two cache lines. The group's 16 scale bytes of a row are one
//    load; lane q uses byte q of word i for MFMA i. The waves' sums are added in wave
//    order through LDS.
//  * Bound by memory's latency: 1 x 4096 x 4096 3.6 us, of which the launch is 2.
#include "l2c_common.h"
#include "l2c_mx4gemm.h"

namespace {

using l2c::f32x4;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

constexpr int kE2M1 = 4;    // MFMA operand format
constexpr int kGroup = 16;  // blocks of a group: four MFMAs
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * L2C_WAVE;
constexpr int kTile = 16;

__device__ __forceinline__ i32x8 wide(u32x4 v) {
  i32x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = static_cast<int>(v[e]);
  return w;
}

// One operand's 16 rows of a group: codes of MFMA i, and a word whose byte q is its scale.
struct Fragments {
  u32x4 codes[4];
  u32x4 scales;

  // row: the lane's, in blocks. `zero`: blocks past the end become zero.
  __device__ __forceinline__ void load(const uint8_t *c, const uint8_t *s, size_t row, int group, int blocks, int q,
                                       bool zero) {
    if ((group + 1) * kGroup <= blocks) {
      const size_t first = row + group * kGroup;
      scales = *reinterpret_cast<const u32x4_any *>(s + first);
#pragma unroll
      for (int i = 0; i < 4; ++i) codes[i] = *reinterpret_cast<const u32x4 *>(c + 16 * (first + 4 * i + q));
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int block = group * kGroup + 4 * i + q;
      const size_t at = row + min(block, blocks - 1);
      scales[i] = static_cast<unsigned>(s[at]) << (8 * q);
      codes[i] = *reinterpret_cast<const u32x4 *>(c + 16 * at);
      if (zero && block >= blocks) codes[i] = u32x4{0u, 0u, 0u, 0u};
    }
  }
};

__global__ __launch_bounds__(kThreads) void mxfp4_rows_kernel(float *__restrict__ out, const uint8_t *__restrict__ X,
                                                              const uint8_t *__restrict__ Xs,
                                                              const uint8_t *__restrict__ W,
                                                              const uint8_t *__restrict__ Ws, int M, int N,
                                                              int blocks) {
  static_assert(kTile * kTile == kThreads, "a lane adds one output");
  __shared__ float partial[kWaves][kThreads];
  const int tile = l2c::xcd_tile(blockIdx.x, gridDim.x);
  const int mtiles = (M + kTile - 1) / kTile;
  const int m0 = tile % mtiles * kTile, n0 = tile / mtiles * kTile;
  const int lane = threadIdx.x % L2C_WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int r = lane % 16, q = lane / 16;
  const size_t xrow = static_cast<size_t>(min(m0 + r, M - 1)) * blocks;
  const size_t wrow = static_cast<size_t>(min(n0 + r, N - 1)) * blocks;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  struct Group {
    Fragments x, w;
  };
  auto load = [&](Group &g, int group) __attribute__((always_inline)) {
    g.w.load(W, Ws, wrow, group, blocks, q, false);
    g.x.load(X, Xs, xrow, group, blocks, q, true);
  };
  auto multiply = [&](const Group &g) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(g.x.codes[k]), wide(g.w.codes[k]), acc, kE2M1,
                                                             kE2M1, 0, static_cast<int>(g.x.scales[k] >> (8 * q)), 0,
                                                             static_cast<int>(g.w.scales[k] >> (8 * q)));
  };
  const int groups = (blocks + kGroup - 1) / kGroup;
  Group even, odd;
  int g = wave;
  if (g < groups) load(even, g);
  while (g < groups) {
    if (g + kWaves < groups) load(odd, g + kWaves);
    multiply(even);
    g += kWaves;
    if (g >= groups) break;
    if (g + kWaves < groups) load(even, g + kWaves);
    multiply(odd);
    g += kWaves;
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) partial[wave][v * L2C_WAVE + lane] = acc[v];
  __syncthreads();
  float sum = partial[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += partial[w][threadIdx.x];
  const int m = m0 + 4 * q + wave, n = n0 + r;  // value `wave` of lane `lane`
  if (m < M && n < N) out[static_cast<size_t>(m) * N + n] = sum;
}

}  // namespace

const l2c::Mx4Tile l2c::mx4_row_tile = {mxfp4_rows_kernel, kTile, kTile, kThreads, 1, 1919, 160, 0.462};

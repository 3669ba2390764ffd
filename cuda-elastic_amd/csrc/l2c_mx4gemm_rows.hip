// MXFP4 x MXFP4 on small tiles straight from memory, for decode batches and products that
// do not fill the CUs with the tiles of l2c_mx4gemm_tiles.hip (l2c_matmul_mxfp4,
// l2c_mx4gemm.hip, which also holds the operands' layout and what happens past the end
// of K).
//
//  * v_mfma_scale_f32_16x16x128_f8f6f4 in format E2M1: lane (r, q) = (l % 16, l / 16)
//    supplies row r's block q, 16 bytes, and its scale byte; value v of lane l of the
//    result is C[4 (l / 16) + v][l % 16]. A fragment is one 16-byte load a lane: nothing is
//    gained by staging what a wave uses once.
//  * A workgroup computes 16 MF x 16 NF outputs; its waves take 512-deep groups of k in
//    turn (group i on wave i % WAVES) and load the next while they multiply, so that
//    one row of weights is read in pieces of 256 contiguous bytes, two cache lines. The
//    group's 16 scale bytes of a row are one load; lane q uses byte q of word i for
//    MFMA i. The waves' sums are added in wave order through LDS.
#include "l2c_common.h"
#include "l2c_mx4gemm.h"

namespace {

using l2c::f32x4;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

constexpr int kE2M1 = 4;    // MFMA operand format
constexpr int kGroup = 16;  // blocks of a group: four MFMAs

__device__ __forceinline__ i32x8 wide(u32x4 v) {
  i32x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = static_cast<int>(v[e]);
  return w;
}

// One operand's 16 F rows of a group: codes of MFMA i, and a word whose byte q is its scale.
template <int F>
struct Fragments {
  u32x4 codes[F][4];
  u32x4 scales[F];

  // rows[f]: the lane's row, in blocks. `zero`: blocks past the end become zero.
  __device__ __forceinline__ void load(const uint8_t *c, const uint8_t *s, const size_t (&rows)[F], int group, int blocks,
                                       int q, bool zero) {
    if ((group + 1) * kGroup <= blocks) {
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const size_t first = rows[f] + group * kGroup;
        scales[f] = *reinterpret_cast<const u32x4_any *>(s + first);
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[f][i] = *reinterpret_cast<const u32x4 *>(c + 16 * (first + 4 * i + q));
      }
      return;
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int block = group * kGroup + 4 * i + q;
        const size_t at = rows[f] + min(block, blocks - 1);
        scales[f][i] = static_cast<unsigned>(s[at]) << (8 * q);
        codes[f][i] = *reinterpret_cast<const u32x4 *>(c + 16 * at);
        if (zero && block >= blocks) codes[f][i] = u32x4{0u, 0u, 0u, 0u};
      }
    }
  }
};

template <int MF, int NF, int WAVES>
__global__ __launch_bounds__(WAVES *L2C_WAVE) void mxfp4_rows_kernel(float *__restrict__ out, const uint8_t *__restrict__ X,
                                                                     const uint8_t *__restrict__ Xs,
                                                                     const uint8_t *__restrict__ W,
                                                                     const uint8_t *__restrict__ Ws, int M, int N,
                                                                     int blocks) {
  constexpr int kTile = 256 * MF * NF;
  __shared__ float partial[WAVES][kTile];
  const int tile = l2c::xcd_tile(blockIdx.x, gridDim.x);
  const int mtiles = (M + 16 * MF - 1) / (16 * MF);
  const int m0 = tile % mtiles * (16 * MF), n0 = tile / mtiles * (16 * NF);
  const int lane = threadIdx.x % L2C_WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int r = lane % 16, q = lane / 16;
  size_t xrows[MF], wrows[NF];
#pragma unroll
  for (int i = 0; i < MF; ++i) xrows[i] = static_cast<size_t>(min(m0 + 16 * i + r, M - 1)) * blocks;
#pragma unroll
  for (int j = 0; j < NF; ++j) wrows[j] = static_cast<size_t>(min(n0 + 16 * j + r, N - 1)) * blocks;
  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Group {
    Fragments<MF> x;
    Fragments<NF> w;
  };
  auto load = [&](Group &g, int group) __attribute__((always_inline)) {
    g.w.load(W, Ws, wrows, group, blocks, q, false);
    g.x.load(X, Xs, xrows, group, blocks, q, true);
  };
  auto multiply = [&](const Group &g) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              wide(g.x.codes[i][k]), wide(g.w.codes[j][k]), acc[i][j], kE2M1, kE2M1, 0,
              static_cast<int>(g.x.scales[i][k] >> (8 * q)), 0, static_cast<int>(g.w.scales[j][k] >> (8 * q)));
  };
  const int groups = (blocks + kGroup - 1) / kGroup;
  Group even, odd;
  int g = wave;
  if (g < groups) load(even, g);
  while (g < groups) {
    if (g + WAVES < groups) load(odd, g + WAVES);
    multiply(even);
    g += WAVES;
    if (g >= groups) break;
    if (g + WAVES < groups) load(even, g + WAVES);
    multiply(odd);
    g += WAVES;
  }
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) partial[wave][((i * NF + j) * 4 + v) * L2C_WAVE + lane] = acc[i][j][v];
  __syncthreads();
  for (int e = threadIdx.x; e < kTile; e += WAVES * L2C_WAVE) {
    float sum = partial[0][e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += partial[w][e];
    const int f = e / 256, v = e / L2C_WAVE % 4;
    const int m = m0 + f / NF * 16 + 4 * q + v, n = n0 + f % NF * 16 + r;
    if (m < M && n < N) out[static_cast<size_t>(m) * N + n] = sum;
  }
}

template <int MF, int NF, int WAVES>
constexpr l2c::Mx4Tile tile(double launch, double per_tile, double per_k) {
  return {mxfp4_rows_kernel<MF, NF, WAVES>, 16 * MF, 16 * NF, WAVES * L2C_WAVE, 1, launch, per_tile, per_k};
}

}  // namespace

const l2c::Mx4Tile l2c::mx4_row_tiles[kMx4RowTiles] = {
    tile<1, 1, 8>(1600, 350, 0.466), tile<1, 2, 8>(1230, 930, 0.745), tile<2, 2, 4>(1600, 650, 0.949),
    tile<2, 2, 8>(920, 1270, 0.949)};

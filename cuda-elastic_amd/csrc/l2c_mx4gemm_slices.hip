// MXFP4 x MXFP4 on tiles whose waves share nothing but the sum, for decode batches and
// other products of few tiles (l2c_matmul_mxfp4, l2c_mx4gemm.hip, which also holds the
// operands' layout and what happens past the end of K).
//
//  * v_mfma_scale_f32_32x32x64_f8f6f4 as in l2c_mx4gemm_tiles.hip. A workgroup computes
//    32 MI x 32 NI outputs; each of its waves multiplies the whole tile over its part of k,
//    in steps of 256, a cache line of codes a row, and has a stage of LDS of its own,
//    (MI + NI) x 4 KB, which LDS DMA fills. So nobody waits for another wave, every fragment
//    is read from LDS once, and what is under way needs no registers. The waves' sums are
//    added in wave order at the end. Eight waves for few tiles of long K, two for many of
//    short K (1024 x 288 x 8012: 28 us with eight, 14 with two).
//  * A wave waits for its stage, reads all of it to registers, asks for the next step
//    and multiplies. The wait is long, but few steps are a wave's: with a barrier twice a
//    step, as large tiles have it, a product of few tiles took 0.28 us a step for eight
//    waves together, whatever it multiplied.
//  * Lane (r, h) takes blocks 4 h to 4 h + 3 of a step, whose scale bytes are the word that
//    the four MFMAs take one byte each from. 16-byte blocks of a row are stored XOR-swizzled
//    by the row.
//  * Rows past the operands re-read the last row, blocks past the end the last block: every
//    access is inside the operands. K >= 256.
//  * Bound by memory and its latency: 1 x 4096 x 11008 6.3 us, 3.8 TB/s; 40 x 4096 x 4096 4.5 us.
#include <type_traits>

#include "l2c_common.h"
#include "l2c_mx4gemm.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64_any __attribute__((aligned(1)));
typedef __attribute__((address_space(3))) void lds_ptr;

constexpr int kE2M1 = 4;
constexpr int kRow = 128;  // code bytes of a row and step

__device__ __forceinline__ i32x8 wide(u32x4 v) {
  i32x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = static_cast<int>(v[e]);
  return w;
}

__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned char *dst, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr *)dst, 16, voffset, soffset, 0, 0);
}

template <int MI, int NI, int WAVES>
__global__ __launch_bounds__(WAVES *L2C_WAVE) void mxfp4_slice_kernel(float *__restrict__ out,
                                                                      const uint8_t *__restrict__ X,
                                                                      const uint8_t *__restrict__ Xs,
                                                                      const uint8_t *__restrict__ W,
                                                                      const uint8_t *__restrict__ Ws, int M, int N,
                                                                      int blocks) {
  constexpr int kThreads = WAVES * L2C_WAVE;
  constexpr int kBM = 32 * MI, kBN = 32 * NI, kF = MI + NI;
  constexpr int kStage = 32 * kF * kRow;
  constexpr int kSum = 1024 * MI * NI;  // values of a tile
  static_assert(kSum * 4 <= kStage, "the waves' sums fit their stages");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[WAVES * kStage];
  const int tile = l2c::xcd_tile(blockIdx.x, gridDim.x);
  const int mtiles = (M + kBM - 1) / kBM;
  const int m0 = tile % mtiles * kBM, n0 = tile / mtiles * kBN;
  const int mrows = min(kBM, M - m0), nrows = min(kBN, N - n0);
  const int lane = threadIdx.x % L2C_WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int r = lane % 32, h = lane / 32;
  const int pitch = 16 * blocks;
  const int full = blocks / 8, rest = blocks % 8, steps = full + (rest != 0);
  const __amdgpu_buffer_rsrc_t rx =
      l2c::buffer_rsrc(X + static_cast<size_t>(m0) * pitch, static_cast<uint32_t>(mrows) * pitch);
  const __amdgpu_buffer_rsrc_t rw =
      l2c::buffer_rsrc(W + static_cast<size_t>(n0) * pitch, static_cast<uint32_t>(nrows) * pitch);
  unsigned char *const stage = lds + wave * kStage;
  // DMA i fills rows 8 i + lane / 8 of the stage, column lane % 8 with block column ^
  // swizzle(row): of even and odd i they differ by 4.
  const int dblock = (lane % 8) ^ swizzle(lane / 8);
  int source[4 * kF];
#pragma unroll
  for (int i = 0; i < 4 * kF; ++i) {
    const int row = 8 * i + lane / 8;
    source[i] = i < 4 * MI ? min(row, mrows - 1) * pitch : min(row - kBM, nrows - 1) * pitch;
  }
  const uint8_t *scales[kF];
#pragma unroll
  for (int f = 0; f < kF; ++f)
    scales[f] = f < MI ? Xs + static_cast<size_t>(m0 + min(32 * f + r, mrows - 1)) * blocks
                       : Ws + static_cast<size_t>(n0 + min(32 * (f - MI) + r, nrows - 1)) * blocks;
  unsigned long long next[kF];  // a row's scales in a step; those of the last step end the row
  auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < kF; ++f) next[f] = *reinterpret_cast<const u64_any *>(scales[f] + min(8 * t, blocks - 8));
#pragma unroll
    for (int i = 0; i < 4 * kF; ++i) {
      const int block = dblock ^ (i % 2 * 4), inside = t < full ? block : min(block, rest - 1);
      dma16(i < 4 * MI ? rx : rw, stage + 1024 * i, source[i] + 16 * inside, kRow * t);
    }
  };
  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
  const int end = static_cast<int>((wave + 1LL) * steps / WAVES);
  int t = static_cast<int>(static_cast<long long>(wave) * steps / WAVES);
  if (t < end) load(t);
  for (; t < end; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    u32x4 codes[kF][4];
    unsigned scale[kF];
    const int past = t < full ? 0 : 8 - rest;  // the last step's blocks past the end: their scales become 0
#pragma unroll
    for (int f = 0; f < kF; ++f) {
      scale[f] = static_cast<unsigned>((next[f] >> (8 * past)) >> (32 * h));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        codes[f][j] = *reinterpret_cast<const u32x4 *>(stage + (32 * f + r) * kRow + 16 * ((4 * h + j) ^ swizzle(r)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + 1 < end) load(t + 1);
    if (past) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * h + j >= rest) codes[i][j] = u32x4{0u, 0u, 0u, 0u};
    }
    auto multiply = [&](auto k) __attribute__((always_inline)) {
      constexpr int c = decltype(k)::value;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(codes[i][c]), wide(codes[MI + j][c]),
                                                                       acc[i][j], kE2M1, kE2M1, c, scale[i], c,
                                                                       scale[MI + j]);
    };
    multiply(std::integral_constant<int, 0>{});
    multiply(std::integral_constant<int, 1>{});
    multiply(std::integral_constant<int, 2>{});
    multiply(std::integral_constant<int, 3>{});
  }
  float *const sums = reinterpret_cast<float *>(lds);  // in the stages: [wave][block][value][lane]
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        sums[wave * (kStage / 4) + ((i * NI + j) * 16 + v) * L2C_WAVE + lane] = acc[i][j][v];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSum / kThreads; ++k) {
    const int e = threadIdx.x + k * kThreads, block = e / 1024, v = e / L2C_WAVE % 16;
    float sum = sums[e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += sums[w * (kStage / 4) + e];
    const int m = 32 * (block / NI) + 8 * (v / 4) + 4 * h + v % 4, n = 32 * (block % NI) + r;
    if (m < mrows && n < nrows) out[static_cast<size_t>(m0 + m) * N + n0 + n] = sum;
  }
}

template <int MI, int NI, int WAVES>
constexpr l2c::Mx4Tile tile(double launch, double per_tile, double per_k) {
  return {mxfp4_slice_kernel<MI, NI, WAVES>, 32 * MI, 32 * NI, WAVES * L2C_WAVE, 8, launch, per_tile, per_k};
}

}  // namespace

const l2c::Mx4Tile l2c::mx4_slice_tiles[kMx4SliceTiles] = {
    tile<1, 1, 2>(2401, 142, 0.484), tile<1, 1, 8>(1884, 595, 0.465), tile<1, 2, 8>(1049, 1747, 0.867)};

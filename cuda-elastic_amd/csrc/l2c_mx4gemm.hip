// MXFP4 x MXFP4: activations quantized on the device and the contraction
//   out[b][r] = sum_k deq(X)[b][k] * deq(W)[r][k]
// on the scaled matrix cores, both operands E2M1 codes, two a byte, row-major, with one
// UE8M0 scale byte per 32 values, row-major too: what l2c_quantize_mxfp4 writes for
// weights and l2c_quantize_mxfp4_bf16 for activations. The codes' products are exact,
// sums are fp32.
//
// Any number of whole blocks a row (K % 32 == 0). In the last step, blocks past the end
// re-read the row's last block and X's codes there are made zero: E2M1 has no Inf or
// NaN, so such a block adds nothing, and a scale that is NaN belongs to a block that
// has made the sum NaN already.
#include <climits>

#include "l2c_common.h"
#include "l2c_mx4gemm.h"
#include "../../include/l2c.h"

namespace {

using l2c::f32x4;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kE2M1 = 4;  // MFMA operand format

// ---------------------------------------------------------------------------
// bf16 activations to MXFP4. A block's shared exponent is floor(log2(maximum)) - 2, at
// least -127: the largest value's code is 4 or 6 (what is above 7 saturates). A block
// that holds an infinity or a NaN, which E2M1 does not have, gets the scale 0xff, NaN,
// and zero codes: whatever is multiplied with it becomes NaN.
//
// A lane reads 8 values in one load, four lanes a block, and writes their 4 bytes of
// codes. Rows are whole blocks and follow each other, so the kernel knows no rows.

constexpr int kQuantThreads = 256;

__global__ __launch_bounds__(kQuantThreads) void quantize_mxfp4_bf16_kernel(uint8_t *__restrict__ codes,
                                                                            uint8_t *__restrict__ scales,
                                                                            const uint16_t *__restrict__ X,
                                                                            long long eighths) {
  const long long i = static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x;
  u32x4 raw = {0u, 0u, 0u, 0u};
  if (i < eighths) raw = reinterpret_cast<const u32x4 *>(X)[i];  // a block's four lanes are in or out together
  unsigned most = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) most = max(most, max(raw[j] & 0x7fffu, (raw[j] >> 16) & 0x7fffu));
  most = max(most, static_cast<unsigned>(__shfl_xor(static_cast<int>(most), 1)));
  most = max(most, static_cast<unsigned>(__shfl_xor(static_cast<int>(most), 2)));
  const int field = static_cast<int>(most >> 7);  // the maximum's exponent field; 255: Inf or NaN
  const int exponent = max(field - 129, -127);
  const float inv = __uint_as_float(static_cast<unsigned>(127 - min(exponent, 126)) << 23);  // 2^-exponent
  float v[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(raw[j] << 16) * inv;
    v[2 * j + 1] = __uint_as_float(raw[j] & 0xffff0000u) * inv;
  }
  // Nearest even, saturating at 6; then negative zeros, which the conversion keeps, made +0.
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
  const unsigned nonzero = ((c & 0x77777777u) + 0x77777777u) & 0x88888888u;  // 8 where magnitude != 0
  c &= nonzero | 0x77777777u;
  if (field == 255) c = 0;
  if (i < eighths) {
    reinterpret_cast<unsigned *>(codes)[i] = c;
    if ((i & 3) == 0) scales[i >> 2] = static_cast<uint8_t>(field == 255 ? 255 : exponent + 127);
  }
}

// ---------------------------------------------------------------------------
// The contraction: a workgroup computes 16 x 16 outputs, its waves every kWaves-th
// 128-deep step each, operands straight from memory into registers.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 in format E2M1: lane (r, q) = (l % 16, l / 16)
// supplies row r's block q (k 32 q .. 32 q + 31), 16 bytes, and its scale byte; value v
// of lane l of the result is C[4 (l / 16) + v][l % 16].

constexpr int kWaves = 4;

__global__ __launch_bounds__(kWaves *L2C_WAVE) void mxfp4_gemm_kernel(float *__restrict__ out,
                                                                      const uint8_t *__restrict__ X,
                                                                      const uint8_t *__restrict__ Xs,
                                                                      const uint8_t *__restrict__ W,
                                                                      const uint8_t *__restrict__ Ws, int M, int N,
                                                                      int blocks) {
  __shared__ float partial[kWaves][256];
  const int tile = l2c::xcd_tile(blockIdx.x, gridDim.x);
  const int mtiles = (M + 15) / 16;
  const int m0 = tile % mtiles * 16, n0 = tile / mtiles * 16;
  const int lane = threadIdx.x % L2C_WAVE, wave = threadIdx.x / L2C_WAVE;
  const int r = lane % 16, q = lane / 16;
  const size_t xrow = static_cast<size_t>(min(m0 + r, M - 1)) * blocks;
  const size_t wrow = static_cast<size_t>(min(n0 + r, N - 1)) * blocks;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = wave; 4 * s < blocks; s += kWaves) {
    const int block = min(4 * s + q, blocks - 1);
    u32x4 x = *reinterpret_cast<const u32x4 *>(X + 16 * (xrow + block));
    const u32x4 w = *reinterpret_cast<const u32x4 *>(W + 16 * (wrow + block));
    const int xs = Xs[xrow + block], ws = Ws[wrow + block];
    if (4 * s + q >= blocks) x = u32x4{0u, 0u, 0u, 0u};
    i32x8 a = {0, 0, 0, 0, 0, 0, 0, 0}, b = a;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = static_cast<int>(x[e]), b[e] = static_cast<int>(w[e]);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, kE2M1, kE2M1, 0, xs, 0, ws);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) partial[wave][v * L2C_WAVE + lane] = acc[v];
  __syncthreads();
  const int v = wave;  // value v of the waves' lanes
  float sum = partial[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += partial[w][threadIdx.x];
  const int m = m0 + 4 * q + v, n = n0 + r;
  if (m < M && n < N) out[static_cast<size_t>(m) * N + n] = sum;
}

}  // namespace

extern "C" int l2c_quantize_mxfp4_bf16(uint8_t *codes, uint8_t *scales, const uint16_t *Xbf16, int rows, int cols,
                                       hipStream_t stream) {
  if (rows < 0 || cols <= 0 || cols % 32 != 0) return hipErrorInvalidValue;
  if (rows == 0) return hipSuccess;
  if (!codes || !scales || !Xbf16 || !l2c_aligned16(Xbf16) || !l2c_aligned16(codes)) return hipErrorInvalidValue;
  const long long eighths = static_cast<long long>(rows) * (cols / 8);
  const long long grid = (eighths + kQuantThreads - 1) / kQuantThreads;
  if (!l2c::launchable(grid, kQuantThreads)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(quantize_mxfp4_bf16_kernel, dim3(static_cast<unsigned>(grid)), dim3(kQuantThreads), 0, stream,
                     codes, scales, Xbf16, eighths);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

extern "C" int l2c_matmul_mxfp4(float *out, const uint8_t *X, const uint8_t *Xscales, const uint8_t *W,
                                const uint8_t *Wscales, int batch, int cols, int rows, hipStream_t stream) {
  if (batch < 0 || cols <= 0 || rows < 0 || cols % 32 != 0) return hipErrorInvalidValue;
  if (batch == 0 || rows == 0) return hipSuccess;
  if (!out || !X || !Xscales || !W || !Wscales || !l2c_aligned16(X) || !l2c_aligned16(W)) return hipErrorInvalidValue;
  if (256LL * (cols / 2) > INT_MAX) return hipErrorInvalidValue;
  if (batch > 128 && l2c_mx4_tiles(out, X, Xscales, W, Wscales, batch, cols / 32, rows, stream)) {
    L2C_LAUNCH_CHECK();
    return hipSuccess;
  }
  const long long tiles = ((batch + 15LL) / 16) * ((rows + 15LL) / 16);
  if (!l2c::launchable(tiles, kWaves * L2C_WAVE)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(mxfp4_gemm_kernel, dim3(static_cast<unsigned>(tiles)), dim3(kWaves * L2C_WAVE), 0, stream, out, X,
                     Xscales, W, Wscales, batch, rows, cols / 32);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

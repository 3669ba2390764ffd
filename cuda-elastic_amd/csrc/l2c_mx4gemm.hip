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

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// bf16 activations to MXFP4. A block's shared exponent is floor(log2(maximum)) - 2, at
// least -127: the largest value's code is 4 or 6 (what is above 7 saturates). A block
// that holds an infinity or a NaN, which E2M1 does not have, gets the scale 0xff, NaN,
// and zero codes: whatever is multiplied with it becomes NaN.
//
// A lane reads 8 values in one load, four lanes a block, and writes their 4 bytes of
// codes. Rows are whole blocks and follow each other, so the kernel knows no rows. Bound by
// HBM: 1024 x 16384 9.6 us, 4.4 TB/s.

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
// Choice of the contraction's tile: the one of least estimated time. Fitted to the times of
// these and 9 other tiles on 132 shapes of 1 to 1024 x 288 to 16384 x 600 to 11008: what a
// CU takes for its tiles in turn is linear in their number and in K to about 12% in the mean,
// and the choice among these nine is 3% slower than the best of all in the mean. Where
// large tiles keep all CUs busy the estimates are too low, by more the larger the tile, but in
// order: 1024 x 16384 x 8192 56 us on 256 x 128 where it takes 82, 83 on 128 x 128 (101), 104
// on 128 x 192 (117). Measured on either side of a border, us: 1 x 4096 x 11008 6.8 on 16 x
// 16 tiles, 6.0 on 32 x 64, 8.1 on 64 x 64; 332 x 512 x 8012 7.1 on 32 x 32 by two waves, 8.0
// on 128 x 128; 64 x 4096 x 11008 11.9 on 32 x 64, 8.9 on 64 x 64; 128 x 4096 x 11008 12.9 on
// 64 x 64, 11.3 on 64 x 128; 512 x 4096 x 11008 32.3 on 128 x 128, 21.4 on 128 x 192, 24.4 on
// 256 x 128; 400 x 4096 x 11008 27.2 on 128 x 128, 21.1 on 256 x 128.

constexpr int kMaxCols = (1 << 24) - 32;  // a tile's 256 rows of codes stay within 31 bits

long long tiles_of(const l2c::Mx4Tile &t, int batch, int rows) {
  return ((batch + static_cast<long long>(t.bm) - 1) / t.bm) * ((rows + static_cast<long long>(t.bn) - 1) / t.bn);
}

const l2c::Mx4Tile *choose(int batch, int blocks, int rows) {
  const l2c::Mx4Tile *best = nullptr;
  double least = 0.0;
  auto consider = [&](const l2c::Mx4Tile &t) {
    const long long tiles = tiles_of(t, batch, rows);
    if (blocks < t.min_blocks || !l2c::launchable(tiles, t.threads)) return;
    const double cost = t.launch + static_cast<double>((tiles + 255) / 256) * (t.tile + t.k * 32.0 * blocks);
    if (!best || cost < least) best = &t, least = cost;
  };
  consider(l2c::mx4_row_tile);
  for (const l2c::Mx4Tile &t : l2c::mx4_slice_tiles) consider(t);
  for (const l2c::Mx4Tile &t : l2c::mx4_lds_tiles) consider(t);
  return best;
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
  if (cols > kMaxCols) return hipErrorInvalidValue;
  const l2c::Mx4Tile *t = choose(batch, cols / 32, rows);
  if (!t) return hipErrorInvalidValue;
  hipLaunchKernelGGL(t->fn, dim3(static_cast<unsigned>(tiles_of(*t, batch, rows))), dim3(t->threads), 0, stream, out, X,
                     Xscales, W, Wscales, batch, rows, cols / 32);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

bool l2c_mx4_launch_shape(int batch, int cols, int rows, int *grid, int *block, const void **fn) {
  const bool known = batch > 0 && rows > 0 && cols > 0 && cols % 32 == 0 && cols <= kMaxCols;
  const l2c::Mx4Tile *t = known ? choose(batch, cols / 32, rows) : nullptr;
  if (!t) return false;
  *grid = static_cast<int>(tiles_of(*t, batch, rows));
  *block = t->threads;
  *fn = reinterpret_cast<const void *>(t->fn);
  return true;
}

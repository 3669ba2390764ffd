// The sum after a block of the decoder and the norm before the next one, in one
// kernel: with block output y, residual stream x and gate g, for every row
//   z = y * (1 / sqrt(mean(y^2) + eps)) * block_weight     (z = y without block_weight)
//   h = residual_scale * x + g * z                          (g = 1 without a gate)
//   n = h * (1 / sqrt(mean(h^2) + eps)) * weight
// h is the new residual stream, n the next block's input. x and h, y, and n are
// fp32 or bf16 each; weights and gates are fp32, and so is all arithmetic. h and n
// are rounded once, to nearest even, when they are stored: n comes from the
// unrounded h.
//
// Bound by HBM: every value read and written once. A workgroup a row of up to 16384
// values, which its lanes hold in registers from the first load to the last store: eight
// values a lane and chunk, whole 16-byte loads and stores at any address the types
// allow. 1024 x 16384, fp32 to fp32 and bf16: 53 us, 4.4 TB/s (74 us with nontemporal
// loads, which pass the MALL by); 1024 x 16384 bf16 30 us; 1 x 4096 2.7 us. Longer rows are
// read three times (from HBM once: the later passes hit the caches), a value a lane and
// load, and wait for each: 16 x 20000 fp32 70 us, 200 x 131072 bf16 1310 (0.16 TB/s).
#include <type_traits>

#include "l2c_common.h"
#include "../../include/l2c.h"

namespace {

struct Args {
  void *normalized, *residual_out;
  const void *residual, *block;
  const float *block_weight, *gate, *weight;
  int size, rows_per_gate;
  float residual_scale, eps;
};

template <bool BF16>
__device__ __forceinline__ float load(const void *p, size_t i) {
  if constexpr (BF16) return __uint_as_float(static_cast<unsigned>(static_cast<const uint16_t *>(p)[i]) << 16);
  return static_cast<const float *>(p)[i];
}

__device__ __forceinline__ uint16_t to_bf16(float f) {
  const unsigned u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40u);  // NaN stays NaN
  return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <bool BF16>
__device__ __forceinline__ void store(void *p, size_t i, float v) {
  if constexpr (BF16) static_cast<uint16_t *>(p)[i] = to_bf16(v);
  else static_cast<float *>(p)[i] = v;
}

// ---------------------------------------------------------------------------
// Rows in registers.

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Values i .. i + 7 of a row.
template <bool BF16>
__device__ __forceinline__ void load8(float (&v)[8], const void *row, int i) {
  if constexpr (BF16) {
    const u32x4_any q = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(row) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(q[e] << 16);
      v[2 * e + 1] = __uint_as_float(q[e] & 0xffff0000u);
    }
  } else {
    const float4 a = l2c::ld4_any(static_cast<const float *>(row) + i);
    const float4 b = l2c::ld4_any(static_cast<const float *>(row) + i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

// The same values stored, but for the first `skip`.
template <bool BF16>
__device__ __forceinline__ void store8(void *row, int i, int skip, const float (&v)[8]) {
  if (skip == 0) {
    if constexpr (BF16) {
      u32x4_any q;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        q[e] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{v[2 * e], v[2 * e + 1]}), bf16x2));
      *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(row) + i) = q;
    } else {
      l2c::st4_any(static_cast<float *>(row) + i, make_float4(v[0], v[1], v[2], v[3]));
      l2c::st4_any(static_cast<float *>(row) + i + 4, make_float4(v[4], v[5], v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int e = 1; e < 8; ++e)
      if (e >= skip) store<BF16>(row, i + e, v[e]);
  }
}

// ss and the squares of v, but for the first `skip`.
__device__ __forceinline__ float add_squares(float ss, const float (&v)[8], int skip) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float u = e >= skip ? v[e] : 0.0f;
    ss = fmaf(u, u, ss);
  }
  return ss;
}

// The wave's sum in every lane: four shifted additions within rows of 16 lanes, two across
// them (adders' own operand paths, no trip through LDS), then lane 63's total.
__device__ __forceinline__ float wave_total(float v) {
  auto shifted = [&](auto control, auto rows) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(control)::value,
                                                      decltype(rows)::value, 0xf, true));
  };
  using std::integral_constant;
  v += shifted(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  v += shifted(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  v += shifted(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  v += shifted(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  v += shifted(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  v += shifted(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// 1 / sqrt(mean + eps) of a row whose lanes hold `ss` of its squares.
template <int THREADS>
__device__ __forceinline__ float row_scale(float ss, float *slots, int size, float eps) {
  ss = wave_total(ss);
  if constexpr (THREADS > L2C_WAVE) {
    if (threadIdx.x % L2C_WAVE == 0) slots[threadIdx.x / L2C_WAVE] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / L2C_WAVE; ++w) ss += slots[w];
  }
  return 1.0f / sqrtf(ss / static_cast<float>(size) + eps);
}

// Lane t has values 8 (t + c THREADS) .. + 7 of the row, c < V. What is left of a row of no
// multiple of eight is read and computed as the row's last eight values, of which the
// first `skip` are another lane's: not counted, not stored, and, where an output takes
// an input's place, perhaps no longer what they were. n >= 8.
template <int V, int THREADS, bool XBF, bool YBF, bool NBF>
__global__ __launch_bounds__(THREADS) void residual_rmsnorm_regs_kernel(Args a) {
  __shared__ float yslots[THREADS / L2C_WAVE], hslots[THREADS / L2C_WAVE];
  const size_t first = static_cast<size_t>(blockIdx.x) * a.size;
  const void *const xrow = static_cast<const char *>(a.residual) + first * (XBF ? 2 : 4);
  const void *const yrow = static_cast<const char *>(a.block) + first * (YBF ? 2 : 4);
  const float *const gate = a.gate ? a.gate + static_cast<size_t>(blockIdx.x / a.rows_per_gate) * a.size : nullptr;
  const int n = a.size;
  auto place = [&](int c) __attribute__((always_inline)) { return 8 * (static_cast<int>(threadIdx.x) + c * THREADS); };
  auto inside = [&](int c) __attribute__((always_inline)) { return place(c) < n; };
  auto at = [&](int c) __attribute__((always_inline)) { return min(place(c), n - 8); };
  auto skip = [&](int c) __attribute__((always_inline)) { return place(c) - at(c); };
  float y[V][8], x[V][8];
#pragma unroll
  for (int c = 0; c < V; ++c)
    if (inside(c)) load8<YBF>(y[c], yrow, at(c));
#pragma unroll
  for (int c = 0; c < V; ++c)
    if (inside(c)) load8<XBF>(x[c], xrow, at(c));
  if (a.block_weight) {
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (inside(c)) ss = add_squares(ss, y[c], skip(c));
    const float scale = row_scale<THREADS>(ss, yslots, n, a.eps);
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (inside(c)) {
        float w[8];
        load8<false>(w, a.block_weight, at(c));
#pragma unroll
        for (int e = 0; e < 8; ++e) y[c][e] *= scale * w[e];
      }
  }
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < V; ++c)
    if (inside(c)) {
      if (gate) {
        float g[8];
        load8<false>(g, gate, at(c));
#pragma unroll
        for (int e = 0; e < 8; ++e) y[c][e] *= g[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] = fmaf(a.residual_scale, x[c][e], y[c][e]);
      ss = add_squares(ss, x[c], skip(c));
    }
  if (a.residual_out) {
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (inside(c)) store8<XBF>(static_cast<char *>(a.residual_out) + first * (XBF ? 2 : 4), at(c), skip(c), x[c]);
  }
  const float scale = row_scale<THREADS>(ss, hslots, n, a.eps);
#pragma unroll
  for (int c = 0; c < V; ++c)
    if (inside(c)) {
      float w[8];
      load8<false>(w, a.weight, at(c));
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] *= scale * w[e];
      store8<NBF>(static_cast<char *>(a.normalized) + first * (NBF ? 2 : 4), at(c), skip(c), x[c]);
    }
}

// ---------------------------------------------------------------------------
// Rows that are streamed.

constexpr int kThreads = 256;

template <bool XBF, bool YBF, bool NBF>
__global__ __launch_bounds__(kThreads) void residual_rmsnorm_kernel(Args a) {
  __shared__ float yslots[kThreads / L2C_WAVE], hslots[kThreads / L2C_WAVE];
  const size_t row = static_cast<size_t>(blockIdx.x) * a.size;
  const float *gate = a.gate ? a.gate + static_cast<size_t>(blockIdx.x / a.rows_per_gate) * a.size : nullptr;
  // 64 bits: of rows whose length is near 2^31 a lane's last index, past the end, is above it (16 x 20000
  // fp32 70.7 us, with unsigned indexes, whose addresses take more instructions, 73.9).
  const long long t = threadIdx.x, size = a.size;
  float yscale = 1.0f;
  if (a.block_weight) {
    float ss = 0.0f;
    for (long long j = t; j < size; j += kThreads) {
      const float y = load<YBF>(a.block, row + j);
      ss = fmaf(y, y, ss);
    }
    yscale = 1.0f / sqrtf(l2c::block_sum(ss, yslots) / static_cast<float>(a.size) + a.eps);
  }
  auto sum = [&](long long j) __attribute__((always_inline)) {
    float z = load<YBF>(a.block, row + j);
    if (a.block_weight) z = z * yscale * a.block_weight[j];
    if (gate) z *= gate[j];
    return fmaf(a.residual_scale, load<XBF>(a.residual, row + j), z);
  };
  float ss = 0.0f;
  for (long long j = t; j < size; j += kThreads) {
    const float h = sum(j);
    ss = fmaf(h, h, ss);
  }
  const float scale = 1.0f / sqrtf(l2c::block_sum(ss, hslots) / static_cast<float>(a.size) + a.eps);
  // A lane writes only what it alone has read, after reading it: outputs may be inputs.
  for (long long j = t; j < size; j += kThreads) {
    const float h = sum(j), n = h * scale * a.weight[j];
    if (a.residual_out) store<XBF>(a.residual_out, row + j, h);
    store<NBF>(a.normalized, row + j, n);
  }
}

using Kernel = void (*)(Args);

struct Config {
  Kernel fn;
  int threads;
};

// Eight values a lane as far as 1024 lanes go, then sixteen. Rows that leave more than a
// quarter of 1024 lanes idle take sixteen values on 512 in large batches, where idle
// waves keep other rows off the CU (fp32, us: 1024 x 5003 15.1 on 512 lanes, 15.9 on 1024;
// 130 x 5003 4.9 and 4.4, 1024 x 8192 27.4 and 26.9). Fewer lanes with more values lose
// by the longer chain of one wave (1 x 4096 fp32: 3.0 us on 512 lanes, 3.7 on 256).
template <bool XBF, bool YBF, bool NBF>
Config choose(int size, int batch) {
  if (size < 8 || size > 16384) return {residual_rmsnorm_kernel<XBF, YBF, NBF>, kThreads};
  if (size <= 512) return {residual_rmsnorm_regs_kernel<1, 64, XBF, YBF, NBF>, 64};
  if (size <= 1024) return {residual_rmsnorm_regs_kernel<1, 128, XBF, YBF, NBF>, 128};
  if (size <= 2048) return {residual_rmsnorm_regs_kernel<1, 256, XBF, YBF, NBF>, 256};
  if (size <= 4096) return {residual_rmsnorm_regs_kernel<1, 512, XBF, YBF, NBF>, 512};
  if (size <= 6144 && batch > 512) return {residual_rmsnorm_regs_kernel<2, 512, XBF, YBF, NBF>, 512};
  if (size <= 8192) return {residual_rmsnorm_regs_kernel<1, 1024, XBF, YBF, NBF>, 1024};
  return {residual_rmsnorm_regs_kernel<2, 1024, XBF, YBF, NBF>, 1024};
}

template <bool XBF, bool YBF>
Config choose(bool n, int size, int batch) {
  return n ? choose<XBF, YBF, true>(size, batch) : choose<XBF, YBF, false>(size, batch);
}

bool known(int type) { return type == L2C_F32 || type == L2C_BF16; }

bool misaligned(const void *p, int type) {
  return (reinterpret_cast<uintptr_t>(p) & (type == L2C_F32 ? 3u : 1u)) != 0;
}

}  // namespace

extern "C" int l2c_residual_rmsnorm(void *normalized, int normalized_type, void *residual_out, const void *residual,
                                    int residual_type, const void *block, int block_type, const float *block_weight,
                                    const float *gate, int rows_per_gate, const float *weight, int size, int batch,
                                    float residual_scale, float eps, hipStream_t stream) {
  if (size <= 0 || batch < 0 || !known(normalized_type) || !known(residual_type) || !known(block_type) ||
      (gate && rows_per_gate <= 0))
    return hipErrorInvalidValue;
  if (batch == 0) return hipSuccess;
  if (!normalized || !residual || !block || !weight || misaligned(normalized, normalized_type) ||
      misaligned(residual_out, residual_type) || misaligned(residual, residual_type) || misaligned(block, block_type) ||
      misaligned(weight, L2C_F32) || misaligned(gate, L2C_F32) || misaligned(block_weight, L2C_F32))
    return hipErrorInvalidValue;
  // Outputs take the place of whole inputs of their own type, and not of each other.
  if (normalized == residual_out || (normalized == residual && normalized_type != residual_type) ||
      (normalized == block && normalized_type != block_type) || (residual_out == block && residual_type != block_type))
    return hipErrorInvalidValue;
  const bool x = residual_type == L2C_BF16, y = block_type == L2C_BF16, n = normalized_type == L2C_BF16;
  const Config c = x ? (y ? choose<true, true>(n, size, batch) : choose<true, false>(n, size, batch))
                     : (y ? choose<false, true>(n, size, batch) : choose<false, false>(n, size, batch));
  if (!l2c::launchable(batch, c.threads)) return hipErrorInvalidValue;
  const Args a = {normalized, residual_out, residual, block, block_weight, gate, weight,
                  size, rows_per_gate, residual_scale, eps};
  hipLaunchKernelGGL(c.fn, dim3(batch), dim3(c.threads), 0, stream, a);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

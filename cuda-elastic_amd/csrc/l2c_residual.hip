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
// A workgroup a row, the row read three times (from HBM once: the later passes hit
// the caches).
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

constexpr int kThreads = 256;

template <bool XBF, bool YBF, bool NBF>
__global__ __launch_bounds__(kThreads) void residual_rmsnorm_kernel(Args a) {
  __shared__ float yslots[kThreads / L2C_WAVE], hslots[kThreads / L2C_WAVE];
  const size_t row = static_cast<size_t>(blockIdx.x) * a.size;
  const float *gate = a.gate ? a.gate + static_cast<size_t>(blockIdx.x / a.rows_per_gate) * a.size : nullptr;
  const int t = threadIdx.x;
  float yscale = 1.0f;
  if (a.block_weight) {
    float ss = 0.0f;
    for (int j = t; j < a.size; j += kThreads) {
      const float y = load<YBF>(a.block, row + j);
      ss = fmaf(y, y, ss);
    }
    yscale = 1.0f / sqrtf(l2c::block_sum(ss, yslots) / static_cast<float>(a.size) + a.eps);
  }
  auto sum = [&](int j) __attribute__((always_inline)) {
    float z = load<YBF>(a.block, row + j);
    if (a.block_weight) z = z * yscale * a.block_weight[j];
    if (gate) z *= gate[j];
    return fmaf(a.residual_scale, load<XBF>(a.residual, row + j), z);
  };
  float ss = 0.0f;
  for (int j = t; j < a.size; j += kThreads) {
    const float h = sum(j);
    ss = fmaf(h, h, ss);
  }
  const float scale = 1.0f / sqrtf(l2c::block_sum(ss, hslots) / static_cast<float>(a.size) + a.eps);
  // A lane writes only what it alone has read, after reading it: outputs may be inputs.
  for (int j = t; j < a.size; j += kThreads) {
    const float h = sum(j), n = h * scale * a.weight[j];
    if (a.residual_out) store<XBF>(a.residual_out, row + j, h);
    store<NBF>(a.normalized, row + j, n);
  }
}

using Kernel = void (*)(Args);

template <bool XBF, bool YBF>
Kernel kernel_for(bool n) {
  return n ? residual_rmsnorm_kernel<XBF, YBF, true> : residual_rmsnorm_kernel<XBF, YBF, false>;
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
  if (!l2c::launchable(batch, kThreads)) return hipErrorInvalidValue;
  const Args a = {normalized, residual_out, residual, block, block_weight, gate, weight,
                  size, rows_per_gate, residual_scale, eps};
  const bool x = residual_type == L2C_BF16, y = block_type == L2C_BF16, n = normalized_type == L2C_BF16;
  const Kernel fn = x ? (y ? kernel_for<true, true>(n) : kernel_for<true, false>(n))
                      : (y ? kernel_for<false, true>(n) : kernel_for<false, false>(n));
  hipLaunchKernelGGL(fn, dim3(batch), dim3(kThreads), 0, stream, a);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

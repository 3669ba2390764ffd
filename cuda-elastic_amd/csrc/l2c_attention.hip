// Attention of new tokens over a cache in pages (include/l2c.h has the formula).
#include <type_traits>

#include "l2c_cache.h"

namespace {

using l2c::Sequences;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Attention {
  uint16_t *out;
  const uint16_t *q;
  const void *keys, *values;
  const float *key_scales, *value_scales;
  long long out_stride, q_stride;
  Sequences s;
  int heads, kv_heads, width, window;
  float scale;
};

// Eight cached values as fp32, without their row's scale.
template <bool E4M3>
__device__ __forceinline__ void load8(float (&v)[8], const void *cache, size_t at) {
  if constexpr (E4M3) {
    const u32x2 q = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(cache) + at);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bf16x2 low = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], 1.0f, false);
      const bf16x2 high = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], 1.0f, true);
      v[4 * i] = static_cast<float>(low[0]), v[4 * i + 1] = static_cast<float>(low[1]);
      v[4 * i + 2] = static_cast<float>(high[0]), v[4 * i + 3] = static_cast<float>(high[1]);
    }
  } else {
    const u32x4 q = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(cache) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
    }
  }
}

// A wave a row and head: 64 positions at a time, a lane's score each; then the lanes have
// values' columns, and go through the positions.
template <bool E4M3>
__global__ __launch_bounds__(L2C_WAVE) void attention_kernel(Attention a) {
  __shared__ float q[L2C_MAX_HEAD];
  const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  int sequence, position;
  if (!a.s.find(row, sequence, position)) return;
  const int kv = head / (a.heads / a.kv_heads);
  for (int i = lane; i < a.width; i += L2C_WAVE)
    q[i] = __uint_as_float(
        static_cast<unsigned>(a.q[row * a.q_stride + static_cast<size_t>(head) * a.width + i]) << 16);
  __syncthreads();
  const int end = min(position, a.s.capacity() - 1);
  float top = -INFINITY, total = 0.0f, acc[L2C_MAX_HEAD / L2C_WAVE] = {};
  const int begin = a.window ? max(0, position - a.window + 1) : 0;
  for (int first = begin; first <= end; first += L2C_WAVE) {
    const int j = first + lane;
    float score = -INFINITY;
    size_t at = 0;
    bool there = false;
    if (j <= end) {
      const int index = a.s.by_page(j), page = a.s.page(sequence, index);
      if (a.s.is_page(page)) {
        there = true;
        at = (static_cast<size_t>(page) * a.kv_heads + kv) * a.s.page_size + (j - index * a.s.page_size);
        float dot = 0.0f;
        for (int i = 0; i < a.width; i += 8) {
          float k[8];
          load8<E4M3>(k, a.keys, at * a.width + i);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = fmaf(q[i + e], k[e], dot);
        }
        if (E4M3) dot *= a.key_scales[at];
        score = dot * a.scale;
      }
    }
    const float most = fmaxf(top, l2c::wave_max(score));
    const float shift = most == -INFINITY ? 0.0f : most;
    const float p = !there ? 0.0f : expf(score - shift), again = expf(top - shift);
    total = total * again + l2c::wave_sum(p);
    top = most;
#pragma unroll
    for (int c = 0; c < L2C_MAX_HEAD / L2C_WAVE; ++c) acc[c] *= again;
    for (int i = 0; i < L2C_WAVE && first + i <= end; ++i) {
      if (!__shfl(static_cast<int>(there), i, L2C_WAVE)) continue;
      float w = __shfl(p, i, L2C_WAVE);
      const size_t from = (static_cast<size_t>(static_cast<unsigned>(__shfl(static_cast<int>(at >> 32), i, L2C_WAVE))) << 32) |
                          static_cast<unsigned>(__shfl(static_cast<int>(at), i, L2C_WAVE));
      if (E4M3) w *= a.value_scales[from];
#pragma unroll
      for (int c = 0; c < L2C_MAX_HEAD / L2C_WAVE; ++c) {
        const int d = c * L2C_WAVE + lane;
        if (d >= a.width) continue;
        float v;
        if constexpr (E4M3)
          v = static_cast<float>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
              static_cast<const uint8_t *>(a.values)[from * a.width + d], 1.0f, false)[0]);
        else
          v = __uint_as_float(static_cast<unsigned>(static_cast<const uint16_t *>(a.values)[from * a.width + d]) << 16);
        acc[c] = fmaf(w, v, acc[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < L2C_MAX_HEAD / L2C_WAVE; ++c) {
    const int d = c * L2C_WAVE + lane;
    if (d >= a.width) continue;
    const f32x2 o = {total == 0.0f ? 0.0f : acc[c] / total, 0.0f};
    a.out[row * a.out_stride + static_cast<size_t>(head) * a.width + d] =
        __builtin_bit_cast(unsigned, __builtin_convertvector(o, bf16x2)) & 0xffffu;
  }
}

}  // namespace

extern "C" size_t l2c_cache_attention_workspace_bytes(int, int, int, int, int, int, int) { return 0; }

extern "C" int l2c_cache_attention(uint16_t *out, long long out_stride, const uint16_t *q, long long q_stride,
                                   const void *keys, const void *values, const float *key_scales,
                                   const float *value_scales, int cache_type, const int *tables, const int *lengths,
                                   const int *starts, int sequences, int rows, int heads, int kv_heads, int width,
                                   int page_size, int pages, int max_pages, int window, float scale, void *workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  if (!l2c::cache_sizes(cache_type, sequences, rows, kv_heads, width, page_size, pages, max_pages) || heads <= 0 ||
      heads > 65535 || heads % kv_heads != 0 || window < 0)
    return hipErrorInvalidValue;
  const long long row = static_cast<long long>(heads) * width;
  if (q_stride < row || out_stride < row || q_stride % 8 != 0 || out_stride % 8 != 0) return hipErrorInvalidValue;
  if (sequences == 0 || rows == 0) return hipSuccess;
  if (!l2c::cache_arguments(cache_type, keys, values, key_scales, value_scales, tables, lengths, starts, sequences,
                            rows) ||
      !q || !out || !l2c_aligned16(q) || !l2c_aligned16(out) ||
      workspace_bytes < l2c_cache_attention_workspace_bytes(sequences, rows, heads, kv_heads, width, page_size, max_pages))
    return hipErrorInvalidValue;
  if (!l2c::launchable(static_cast<long long>(rows) * heads, L2C_WAVE)) return hipErrorInvalidValue;
  const Attention a = {out, q, keys, values, key_scales, value_scales, out_stride, q_stride,
                       l2c::sequences_of(tables, lengths, starts, sequences, rows, max_pages, page_size, pages),
                       heads, kv_heads, width, window, scale};
  auto fn = cache_type == L2C_BF16 ? attention_kernel<false> : attention_kernel<true>;
  hipLaunchKernelGGL(fn, dim3(rows, heads), dim3(L2C_WAVE), 0, stream, a);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

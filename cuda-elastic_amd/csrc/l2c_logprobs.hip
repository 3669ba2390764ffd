// Log probabilities of given tokens, the rows' entropies and their largest logits
// (include/l2c.h has the formulas).
#include <climits>

#include "l2c_common.h"
#include "../../include/l2c.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / L2C_WAVE;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, L2C_WAVE);
  return v;
}

// A workgroup a row: the maximum, the sums, and the alternatives one after the other.
__global__ __launch_bounds__(kThreads) void logprobs_kernel(float *logprobs, float *entropies, int *top_tokens,
                                                            float *top_logprobs, const float *logits, const int *tokens,
                                                            int vocab, int top) {
  __shared__ float maxima[kWaves];
  __shared__ int bad[kWaves], places[kWaves];
  __shared__ double sums[kWaves], products[kWaves];
  const int row = blockIdx.x, t = threadIdx.x, lane = t % L2C_WAVE, wave = t / L2C_WAVE;
  const float *const x = logits + static_cast<size_t>(row) * vocab;
  float m = -INFINITY;
  bool wrong = false;
  for (long long i = t; i < vocab; i += kThreads) {
    wrong |= !(x[i] < INFINITY);
    m = fmaxf(m, x[i]);
  }
  m = l2c::wave_max(m);
  wrong = __ballot(wrong) != 0;
  if (lane == 0) maxima[wave] = m, bad[wave] = wrong;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, maxima[w]), wrong |= bad[w] != 0;
  wrong |= m == -INFINITY;
  double sum = 0.0, product = 0.0;
  if (!wrong)
    for (long long i = t; i < vocab; i += kThreads) {
      if (x[i] == -INFINITY) continue;
      const double away = static_cast<double>(x[i]) - m;
      const double e = expf(static_cast<float>(away));
      sum += e;
      product += e * away;
    }
  sum = wave_sum(sum), product = wave_sum(product);
  if (lane == 0) sums[wave] = sum, products[wave] = product;
  __syncthreads();
  sum = product = 0.0;
  for (int w = 0; w < kWaves; ++w) sum += sums[w], product += products[w];
  const double z = log(sum);
  const float nan = __uint_as_float(0x7fc00000u);
  if (t == 0) {
    if (logprobs) {
      const int token = tokens[row];
      logprobs[row] = wrong || token < 0 || token >= vocab ? nan : static_cast<float>(static_cast<double>(x[token]) - m - z);
    }
    if (entropies) entropies[row] = wrong ? nan : static_cast<float>(z - product / sum);
  }
  float before = INFINITY;  // the alternative found last
  int at = -1;
  for (int k = 0; k < top; ++k) {
    float best = -INFINITY;
    int place = INT_MAX;
    if (!wrong)
      for (long long i = t; i < vocab; i += kThreads)
        if ((x[i] < before || (x[i] == before && i > at)) && x[i] > best) best = x[i], place = static_cast<int>(i);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float v = __shfl_xor(best, o, L2C_WAVE);
      const int p = __shfl_xor(place, o, L2C_WAVE);
      if (v > best || (v == best && p < place)) best = v, place = p;
    }
    __syncthreads();
    if (lane == 0) maxima[wave] = best, places[wave] = place;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
      if (maxima[w] > best || (maxima[w] == best && places[w] < place)) best = maxima[w], place = places[w];
    before = best, at = place;
    if (t == 0) {
      const bool none = place == INT_MAX;
      top_tokens[static_cast<size_t>(row) * top + k] = none ? -1 : place;
      top_logprobs[static_cast<size_t>(row) * top + k] =
          wrong ? nan : none ? -INFINITY : static_cast<float>(static_cast<double>(best) - m - z);
    }
  }
}

}  // namespace

extern "C" size_t l2c_decoder_logprobs_workspace_bytes(int, int, int) { return 0; }

extern "C" int l2c_decoder_logprobs(float *logprobs, float *entropies, int *top_tokens, float *top_logprobs,
                                    const float *logits, const int *tokens, int vocab, int top, int rows,
                                    void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (vocab <= 0 || top < 0 || top > L2C_MAX_ALTERNATIVES || rows < 0 || !logprobs != !tokens)
    return hipErrorInvalidValue;
  if (rows == 0) return hipSuccess;
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & 3u) != 0 || (top > 0 && (!top_tokens || !top_logprobs)) ||
      workspace_bytes < l2c_decoder_logprobs_workspace_bytes(vocab, top, rows) || !l2c::launchable(rows, kThreads))
    return hipErrorInvalidValue;
  hipLaunchKernelGGL(logprobs_kernel, dim3(rows), dim3(kThreads), 0, stream, logprobs, entropies, top_tokens,
                     top_logprobs, logits, tokens, vocab, top);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

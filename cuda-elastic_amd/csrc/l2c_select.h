// Selection of the largest of many numbers by their keys: reductions and scans over a wave
// without LDS, bounds by ballots, ranks by comparison. Shared by l2c_beam.hip and
// l2c_logprobs.hip.
#pragma once

#include <climits>

#include "l2c_common.h"

namespace l2c {

typedef unsigned long long u64;

// Unsigned keys in the order of the numbers; 0 is below every number's key and NaN's.
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned u = __float_as_uint(v + 0.0f);  // -0 counts as 0
  return v == v ? ((u & 0x80000000u) ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float number_of(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ u64 key_of(double v) {
  const u64 u = __double_as_longlong(v + 0.0);
  return v == v ? ((u >> 63) ? ~u : u | (1ULL << 63)) : 0ULL;
}
__device__ __forceinline__ double number_of(u64 key) {
  return __longlong_as_double((key >> 63) ? key & ~(1ULL << 63) : ~key);
}

// exp(t) for t <= 0: the hardware's exp2 of t log2(e) rounded, times 1 + ln(2) times what
// the rounding left, to about 1.2 ulp; NaN stays NaN, results below 2^-126 may be 0.
__device__ __forceinline__ float exp_nonpositive(float t) {
  constexpr float kLog2e = 1.44269504088896340736f;
  constexpr float kLog2eLow = 1.925963033500011e-08f;  // log2(e) - kLog2e
  constexpr float kLn2 = 0.693147180559945309417f;
  t = t < -150.0f ? -150.0f : t;
  const float high = t * kLog2e;
  const float low = fmaf(t, kLog2eLow, fmaf(t, kLog2e, -high));
  const float e = __builtin_amdgcn_exp2f(high);
  return fmaf(e, low * kLn2, e);
}

// Values of other lanes through the adders' operand paths (DPP), which take a tenth of a
// trip through LDS: from 1, 2, 4 or 8 lanes before in rows of 16, from the row before's
// last lane, from the lower half's last lane; or rotated in rows of 16.
enum Dpp { kBefore1 = 0x111, kBefore2 = 0x112, kBefore4 = 0x114, kBefore8 = 0x118, kRowBefore = 0x142,
           kHalfBefore = 0x143, kRotate1 = 0x121, kRotate2 = 0x122, kRotate4 = 0x124, kRotate8 = 0x128 };

// `none` where there is no such lane.
template <int FROM>
__device__ __forceinline__ int other(int v, int none = 0) {
  constexpr int kRows = FROM == kRowBefore ? 0xa : FROM == kHalfBefore ? 0xc : 0xf;
  return __builtin_amdgcn_update_dpp(none, v, FROM, kRows, 0xf, false);
}
template <int FROM>
__device__ __forceinline__ float other(float v, float none) {
  return __int_as_float(other<FROM>(__float_as_int(v), __float_as_int(none)));
}
template <int FROM>
__device__ __forceinline__ double other(double v) {  // none: 0
  const long long bits = __double_as_longlong(v);
  const unsigned low = other<FROM>(static_cast<int>(bits)), high = other<FROM>(static_cast<int>(bits >> 32));
  return __longlong_as_double(static_cast<long long>(high) << 32 | low);
}

// The sum of v over this lane and those before it; lane 63 has the wave's.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += other<kBefore1>(v);
  v += other<kBefore2>(v);
  v += other<kBefore4>(v);
  v += other<kBefore8>(v);
  v += other<kRowBefore>(v);
  v += other<kHalfBefore>(v);
  return v;
}
// Lane 63 has the wave's maximum.
__device__ __forceinline__ float wave_top(float v) {
  v = fmaxf(v, other<kBefore1>(v, v));
  v = fmaxf(v, other<kBefore2>(v, v));
  v = fmaxf(v, other<kBefore4>(v, v));
  v = fmaxf(v, other<kBefore8>(v, v));
  v = fmaxf(v, other<kRowBefore>(v, v));
  return fmaxf(v, other<kHalfBefore>(v, v));
}
__device__ __forceinline__ unsigned wave_top(unsigned v) {  // in every lane
  v = max(v, static_cast<unsigned>(other<kBefore1>(static_cast<int>(v))));
  v = max(v, static_cast<unsigned>(other<kBefore2>(static_cast<int>(v))));
  v = max(v, static_cast<unsigned>(other<kBefore4>(static_cast<int>(v))));
  v = max(v, static_cast<unsigned>(other<kBefore8>(static_cast<int>(v))));
  v = max(v, static_cast<unsigned>(other<kRowBefore>(static_cast<int>(v))));
  v = max(v, static_cast<unsigned>(other<kHalfBefore>(static_cast<int>(v))));
  return __builtin_amdgcn_readlane(v, L2C_WAVE - 1);
}
// Every lane has its 16 lanes' maximum, or sum.
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, other<kRotate8>(v, v));
  v = fmaxf(v, other<kRotate4>(v, v));
  v = fmaxf(v, other<kRotate2>(v, v));
  return fmaxf(v, other<kRotate1>(v, v));
}
__device__ __forceinline__ double row_sum(double v) {
  v += other<kRotate8>(v);
  v += other<kRotate4>(v);
  v += other<kRotate2>(v);
  return v + other<kRotate1>(v);
}

// A bound that at least k of the wave's 64 values reach: exactly k of them, or, where the
// k-th largest ties with the next, all that are as large, and the bound is that value. 0 if
// fewer than k are not 0. A bit at a time, to where just k are left: the steps wait for
// each other, but are scalar instructions for the most part, which other waves leave idle
// (starting at the first bit in which the values differ, or two bits a step, measured 20%
// slower for 256 x 4 x 32003).
__device__ __forceinline__ int wave_reach(unsigned v, unsigned bound) { return __popcll(__ballot(v >= bound)); }
__device__ __forceinline__ unsigned wave_bound(unsigned v, int k) {
  unsigned bound = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned next = bound | 1u << bit;
    const int reach = wave_reach(v, next);
    if (reach >= k) bound = next;
    if (reach == k) break;
  }
  return bound;
}
// The same where one wave's time counts, because nothing else runs: a maximum at a time, and for
// larger k two bits a step, whose ballots do not wait for each other.
__device__ __forceinline__ unsigned lone_wave_bound(unsigned v, int k) {
  if (wave_reach(v, 1) < k) return 0;
  unsigned bound = 0;
  if (k <= 8) {
    for (int reached = 0; reached < k;) {
      bound = wave_top(v);
      const u64 lanes = __ballot(v == bound);
      reached += __popcll(lanes);
      v = v == bound ? 0u : v;
    }
    return bound;
  }
  for (int bit = 30; bit >= 0; bit -= 2) {
    const unsigned one = bound | 1u << bit, two = bound | 2u << bit, three = one | two;
    const int reach1 = wave_reach(v, one), reach2 = wave_reach(v, two), reach3 = wave_reach(v, three);
    bound = reach3 >= k ? three : reach2 >= k ? two : reach1 >= k ? one : bound;
    if (reach3 == k || reach2 == k || reach1 == k) break;
  }
  return bound;
}

// How many of n values (16-byte aligned) are larger, and how many equal. Reads in eights, up to
// seven past the end: one after the other they would wait for LDS each time.
struct Order {
  int larger, equal;
};
__device__ __forceinline__ Order order(const unsigned *values, int n, unsigned than) {
  Order count = {0, 0};
  auto eight = [&](int o, int inside) __attribute__((always_inline)) {
    const uint4 a = *reinterpret_cast<const uint4 *>(values + o), b = *reinterpret_cast<const uint4 *>(values + o + 4);
    const unsigned v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      count.larger += u < inside && v[u] > than;
      count.equal += u < inside && v[u] == than;
    }
  };
  int o = 0;
  for (; o + 8 <= n; o += 8) eight(o, 8);
  if (o < n) eight(o, n - o);
  return count;
}
// How many of n entries have the key and come before `before` (a larger number).
__device__ __forceinline__ int earlier(const unsigned *keys, const unsigned *befores, int n, unsigned key,
                                       unsigned before) {
  int count = 0;
#pragma unroll 8
  for (int o = 0; o < n; ++o) count += static_cast<int>(keys[o] == key) & static_cast<int>(befores[o] > before);
  return count;
}

}  // namespace l2c

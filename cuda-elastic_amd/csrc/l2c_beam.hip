// Beam search for the batched decoder: the choice of a request's next beams among
// beams x vocabulary, and the states that follow the chosen beams' parents.
//
// Selection, for each request, with scores s_k of its beams and their logits x_k:
//   s_k + x_k[v] - log sum_u exp(x_k[u])
// over all beams k and tokens v; the `beams` largest are the next beams. Two kernels:
//
//  * beam_chunks_kernel, a workgroup per chunk of a row of logits: one pass over the
//    data, 1024 V logits at a time, which the lanes hold in registers. It leaves the
//    chunk's maximum, its sum of exponentials and its `beams` largest logits in order.
//    Nothing is sorted: each of the four waves finds the K/4-th largest of its lanes' maxima,
//    bit by bit, by ballots (for K <= 4 its maximum); the least of the four is a bound that at
//    least K values reach, and few more do. Those go to a list in LDS, where each finds its
//    rank by comparison with the others. So that the list has a length, a wave of which more
//    than K lanes reach the bound goes by the K-th largest of its own.
//  * beam_join_kernel, a workgroup per request: the rows' sums, and the same choice
//    among the chunks' lists by their 64-bit scores. The lists are found by their firsts.
//
// The order is total: larger first, then the lower beam, its larger logit, the lower
// token. Results do not depend on the order of the list's atomics. Sums of exponentials are
// fp32 within a lane and 64-bit across lanes, scores 64-bit until they are stored: beams'
// scores lie close together, and a rounding there would change which tokens are chosen.
#include <climits>

#include "l2c_common.h"
#include "../../include/l2c.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / L2C_WAVE;
constexpr int kMaxBeams = L2C_MAX_BEAMS;

typedef unsigned long long u64;

// The workspace: what every chunk of every row leaves, [row][chunk]; then the candidates,
// [request][rank][beam][chunk]: the join's lanes read the chunks' best side by side.
struct ChunkStat {
  double sum;  // of exp(x - maximum); NaN if the chunk holds a NaN or +Inf
  float maximum;
  int unused;
};
struct Candidate {
  float logit;
  int token;  // -1: none
};

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
// The same for the 64-bit values from `first` on themselves, 64 for the workgroup's four waves:
// lane l of wave l / 16 gets those of value first + l. The lanes hold the values that a
// wave's sixteen are compared with, one ballot for 64 comparisons: the chain of a lane that
// goes through them by itself is four to five times as long. (Where many workgroups share the
// CUs, as the chunks' do, it costs more than it saves.)
__device__ __forceinline__ Order order_of_64(const u64 *values, int n, int first) {
  constexpr int kEach = L2C_WAVE / kWaves;
  const int lane = threadIdx.x % L2C_WAVE;
  const int from = kEach * __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  Order count = {0, 0};
  if (first + from >= n) return count;
  const u64 mine = first + lane < n ? values[first + lane] : 0ULL;
  for (int o = 0; o < n; o += L2C_WAVE) {
    const u64 v = o == first ? mine : o + lane < n ? values[o + lane] : 0ULL;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const unsigned low = __builtin_amdgcn_readlane(static_cast<unsigned>(mine), from + u);
      const unsigned high = __builtin_amdgcn_readlane(static_cast<unsigned>(mine >> 32), from + u);
      const u64 than = static_cast<u64>(high) << 32 | low;
      const int larger = __popcll(__ballot(v > than)), equal = __popcll(__ballot(v == than));
      count.larger += lane == from + u ? larger : 0;
      count.equal += lane == from + u ? equal : 0;
    }
  }
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

// V float4 a lane. A row is `chunks` chunks of `parts` parts of kThreads * 4 V logits (the
// last ones shorter); MANY: of more than one part. Of 64 registers eight waves fit a SIMD (100 x
// 10 x 10000 20.2 us, 21.0 with 68 and seven).
template <int V, bool MANY>
__global__ __launch_bounds__(kThreads, MANY ? 1 : 8) void beam_chunks_kernel(unsigned char *__restrict__ workspace,
                                                               const float *__restrict__ logits,
                                                               const float *__restrict__ scores,
                                                               const int *__restrict__ tokens, int eos, int vocab,
                                                               int beams, int chunks, int parts) {
  constexpr int kPart = kThreads * 4 * V;
  // Keys and UINT_MAX - place of the list: `beams` lanes' values of each wave at most, and what
  // order() may read.
  extern __shared__ uint4 lists[];
  unsigned *const list_key = reinterpret_cast<unsigned *>(lists);
  unsigned *const list_before = list_key + kWaves * 4 * V * beams + 8;
  __shared__ __attribute__((aligned(16))) unsigned kept_key[2][kMaxBeams + 8];  // the largest so far, in order
  __shared__ unsigned kept_before[2][kMaxBeams + 8];
  __shared__ unsigned bounds[kWaves];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ int length;
  const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
  const int token = tokens[row];  // both loads before either is waited for
  const float score = scores[row];
  const bool ended = eos >= 0 && token == eos, dead = !(fabsf(score) <= FLT_MAX);
  if (ended | dead) return;  // its logits do not count, or it has no continuations
  const int t = threadIdx.x, lane = t % L2C_WAVE, wave = t / L2C_WAVE;
  const long long size = static_cast<long long>(parts) * kPart;
  const int first = static_cast<int>(chunk * size);  // below vocab: no chunk is empty
  const int whole = static_cast<int>(min(size, static_cast<long long>(vocab - first)));
  const float *const x = logits + static_cast<size_t>(row) * vocab + first;
  auto load = [&](float4 (&q)[V], int start) __attribute__((always_inline)) {
    const int n = min(kPart, whole - start);
#pragma unroll
    for (int c = 0; c < V; ++c) {  // -Inf past the end
      const int j = 4 * (t + c * kThreads);
      const float *const p = x + start + j;
      q[c] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (j + 4 <= n) {
        q[c] = l2c::ld4_any(p);
      } else if (j < n) {
        q[c].x = p[0];
        if (j + 1 < n) q[c].y = p[1];
        if (j + 2 < n) q[c].z = p[2];
      }
    }
  };
  float4 q[V];
  load(q, 0);
  if (t == 0) length = 0;
  double total = 0.0;          // the lane's sum of exp(x - shift)
  float shift = -INFINITY;     // the largest so far
  int count = 0;               // of `kept`
  int turn = 0;
  for (int start = 0;;) {
    const int n = min(kPart, whole - start);
    const bool more = MANY && whole - start > kPart;
    float v[4 * V];
#pragma unroll
    for (int c = 0; c < V; ++c) v[4 * c] = q[c].x, v[4 * c + 1] = q[c].y, v[4 * c + 2] = q[c].z, v[4 * c + 3] = q[c].w;
    if (more) load(q, start + kPart);
    auto place = [&](int i) __attribute__((always_inline)) { return 4 * (t + i / 4 * kThreads) + i % 4; };
    // The lane's largest, -Inf where all are NaN; 0 past the row.
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) top = fmaxf(top, v[i]);
    const unsigned best = place(0) < n ? key_of(top) : 0u;
    const float largest = wave_top(top);  // of the last lane
    // Of the waves whose lanes all have values each has its share of the largest.
    const int sharing = min(kWaves, max(1, n / (4 * L2C_WAVE))), share = (beams + sharing - 1) / sharing;
    const unsigned bound = share == 1 ? key_of(largest) : wave_bound(best, share);
    if (lane == L2C_WAVE - 1) {
      bounds[wave] = bound;
      tops[wave] = largest;
    }
    __syncthreads();
    unsigned least = bounds[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
      if (w < sharing) least = min(least, bounds[w]);
    if (MANY && count == beams) least = max(least, kept_key[turn][beams - 1]);
    least = max(least, key_of(-FLT_MAX));  // -Inf is no candidate: no list has it, however many there are
    float maximum = shift;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) maximum = fmaxf(maximum, tops[w]);
    if (maximum > shift) {  // the lane's sum so far is of exp(x - the old maximum)
      if (MANY && start > 0) total *= exp(static_cast<double>(shift) - static_cast<double>(maximum));
      shift = maximum;
    }
    const float subtract = shift == -INFINITY ? 0.0f : shift;  // nothing but -Inf and NaN: no maximum
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) sum += exp_nonpositive(v[i] - subtract);
    total += static_cast<double>(sum);
    // The values that reach the bound into the list, a wave's after each other's. If more than
    // `beams` of its lanes have such, only those of the `beams` lanes with the largest, and
    // of lanes that tie, with the lowest places of it: no other value can be among the chosen.
    unsigned last = 0;  // of lanes that tie: UINT_MAX - place of the last one's value
    if (wave_reach(best, least) > beams) {
      least = wave_bound(best, beams);
      if (wave_reach(best, least) > beams) {
        const int larger = __popcll(__ballot(best > least));
        const float tie = number_of(least);
        unsigned before = 0;
#pragma unroll
        for (int i = 4 * V - 1; i >= 0; --i)
          if (v[i] == tie) before = UINT_MAX - (static_cast<unsigned>(start) + place(i));
        last = wave_bound(best == least ? before : 0u, beams - larger);
      }
    }
    const float limit = number_of(least);  // NaN does not reach it, nor does what is past the end
    unsigned reach = 0;
    if (last == 0) {
#pragma unroll
      for (int i = 0; i < 4 * V; ++i) reach |= v[i] >= limit ? 1u << i : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 4 * V; ++i)
        if (v[i] > limit || (v[i] == limit && UINT_MAX - (static_cast<unsigned>(start) + place(i)) >= last))
          reach |= 1u << i;
    }
    if (__ballot(reach != 0)) {
      const int count_here = __popc(reach), upto = wave_scan(count_here);
      int base = 0;
      if (lane == L2C_WAVE - 1) base = atomicAdd(&length, upto);
      int to = __builtin_amdgcn_readlane(base, L2C_WAVE - 1) + upto - count_here;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        if (__ballot(reach >> 4 * c & 15u) == 0) continue;
#pragma unroll
        for (int i = 4 * c; i < 4 * c + 4; ++i)
          if (reach >> i & 1) {
            list_key[to] = key_of(v[i]);
            list_before[to++] = UINT_MAX - (static_cast<unsigned>(start) + place(i));
          }
      }
    }
    __syncthreads();
    const int m = __builtin_amdgcn_readfirstlane(length), all = count + m;
    for (int e = t; e < all; e += kThreads) {
      const bool old = MANY && e < count;
      const unsigned mine = old ? kept_key[turn][e] : list_key[e - count];
      const unsigned before = old ? kept_before[turn][e] : list_before[e - count];
      Order among = order(list_key, m, mine);
      if (MANY) {
        const Order among_kept = order(kept_key[turn], count, mine);
        among.larger += among_kept.larger, among.equal += among_kept.equal;
      }
      if (among.equal > 1) {  // it and others
        among.larger += earlier(list_key, list_before, m, mine, before);
        if (MANY) among.larger += earlier(kept_key[turn], kept_before[turn], count, mine, before);
      }
      if (among.larger < beams) kept_key[turn ^ 1][among.larger] = mine, kept_before[turn ^ 1][among.larger] = before;
    }
    count = min(all, beams);
    turn ^= 1;
    __syncthreads();
    if (!more) break;
    if (t == 0) length = 0;  // before the next barrier, after which it is counted again
    start += kPart;
  }
  ChunkStat *const stats = reinterpret_cast<ChunkStat *>(workspace);
  if (t < beams) {
    const int request = row / beams;
    const size_t place = (static_cast<size_t>(request) * beams + t) * beams + (row - request * beams);
    Candidate *const out = reinterpret_cast<Candidate *>(stats + gridDim.x) + place * chunks + chunk;
    *out = {-INFINITY, -1};
    if (t < count) *out = {number_of(kept_key[turn][t]), first + static_cast<int>(UINT_MAX - kept_before[turn][t])};
  }
  total = wave_scan(total);
  if (lane == L2C_WAVE - 1) sums[wave] = total;
  __syncthreads();
  if (t == 0) {
    total = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) total += sums[w];
    stats[blockIdx.x] = {total, shift, 0};  // [row][chunk]
  }
}

// Quotients of values below 2^16 by one of 1 to 2^16, without a division each.
struct Quotient {
  unsigned by;
  __device__ explicit Quotient(int divisor) : by(divisor > 1 ? UINT_MAX / divisor + 1 : 0) {}
  __device__ __forceinline__ int operator()(int v) const { return by ? __umulhi(v, by) : v; }
};

constexpr int kJoinLists = 4 * kThreads;  // at most
constexpr int kChosenCandidates = kMaxBeams * (kMaxBeams + 1) / 2;

// DIRECT: the lanes hold all candidates, one each. Else they hold the lists' firsts, HELD
// each. The `beams` lists with the largest firsts have all that can be chosen, of the one
// in place p (from 0) the first beams - p, and these follow from memory.
template <int HELD, bool DIRECT>
__global__ __launch_bounds__(kThreads) void beam_join_kernel(float *scores_out, int *tokens_out, int *parents,
                                                             int *generated, const unsigned char *workspace,
                                                             const float *scores, const int *tokens, int eos,
                                                             int beams, int chunks, int steps, int step) {
  constexpr int kEntries = DIRECT || HELD * kThreads > kChosenCandidates ? HELD * kThreads : kChosenCandidates;
  // A beam's scores are base + (logit - top), in this order: logits of the lowest value
  // would take the rest of the sum with them. NaN: no candidates.
  __shared__ double base[kMaxBeams];
  __shared__ float tops[kMaxBeams];
  __shared__ bool ended[kMaxBeams];
  __shared__ u64 list_key[kEntries], list_logit[kEntries];
  __shared__ int list_at[kEntries];
  __shared__ int chosen[kMaxBeams];
  __shared__ unsigned slots[kWaves];
  __shared__ u64 last_first;
  __shared__ int lengths[2];
  constexpr int kGroup = 16;  // lanes a beam for its chunks' sums
  const int t = threadIdx.x, lane = t % L2C_WAVE, wave = t / L2C_WAVE;
  const int first = blockIdx.x * beams;
  const ChunkStat *const stats = reinterpret_cast<const ChunkStat *>(workspace);
  auto stat = [&](int beam, int chunk) __attribute__((always_inline)) {
    return stats + static_cast<size_t>(first + beam) * chunks + chunk;
  };
  // Candidate i: rank i / lists of list i % lists, a list a chunk, beam after beam: the first
  // lanes have the lists' firsts, and their maxima are a good bound.
  const int lists = beams * chunks, candidates = lists * beams, entries = DIRECT ? candidates : lists;
  const Quotient by_lists(lists), by_chunks(chunks), by_beams(beams);
  const Candidate *const all = reinterpret_cast<const Candidate *>(stats + static_cast<size_t>(gridDim.x) * lists) +
                               static_cast<size_t>(blockIdx.x) * candidates;
  Candidate held[HELD];
#pragma unroll
  for (int r = 0; r < HELD; ++r) held[r] = all[min(t + r * kThreads, entries - 1)];  // together, without a branch
  if (t < 2) lengths[t] = 0;
  // The sums of beams t / 16 and, of more than 16, t / 16 + 16. What most rows have is loaded together.
  // Of ended and dead rows the workspace holds nothing; what is read there is not used.
  constexpr int kBeams = kThreads / kGroup, kRounds = kMaxBeams / kBeams, kStats = 2;
  const int member = t % kGroup, row = t / kGroup;
  ChunkStat held_stat[kRounds][kStats];
  const float score = scores[first + min(t, beams - 1)];
  const int token = tokens[first + min(t, beams - 1)];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (r * kBeams >= beams) break;
    const int k = min(row + r * kBeams, beams - 1);
#pragma unroll
    for (int u = 0; u < kStats; ++u) held_stat[r][u] = *stat(k, min(member + u * kGroup, chunks - 1));
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (r * kBeams >= beams) break;
    const int k = min(row + r * kBeams, beams - 1);
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < kStats; ++u) m = fmaxf(m, held_stat[r][u].maximum);
    for (int c = member + kStats * kGroup; c < chunks; c += kGroup) m = fmaxf(m, stat(k, c)->maximum);
    m = row_max(m);
    double sum = 0.0;
    auto add = [&](const ChunkStat &s) __attribute__((always_inline)) {
      // A chunk of -Inf has sum 0; NaN stays NaN.
      sum += s.maximum == m ? s.sum
             : s.maximum == -INFINITY ? s.sum * 0.0
                                      : s.sum * exp(static_cast<double>(s.maximum) - static_cast<double>(m));
    };
#pragma unroll
    for (int u = 0; u < kStats; ++u)
      if (member + u * kGroup < chunks) add(held_stat[r][u]);
    for (int c = member + kStats * kGroup; c < chunks; c += kGroup) add(*stat(k, c));
    sum = row_sum(sum);
    if (member == 0) base[k] = sum, tops[k] = m;
  }
  __syncthreads();
  if (t < beams) {
    // Of a row of -Inf the sum is 0 and b +Inf, of one with NaN or +Inf it is NaN.
    const bool end = eos >= 0 && token == eos;
    const double b = end ? static_cast<double>(score) : static_cast<double>(score) - log(base[t]);
    base[t] = b >= -DBL_MAX && b <= DBL_MAX ? b : __longlong_as_double(0x7ff8000000000000LL);
    ended[t] = end;
  }
  __syncthreads();
  // The key of candidate `rank` of `list`, 0 where it is none.
  auto key_at = [&](int list, int rank, Candidate c) __attribute__((always_inline)) -> u64 {
    const int beam = by_chunks(list);
    const bool end = ended[beam];
    const double score = base[beam] + (end ? 0.0 : static_cast<double>(c.logit) - static_cast<double>(tops[beam]));
    const bool is = end ? rank == 0 && list == beam * chunks : c.token >= 0;
    return is ? key_of(score) : 0ULL;
  };
  // Entry `to`. What decides between equal keys: the lower beam and its larger logit, then
  // the lower `at`.
  auto enter = [&](int to, u64 key, int list, Candidate c, int at) __attribute__((always_inline)) {
    const int beam = by_chunks(list);
    list_key[to] = key;
    list_logit[to] = static_cast<u64>(beam) << 32 | (ended[beam] ? 0u : UINT_MAX - key_of(c.logit));
    list_at[to] = at;
  };
  auto token_of = [&](int list, Candidate c) __attribute__((always_inline)) {
    return ended[by_chunks(list)] ? eos : c.token;
  };
  // act(e, rank) for every entry.
  auto rank = [&](int m, auto act) __attribute__((always_inline)) {
    for (int first = 0; first < m; first += L2C_WAVE) {
      const Order among = order_of_64(list_key, m, first);
      const int e = first + lane;
      if (lane / (L2C_WAVE / kWaves) != wave || e >= m) continue;
      int at = among.larger;
      if (among.equal > 1) {  // it and others
        const u64 key = list_key[e], logit = list_logit[e];
        const int last = list_at[e];
#pragma unroll 4
        for (int o = 0; o < m; ++o)
          at += (list_key[o] == key) & ((list_logit[o] < logit) | ((list_logit[o] == logit) & (list_at[o] < last)));
      }
      act(e, at);
    }
  };

  // A bound that at least `beams` entries reach, from the upper halves of the lanes' best keys.
  u64 best = 0, held_key[HELD];
#pragma unroll
  for (int r = 0; r < HELD; ++r) {
    const int i = t + r * kThreads, rank = DIRECT ? by_lists(i) : 0;
    const int list = DIRECT ? i - rank * lists : min(i, lists - 1);
    held_key[r] = i < entries ? key_at(list, rank, held[r]) : 0ULL;
    best = max(best, held_key[r]);
  }
  // Of all four waves, if they have entries, a quarter each; else of the one that has the most.
  // So few that they are ranked together as quickly as some of them need no bound.
  const bool few = entries <= L2C_WAVE, quarters = beams > 8 && entries >= kThreads;
  const unsigned bound =
      few ? 1u : lone_wave_bound(static_cast<unsigned>(best >> 32), quarters ? (beams + 3) / 4 : beams);
  if (lane == 0) slots[wave] = bound;
  __syncthreads();
  unsigned most = slots[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) most = quarters ? min(most, slots[w]) : max(most, slots[w]);
  u64 least = static_cast<u64>(max(most, 1u)) << 32;  // a candidate's key is larger
  unsigned reach = 0;
#pragma unroll
  for (int r = 0; r < HELD; ++r) reach |= held_key[r] >= least ? 1u << r : 0u;
  if (__ballot(reach != 0)) {
    const int count_here = __popc(reach), upto = wave_scan(count_here);
    int from = 0;
    if (lane == L2C_WAVE - 1) from = atomicAdd(&lengths[0], upto);
    int to = __builtin_amdgcn_readlane(from, L2C_WAVE - 1) + upto - count_here;
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
      if (reach >> r & 1) {
        const int i = t + r * kThreads, list = DIRECT ? i - by_lists(i) * lists : i;
        enter(to++, held_key[r], list, held[r], DIRECT ? token_of(list, held[r]) : list);
      }
    }
  }
  __syncthreads();
  int m = __builtin_amdgcn_readfirstlane(lengths[0]);
  if (!DIRECT) {
    rank(m, [&](int e, int at) __attribute__((always_inline)) {
      if (at < beams) chosen[at] = list_at[e];
      if (at == beams - 1) last_first = list_key[e];
    });
    if (m < beams && t == 0) last_first = 1;
    __syncthreads();
    constexpr int kEach = kMaxBeams * kMaxBeams / kThreads;
    const int count = min(m, beams);
    least = last_first;
    Candidate c[kEach];
    int list[kEach], place[kEach];
    // Neighbours in a list go to different waves: each has its share of the largest.
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      if (u * kThreads >= beams * beams) break;
      const int i = lane * kWaves + wave + u * kThreads, which = by_beams(i);
      place[u] = i - which * beams;
      list[u] = which < count && which + place[u] < beams ? chosen[which] : -1;
      c[u] = all[list[u] >= 0 ? place[u] * lists + list[u] : 0];
    }
    u64 key[kEach];
    best = 0;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      if (u * kThreads >= beams * beams) break;
      key[u] = list[u] >= 0 ? key_at(list[u], place[u], c[u]) : 0ULL;
      best = max(best, key[u]);
    }
    if (beams > 8) {
      // Where the lists are hardly more than the beams, the last list's first is a poor bound.
      const unsigned quarter = lone_wave_bound(static_cast<unsigned>(best >> 32), (beams + 3) / 4);
      if (lane == 0) slots[wave] = quarter;
      __syncthreads();
      most = slots[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = min(most, slots[w]);
      least = max(least, static_cast<u64>(most) << 32);
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      if (u * kThreads >= beams * beams) break;
      if (list[u] >= 0 && key[u] >= least)
        enter(atomicAdd(&lengths[1], 1), key[u], list[u], c[u], token_of(list[u], c[u]));
    }
    __syncthreads();
    m = __builtin_amdgcn_readfirstlane(lengths[1]);
  }
  auto write = [&](int rank, u64 key, int parent, int token) __attribute__((always_inline)) {
    const int to = first + rank;
    scores_out[to] = key ? static_cast<float>(number_of(key)) : -INFINITY;
    tokens_out[to] = token;
    parents[to] = parent;
    if (generated) generated[static_cast<size_t>(to) * steps + step] = token;
  };
  rank(m, [&](int e, int at) __attribute__((always_inline)) {
    if (at < beams) write(at, list_key[e], static_cast<int>(list_logit[e] >> 32), list_at[e]);
  });
  for (int e = m + t; e < beams; e += kThreads) write(e, 0, -1, -1);
}

using ChunkKernel = void (*)(unsigned char *, const float *, const float *, const int *, int, int, int, int, int);

struct ChunkConfig {
  ChunkKernel fn;
  int values;         // of a lane
  int chunks, parts;  // chunks a row, parts a chunk
};

// Chunks of several parts: only with 8 float4 a lane, since chunk_config takes fewer only where
// no chunk needs more than one part.
template <int V>
ChunkConfig config(int vocab, int most_chunks) {
  const int parts = (vocab - 1) / (kThreads * 4 * V) + 1;
  if constexpr (V == 8) {
    const int each = (parts - 1) / most_chunks + 1;
    if (each > 1) return {beam_chunks_kernel<V, true>, 4 * V, (parts - 1) / each + 1, each};
  }
  return {beam_chunks_kernel<V, false>, 4 * V, parts, 1};
}

// 2048 logits a chunk as long as that makes at most 2048 chunks, and then 4096 logits: small
// chunks have the least latency (1 x 4 x 32000, chunks and join as they were then: 8.1 us in
// chunks of 2048, 9.3 of 4096, 10.9 of 8192). Else 8192, which cost the least instructions a
// logit (256 x 4 x 32003: 42.6, 35.4, 33.8, and 31.3 since; 8 x 8 x 131072 in 2048 chunks of
// 4096 18.2, in 4096 of 2048 21.8; 500 x 4 x 2048 in one chunk a row 12.0, in chunks for
// 8192 17.1). No more lists a request than the join takes.
ChunkConfig chunk_config(int vocab, int beams, int batch) {
  const int most = kJoinLists / beams;
  const double rows = static_cast<double>(batch) * beams;
  auto fits = [&](int part) {
    const int parts = (vocab - 1) / part + 1;
    return parts == 1 || (parts <= most && rows * parts <= 2048);
  };
  if (fits(2048)) return config<2>(vocab, most);
  if (fits(4096)) return config<4>(vocab, most);
  return config<8>(vocab, most);
}

}  // namespace

extern "C" size_t l2c_decoder_beam_workspace_bytes(int vocab, int beams, int batch) {
  if (vocab <= 0 || beams <= 0 || beams > kMaxBeams || batch <= 0) return 0;
  return static_cast<size_t>(batch) * beams * chunk_config(vocab, beams, batch).chunks *
         (sizeof(ChunkStat) + sizeof(Candidate) * static_cast<size_t>(beams));
}

extern "C" int l2c_decoder_beam_select(float *scores_out, int *tokens_out, int *parents, int *generated,
                                       const float *logits, const float *scores, const int *tokens, int eos, int vocab,
                                       int beams, int batch, int steps, int step, void *workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  if (vocab <= 0 || beams <= 0 || beams > kMaxBeams || batch < 0 || eos >= vocab ||
      (generated && (steps <= 0 || step < 0 || step >= steps)))
    return hipErrorInvalidValue;
  if (batch == 0) return hipSuccess;
  if (!scores_out || !tokens_out || !parents || !logits || !scores || !tokens || !workspace ||
      !l2c_aligned16(workspace) || workspace_bytes < l2c_decoder_beam_workspace_bytes(vocab, beams, batch))
    return hipErrorInvalidValue;
  const ChunkConfig c = chunk_config(vocab, beams, batch);
  const long long grid = static_cast<long long>(batch) * beams * c.chunks;
  if (static_cast<long long>(batch) * beams > INT_MAX || grid > INT_MAX || !l2c::launchable(grid, kThreads))
    return hipErrorInvalidValue;
  unsigned char *w = static_cast<unsigned char *>(workspace);
  const size_t list = 2 * sizeof(unsigned) * (kWaves * static_cast<size_t>(beams) * c.values + 8);
  hipLaunchKernelGGL(c.fn, dim3(static_cast<unsigned>(grid)), dim3(kThreads), list, stream, w, logits, scores, tokens,
                     eos, vocab, beams, c.chunks, c.parts);
  L2C_LAUNCH_CHECK();
  const int lists = beams * c.chunks;
  auto join = beams * lists <= kThreads ? beam_join_kernel<1, true>
              : lists <= kThreads       ? beam_join_kernel<1, false>
                                        : beam_join_kernel<4, false>;
  hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(batch)), dim3(kThreads), 0, stream, scores_out, tokens_out,
                     parents, generated, w, scores, tokens, eos, beams, c.chunks, steps, step);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

// ---------------------------------------------------------------------------
// States that follow their beams.
//
// out[g][b][k] = in[g][b][parents[b][k]], bounded by memory: each row is written and
// each row that is some beam's parent is read once, whatever further beams share it
// comes out of a cache. A piece is cut into columns of 16 bytes, and of one byte for
// what is left of it.
//
// Out of place a workgroup copies 256 columns of one row, and the rows of a request are
// neighbours in the launch, so that those of one parent are read at the same time. In
// place a lane takes a column of all beams, which nobody else touches, and has loaded
// it when it stores the first of it; a beam that is its own parent costs nothing. One
// kernel for both, a lane to a column of all beams, took 181 us out of place where the
// copy takes 117 (8 groups x 8 requests x 8 beams of 786 KB: 5.7 TB/s); in place, 89 us.

namespace {

constexpr int kGridY = 65535;  // groups a launch

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// Where column i of a row lies, and whether it has 16 bytes.
struct Columns {
  unsigned columns, wide, all;
  long long piece_stride;
  __device__ __forceinline__ bool at(unsigned i, long long &offset) const {
    const unsigned piece = i / columns, c = i - piece * columns;
    offset = piece * piece_stride + (c < wide ? 16LL * c : 16LL * wide + (c - wide));
    return c < wide;
  }
};

// blockIdx.y: the group. blockIdx.x: parts of rows, ordered by request, part of the row,
// beam; one a workgroup, or with SHORT rows `rows` whole ones (4096 x 8 of 400 bytes:
// 6 us, 21 with one).
template <bool SHORT>
__global__ __launch_bounds__(kThreads) void beam_copy_kernel(unsigned char *__restrict__ out,
                                                             const unsigned char *__restrict__ in,
                                                             const int *__restrict__ parents, int beams, int batch,
                                                             Columns cols, unsigned rows, unsigned blocks,
                                                             long long group_stride, long long row_stride) {
  const unsigned row = SHORT ? threadIdx.x / cols.all : 0, index = SHORT ? blockIdx.x * rows + row : blockIdx.x;
  const unsigned parts = index / beams, k = index - parts * beams;
  const unsigned request = parts / blocks, part = parts - request * blocks;
  if (SHORT && (row >= rows || request >= static_cast<unsigned>(batch))) return;
  const unsigned i = part * kThreads + threadIdx.x - row * cols.all;
  const int from = parents[static_cast<size_t>(request) * beams + k];
  if (i >= cols.all || from < 0 || from >= beams) return;
  long long at;
  const bool wide = cols.at(i, at);
  at += blockIdx.y * group_stride + static_cast<long long>(request) * beams * row_stride;
  const unsigned char *src = in + at + from * row_stride;
  unsigned char *dst = out + at + k * row_stride;
  if (wide) *reinterpret_cast<u32x4_any *>(dst) = *reinterpret_cast<const u32x4_any *>(src);
  else *dst = *src;
}

// COLUMNS columns of all beams a lane. With SHORT rows a workgroup takes those of `rows`
// requests (4096 x 8 of 400 bytes: 5.6 us, 9 with one; 4096 x 32 of 100 bytes: 16 us, 33).
template <int BEAMS, int COLUMNS, bool SHORT>
__global__ __launch_bounds__(kThreads) void beam_permute_kernel(unsigned char *state, const int *__restrict__ parents,
                                                                int beams, int batch, Columns cols, unsigned rows,
                                                                unsigned blocks, long long group_stride,
                                                                long long row_stride) {
  const unsigned row = SHORT ? threadIdx.x / cols.all : 0;
  const unsigned request = SHORT ? blockIdx.x * rows + row : blockIdx.x / blocks, part = blockIdx.x - request * blocks;
  if (SHORT && (row >= rows || request >= static_cast<unsigned>(batch))) return;
  state += blockIdx.y * group_stride + static_cast<long long>(request) * beams * row_stride;
  int from[BEAMS];  // the row that row k becomes, -1 where it stays
#pragma unroll
  for (int k = 0; k < BEAMS; ++k) {
    const int p = k < beams ? parents[static_cast<size_t>(request) * beams + k] : -1;
    from[k] = p < beams && p != k ? p : -1;
  }
  long long at[COLUMNS];
  bool wide[COLUMNS], in[COLUMNS];
  u32x4_any v[COLUMNS][BEAMS];
#pragma unroll
  for (int u = 0; u < COLUMNS; ++u) {
    const unsigned i = SHORT ? threadIdx.x - row * cols.all : (part * COLUMNS + u) * kThreads + threadIdx.x;
    in[u] = i < cols.all;
    wide[u] = cols.at(i, at[u]);
    if (in[u] && wide[u]) {
#pragma unroll
      for (int k = 0; k < BEAMS; ++k)
        if (from[k] >= 0) v[u][k] = *reinterpret_cast<const u32x4_any *>(state + at[u] + from[k] * row_stride);
    } else if (in[u]) {
#pragma unroll
      for (int k = 0; k < BEAMS; ++k)
        if (from[k] >= 0) v[u][k].x = state[at[u] + from[k] * row_stride];
    }
  }
#pragma unroll
  for (int u = 0; u < COLUMNS; ++u) {
    if (in[u] && wide[u]) {
#pragma unroll
      for (int k = 0; k < BEAMS; ++k)
        if (from[k] >= 0) *reinterpret_cast<u32x4_any *>(state + at[u] + k * row_stride) = v[u][k];
    } else if (in[u]) {
#pragma unroll
      for (int k = 0; k < BEAMS; ++k)
        if (from[k] >= 0) state[at[u] + k * row_stride] = static_cast<unsigned char>(v[u][k].x);
    }
  }
}

}  // namespace

extern "C" int l2c_decoder_beam_reorder(void *out, const void *in, const int *parents, int beams, int batch,
                                        int groups, int pieces, long long group_stride, long long row_stride,
                                        long long piece_stride, long long piece_bytes, hipStream_t stream) {
  if (beams <= 0 || beams > kMaxBeams || batch < 0 || groups < 0 || pieces < 0 || piece_bytes < 0)
    return hipErrorInvalidValue;
  if (batch == 0 || groups == 0 || pieces == 0 || piece_bytes == 0) return hipSuccess;
  if (!out || !in || !parents) return hipErrorInvalidValue;
  // Pieces, rows and groups follow each other without overlap, within 63 bits.
  typedef __int128 wide_t;
  const wide_t row = static_cast<wide_t>(pieces - 1) * piece_stride + piece_bytes;
  const wide_t group = (static_cast<wide_t>(batch) * beams - 1) * row_stride + row;
  const wide_t span = static_cast<wide_t>(groups - 1) * group_stride + group;
  if ((pieces > 1 && piece_stride < piece_bytes) || (static_cast<wide_t>(batch) * beams > 1 && row_stride < row) ||
      (groups > 1 && group_stride < group) || span > LLONG_MAX)
    return hipErrorInvalidValue;
  const uintptr_t o = reinterpret_cast<uintptr_t>(out), s = reinterpret_cast<uintptr_t>(in);
  if (o != s && o < s + static_cast<uintptr_t>(span) && s < o + static_cast<uintptr_t>(span))
    return hipErrorInvalidValue;
  const wide_t columns = piece_bytes / 16 + piece_bytes % 16, all = columns * pieces;
  if (all > INT_MAX) return hipErrorInvalidValue;
  const Columns cols = {static_cast<unsigned>(columns), static_cast<unsigned>(piece_bytes / 16),
                        static_cast<unsigned>(all), piece_stride};
  const bool in_place = o == s, few = all <= kThreads / 2;
  // In place two columns a lane keep more in flight; from 16 beams on one is enough, 98 us
  // against 102 for 16 beams of 8 x 4 requests with 786 KB a beam.
  const long long lanes = static_cast<long long>(kThreads) * (in_place && beams <= 8 && !few ? 2 : 1);
  const unsigned blocks = static_cast<unsigned>((static_cast<long long>(all) + lanes - 1) / lanes);
  const unsigned rows = few ? kThreads / static_cast<unsigned>(all) : 1;
  const wide_t parts = static_cast<wide_t>(blocks) * batch * (in_place ? 1 : beams), grid = (parts + rows - 1) / rows;
  if (parts > INT_MAX || !l2c::launchable(static_cast<long long>(grid), kThreads)) return hipErrorInvalidValue;
  auto permute = beams <= 4    ? few ? beam_permute_kernel<4, 1, true> : beam_permute_kernel<4, 2, false>
                 : beams <= 8  ? few ? beam_permute_kernel<8, 1, true> : beam_permute_kernel<8, 2, false>
                 : beams <= 16 ? few ? beam_permute_kernel<16, 1, true> : beam_permute_kernel<16, 1, false>
                 : few         ? beam_permute_kernel<32, 1, true>
                               : beam_permute_kernel<32, 1, false>;
  auto copy = few ? beam_copy_kernel<true> : beam_copy_kernel<false>;
  for (int first = 0; first < groups; first += kGridY) {
    const dim3 size(static_cast<unsigned>(grid), groups - first < kGridY ? groups - first : kGridY);
    unsigned char *to = static_cast<unsigned char *>(out) + first * group_stride;
    const unsigned char *of = static_cast<const unsigned char *>(in) + first * group_stride;
    if (in_place)
      hipLaunchKernelGGL(permute, size, dim3(kThreads), 0, stream, to, parents, beams, batch, cols, rows, blocks,
                         group_stride, row_stride);
    else
      hipLaunchKernelGGL(copy, size, dim3(kThreads), 0, stream, to, of, parents, beams, batch, cols, rows, blocks,
                         group_stride, row_stride);
    L2C_LAUNCH_CHECK();
    if (groups - first <= kGridY) break;
  }
  return hipSuccess;
}

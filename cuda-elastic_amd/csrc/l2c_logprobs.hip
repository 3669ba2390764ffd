// Log probabilities of given tokens, the rows' entropies and their largest logits, from one pass over
// the logits x: with a maximum m so far, Z = sum exp(x - m) and T = sum exp(x - m) (x - m),
//   log p(v) = x_v - m - log Z,   H = log Z - T / Z,
// and a larger maximum m' = m + d makes Z to Z e^-d and T to (T - d Z) e^-d.
//
// Bound by HBM. A workgroup goes through a row, or a chunk of one where there are few rows,
// 1024 V logits at a time in registers, with the next ones on their way. A wave has its own maximum, so
// that its sums wait for nobody; the largest logits so far lie in LDS, in order, and the least of them is
// a bound that most parts have nothing above. Where there is none yet, the bound comes from the lanes'
// maxima by ballots, as in the beam selection. Chunks leave their sums and their lists, which a second
// kernel joins. 2048 rows of 32003 take 51 us without alternatives (5.2 TB/s), 67 to 70 with 20; one of 32000
// in 16 chunks 6.2 and the join 3.6, where every step waits for the one before.
#include "l2c_select.h"
#include "../../include/l2c.h"

namespace {

using namespace l2c;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / L2C_WAVE;
constexpr int kMost = L2C_MAX_ALTERNATIVES;
constexpr int kMaxChunks = L2C_WAVE;  // a row: a lane of the join each

// The workspace: what every chunk of every row leaves, [row][chunk], then the alternatives, [row][chunk][rank].
struct Sums {
  double z, t;  // NaN if the chunk holds a NaN or a +Inf
  float m;
  int unused;
};
struct Candidate {
  float logit;
  int token;  // -1: none
};

struct Args {
  float *logprobs, *entropies;
  int *top_tokens;
  float *top_logprobs;
  const float *logits;
  const int *tokens;
  unsigned char *workspace;
  int vocab, top, chunks, chunk;  // logits a chunk
};

__device__ __forceinline__ float nan_value() { return __uint_as_float(0x7fc00000u); }

// exp(from - to), the factor of sums whose maximum rises; of sums of nothing 0.
__device__ __forceinline__ double lowered(float from, float to) {
  return from == -INFINITY ? 0.0 : exp(static_cast<double>(from) - static_cast<double>(to));
}
__device__ __forceinline__ void raise(double &z, double &t, float &m, float to) {
  if (m == to) return;
  const double by = lowered(m, to), d = m == -INFINITY ? 0.0 : static_cast<double>(to) - static_cast<double>(m);
  t = (t - d * z) * by;
  if (m == -INFINITY) t = z * 0.0;  // NaN stays NaN
  z = m == -INFINITY ? z * 0.0 : z * by;
  m = to;
}

// What a row's sums give; `wrong`: the row has no log probabilities.
struct Row {
  double z, t, log_z;
  float m;
  bool wrong;
  __device__ __forceinline__ Row(double z_, double t_, float m_) : z(z_), t(t_), m(m_) {
    wrong = !(z > 0.0 && z <= DBL_MAX);  // nothing but -Inf, or a NaN or a +Inf
    log_z = log(z);
  }
  __device__ __forceinline__ float logprob(float x) const {
    return wrong ? nan_value() : static_cast<float>(static_cast<double>(x) - static_cast<double>(m) - log_z);
  }
  __device__ __forceinline__ void store(const Args &a, int row, float x, bool inside) const {
    if (a.logprobs) a.logprobs[row] = inside ? logprob(x) : nan_value();
    if (a.entropies) a.entropies[row] = wrong ? nan_value() : static_cast<float>(log_z - t / z);
  }
  __device__ __forceinline__ void alternative(const Args &a, int row, int rank, float x, int token) const {
    const size_t to = static_cast<size_t>(row) * a.top + rank;
    a.top_tokens[to] = wrong ? -1 : token;
    a.top_logprobs[to] = wrong ? nan_value() : token < 0 ? -INFINITY : logprob(x);
  }
};

// V float4 a lane. WHOLE: a chunk is a row, and the results are stored.
template <int V, bool WHOLE>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  constexpr int kPart = kThreads * 4 * V;
  // Keys and UINT_MAX - place of the list: of two parts `top` lanes' values of each wave at most, and
  // what order() may read.
  extern __shared__ uint4 lists[];
  unsigned *const list_key = reinterpret_cast<unsigned *>(lists);
  const int unit = kWaves * 4 * V * a.top;  // values that one part can add
  unsigned *const list_before = list_key + 2 * unit + 8;
  __shared__ __attribute__((aligned(16))) unsigned kept_key[2][kMost + 8];  // the largest so far, in order
  __shared__ unsigned kept_before[2][kMost + 8];
  __shared__ unsigned bounds[kWaves];
  __shared__ int lengths[3];  // of this part, the next and the last: set to 0 by turns
  __shared__ float tops[kWaves];
  __shared__ double zs[kWaves], ts[kWaves];
  const int row = WHOLE ? blockIdx.x : blockIdx.x / a.chunks, chunk = WHOLE ? 0 : blockIdx.x - row * a.chunks;
  const int t = threadIdx.x, lane = t % L2C_WAVE, wave = t / L2C_WAVE;
  const long long first = static_cast<long long>(chunk) * a.chunk;  // below vocab: no chunk is empty
  const int whole = static_cast<int>(min(static_cast<long long>(a.chunk), a.vocab - first));
  const float *const x = a.logits + static_cast<size_t>(row) * a.vocab + first;
  const int top = a.top;
  float given = 0.0f;  // the token's logit
  bool inside = false;
  if (WHOLE && t == 0 && a.tokens) {
    const int token = a.tokens[row];
    inside = token >= 0 && token < a.vocab;
    if (inside) given = x[token];
  }
  auto load = [&](float4 (&q)[V], int start) __attribute__((always_inline)) {
    const int n = min(kPart, whole - start);
#pragma unroll
    for (int c = 0; c < V; ++c) {  // -Inf past the end
      const int j = 4 * (t + c * kThreads);
      const float *const p = x + start + j;
      q[c] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (j + 4 <= n) {
        q[c] = ld4_any(p);
      } else if (j < n) {
        q[c].x = p[0];
        if (j + 1 < n) q[c].y = p[1];
        if (j + 2 < n) q[c].z = p[2];
      }
    }
  };
  float4 q[V];
  load(q, 0);
  if (t < 3) lengths[t] = 0;
  double z = 0.0, s = 0.0;
  float m = -INFINITY;
  int count = 0, turn = 0, part = 0;  // `kept` has count values,
  int pending = 0;                    // and the list as many
  if (top > 0) __syncthreads();
  for (int start = 0;; ++part) {
    const int n = min(kPart, whole - start);
    const bool more = whole - start > kPart;
    float v[4 * V];
#pragma unroll
    for (int c = 0; c < V; ++c) v[4 * c] = q[c].x, v[4 * c + 1] = q[c].y, v[4 * c + 2] = q[c].z, v[4 * c + 3] = q[c].w;
    if (more) load(q, start + kPart);
    auto place = [&](int i) __attribute__((always_inline)) { return 4 * (t + i / 4 * kThreads) + i % 4; };
    float best_value = -INFINITY;  // the lane's largest, -Inf where all are NaN
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) best_value = fmaxf(best_value, v[i]);
    const unsigned last = __builtin_amdgcn_readlane(__float_as_uint(wave_top(best_value)), L2C_WAVE - 1);
    const float largest = __uint_as_float(last);
    if (largest > m) raise(z, s, m, largest);
    const float subtract = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, product = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) {
      float away = v[i] - subtract;
      away = away < -150.0f ? -150.0f : away;  // exp is 0 there; -Inf times it would be NaN
      const float e = exp_nonpositive(away);
      sum += e;
      product = fmaf(e, away, product);
    }
    z += static_cast<double>(sum);
    s += static_cast<double>(product);
    if (top > 0) {
      // A bound that all of the `top` largest so far reach. If there are as many before this part, only larger
      // ones count: of equal ones the earlier are there.
      const unsigned best = place(0) < n ? key_of(best_value) : 0u;
      unsigned least;
      if (count == top) {
        least = kept_key[turn][top - 1] + 1;
      } else {
        const int sharing = min(kWaves, max(1, n / (4 * L2C_WAVE))), share = (top + sharing - 1) / sharing;
        const unsigned bound = share == 1 ? key_of(largest) : wave_bound(best, share);
        if (lane == L2C_WAVE - 1) bounds[wave] = bound;
        __syncthreads();
        least = bounds[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
          if (w < sharing) least = min(least, bounds[w]);
      }
      least = max(least, key_of(-FLT_MAX));  // -Inf is no alternative
      // The values that reach the bound into the list. If more than `top` of the wave's lanes have such, only
      // those of the `top` lanes with the largest, and of lanes that tie, with the lowest places of it.
      unsigned last = 0;
      if (wave_reach(best, least) > top) {
        least = wave_bound(best, top);
        if (wave_reach(best, least) > top) {
          const int larger = __popcll(__ballot(best > least));
          const float tie = number_of(least);
          unsigned before = 0;
#pragma unroll
          for (int i = 4 * V - 1; i >= 0; --i)
            if (v[i] == tie) before = UINT_MAX - (static_cast<unsigned>(start) + place(i));
          last = wave_bound(best == least ? before : 0u, top - larger);
        }
      }
      const float limit = number_of(least);  // NaN does not reach it, nor does what is past the end
      unsigned reach = 0;
      if (__ballot(best >= least)) {
        if (last == 0) {
#pragma unroll
          for (int i = 0; i < 4 * V; ++i) reach |= v[i] >= limit ? 1u << i : 0u;
        } else {
#pragma unroll
          for (int i = 0; i < 4 * V; ++i)
            if (v[i] > limit || (v[i] == limit && UINT_MAX - (static_cast<unsigned>(start) + place(i)) >= last))
              reach |= 1u << i;
        }
      }
      if (__ballot(reach != 0)) {
        const int count_here = __popc(reach), upto = wave_scan(count_here);
        int base = 0;
        if (lane == L2C_WAVE - 1) base = atomicAdd(&lengths[part % 3], upto);
        int to = pending + __builtin_amdgcn_readlane(base, L2C_WAVE - 1) + upto - count_here;
        // Their places alone; the values are read again where they are put in order.
        while (__ballot(reach != 0)) {
          if (reach != 0) {
            const int i = __ffs(reach) - 1;
            list_before[to++] = UINT_MAX - (static_cast<unsigned>(start) + place(i));
            reach &= reach - 1;
          }
        }
      }
      __syncthreads();
      pending += __builtin_amdgcn_readfirstlane(lengths[part % 3]);
      if (t == 0) lengths[(part + 2) % 3] = 0;  // read before this barrier, used after the next
      // While there is a bound the list only grows, until there are enough of them to find a closer bound by (2048 x
      // 32003, top 20: 70 us with 64, 74 with 128, 77 as long as they fit); then, or at the end, its values and
      // the kept ones are put in order.
      if (pending > 0 && (!more || count < top || pending > min(unit, 64))) {
        const int listed = pending, all = count + listed;
        for (int e = t; e < listed; e += kThreads) list_key[e] = key_of(x[UINT_MAX - list_before[e]]);
        __syncthreads();
        for (int e = t; e < all; e += kThreads) {
          const bool old = e < count;
          const unsigned mine = old ? kept_key[turn][e] : list_key[e - count];
          const unsigned before = old ? kept_before[turn][e] : list_before[e - count];
          Order among = order(list_key, listed, mine);
          const Order among_kept = order(kept_key[turn], count, mine);
          among.larger += among_kept.larger, among.equal += among_kept.equal;
          if (among.equal > 1) {  // it and others
            among.larger += earlier(list_key, list_before, listed, mine, before);
            among.larger += earlier(kept_key[turn], kept_before[turn], count, mine, before);
          }
          if (among.larger < top) kept_key[turn ^ 1][among.larger] = mine, kept_before[turn ^ 1][among.larger] = before;
        }
        count = min(all, top);
        pending = 0;
        turn ^= 1;
        __syncthreads();
      }
    }
    if (!more) break;
    start += kPart;
  }
  z = wave_scan(z), s = wave_scan(s);
  if (lane == L2C_WAVE - 1) zs[wave] = z, ts[wave] = s, tops[wave] = m;
  __syncthreads();
  float most = tops[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) most = fmaxf(most, tops[w]);
  if (WHOLE ? t >= max(top, 1) : t != 0 && t >= top) return;
  if (WHOLE || t == 0) {
    z = s = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      double zw = zs[w], tw = ts[w];
      float mw = tops[w];
      raise(zw, tw, mw, most);
      z += zw, s += tw;
    }
  }
  const bool is = t < count;
  const float logit = is ? number_of(kept_key[turn][t]) : -INFINITY;
  const int token = is ? static_cast<int>(first + (UINT_MAX - kept_before[turn][t])) : -1;
  if constexpr (WHOLE) {
    const Row r(z, s, most);
    if (t == 0) r.store(a, row, given, inside);
    if (t < top) r.alternative(a, row, t, logit, token);
  } else {
    Sums *const sums = reinterpret_cast<Sums *>(a.workspace);
    if (t == 0) sums[blockIdx.x] = {z, s, most, 0};
    Candidate *const to = reinterpret_cast<Candidate *>(sums + gridDim.x) + static_cast<size_t>(blockIdx.x) * top;
    if (t < top) to[t] = {logit, token};
  }
}

// A wave a row, a lane a chunk: the sums; and `top` times the largest first of the chunks' lists, of equal ones
// the one of the first chunk.
__global__ __launch_bounds__(L2C_WAVE) void logprobs_join_kernel(Args a, unsigned rows) {
  extern __shared__ uint4 lists[];
  Candidate *const list = reinterpret_cast<Candidate *>(lists);
  const int row = blockIdx.x, lane = threadIdx.x, n = a.chunks * a.top;
  const Sums *const sums = reinterpret_cast<const Sums *>(a.workspace);
  const Candidate *const from =
      reinterpret_cast<const Candidate *>(sums + static_cast<size_t>(rows) * a.chunks) + static_cast<size_t>(row) * n;
  Sums mine = {0.0, 0.0, -INFINITY, 0};
  if (lane < a.chunks) mine = sums[static_cast<size_t>(row) * a.chunks + lane];
  float given = 0.0f;
  bool inside = false;
  if (a.tokens) {
    const int token = a.tokens[row];
    inside = token >= 0 && token < a.vocab;
    if (inside) given = a.logits[static_cast<size_t>(row) * a.vocab + token];
  }
  for (int i = lane; i < n; i += L2C_WAVE) list[i] = from[i];
  const float most = l2c::wave_max(mine.m);
  if (lane < a.chunks) raise(mine.z, mine.t, mine.m, most);
  const double z = wave_scan(mine.z), t = wave_scan(mine.t);
  auto last = [](double v) __attribute__((always_inline)) {
    const long long bits = __double_as_longlong(v);
    const unsigned low = __builtin_amdgcn_readlane(static_cast<unsigned>(bits), L2C_WAVE - 1);
    const unsigned high = __builtin_amdgcn_readlane(static_cast<unsigned>(bits >> 32), L2C_WAVE - 1);
    return __longlong_as_double(static_cast<long long>(static_cast<u64>(high) << 32 | low));
  };
  const Row r(last(z), last(t), most);
  if (lane == 0) r.store(a, row, given, inside);
  __syncthreads();
  int at = 0, token = -1;  // of the lane's list; what the lane's alternative is
  float logit = -INFINITY;
  Candidate head = {-INFINITY, -1};
  if (lane < a.chunks && a.top > 0) head = list[lane * a.top];
  for (int rank = 0; rank < a.top; ++rank) {
    const unsigned key = head.token >= 0 ? key_of(head.logit) : 0u;
    const unsigned best = wave_top(key);
    if (best == 0) break;
    const int winner = __ffsll(__ballot(key == best)) - 1;
    const float x = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(head.logit), winner));
    const int y = __builtin_amdgcn_readlane(head.token, winner);
    if (lane == rank) logit = x, token = y;
    if (lane == winner) head = ++at < a.top ? list[lane * a.top + at] : Candidate{-INFINITY, -1};
  }
  if (lane < a.top) r.alternative(a, row, lane, logit, token);
}

struct Plan {
  int chunks, chunk, v;
};

// A row a workgroup from 512 rows on (or of no more than 2048 logits), else chunks for about 1024
// workgroups, of 2048 logits at least. No more than 4096 logits in registers at a time: 8192 leave two
// waves a SIMD (2048 x 32003 78 us, 96 so).
Plan plan(int vocab, int rows) {
  int chunks = 1;
  if (rows < 512) {
    const int parts = (vocab - 1) / 2048 + 1;
    chunks = min(min(parts, kMaxChunks), max(1, 1024 / rows));
  }
  Plan p;
  p.chunk = (vocab - 1) / chunks + 1;
  p.chunks = (vocab - 1) / p.chunk + 1;
  p.v = p.chunk <= 1024 ? 1 : p.chunk <= 2048 ? 2 : 4;
  return p;
}

using Kernel = void (*)(Args);
Kernel kernel(const Plan &p) {  // chunks of a row have more than 1024 logits
  if (p.chunks > 1) return p.v == 2 ? logprobs_kernel<2, false> : logprobs_kernel<4, false>;
  return p.v == 1 ? logprobs_kernel<1, true> : p.v == 2 ? logprobs_kernel<2, true> : logprobs_kernel<4, true>;
}

}  // namespace

extern "C" size_t l2c_decoder_logprobs_workspace_bytes(int vocab, int top, int rows) {
  if (vocab <= 0 || top < 0 || top > kMost || rows <= 0) return 0;
  const Plan p = plan(vocab, rows);
  return p.chunks == 1 ? 0 : static_cast<size_t>(rows) * p.chunks * (sizeof(Sums) + top * sizeof(Candidate));
}

extern "C" int l2c_decoder_logprobs(float *logprobs, float *entropies, int *top_tokens, float *top_logprobs,
                                    const float *logits, const int *tokens, int vocab, int top, int rows,
                                    void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (vocab <= 0 || top < 0 || top > kMost || rows < 0 || !logprobs != !tokens) return hipErrorInvalidValue;
  if (rows == 0) return hipSuccess;
  const size_t need = l2c_decoder_logprobs_workspace_bytes(vocab, top, rows);
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & 3u) != 0 || (top > 0 && (!top_tokens || !top_logprobs)) ||
      workspace_bytes < need || (need > 0 && (!workspace || !l2c_aligned16(workspace))))
    return hipErrorInvalidValue;
  const Plan p = plan(vocab, rows);
  const long long grid = static_cast<long long>(rows) * p.chunks;
  if (!l2c::launchable(grid, kThreads)) return hipErrorInvalidValue;
  const Args a = {logprobs, entropies, top_tokens, top_logprobs, logits, tokens,
                  static_cast<unsigned char *>(workspace), vocab, top, p.chunks, p.chunk};
  const size_t list = 2 * sizeof(unsigned) * (2 * kWaves * static_cast<size_t>(top) * 4 * p.v + 8);
  hipLaunchKernelGGL(kernel(p), dim3(static_cast<unsigned>(grid)), dim3(kThreads), list, stream, a);
  L2C_LAUNCH_CHECK();
  if (p.chunks == 1) return hipSuccess;
  hipLaunchKernelGGL(logprobs_join_kernel, dim3(rows), dim3(L2C_WAVE),
                     sizeof(Candidate) * static_cast<size_t>(p.chunks) * top, stream, a, static_cast<unsigned>(rows));
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

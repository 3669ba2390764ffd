// Beam search for the batched decoder: the choice of a request's next beams among
// beams x vocabulary, and the states that follow the chosen beams' parents.
//
// Selection, for each request, with scores s_k of its beams and their logits x_k:
//   s_k + x_k[v] - log sum_u exp(x_k[u])
// over all beams k and tokens v; the `beams` largest are the next beams. Two kernels:
//
//  * beam_chunks_kernel, a workgroup per chunk of a row of logits: one pass over the
//    data, which the lanes hold in registers. It leaves the chunk's maximum, its sum of
//    exponentials and its `beams` largest logits in order. Nothing is sorted: the K-th
//    largest of a wave's 64 lane maxima is a bound that at least K values of the chunk
//    reach, and few more do. It is found bit by bit, a ballot a bit. The values that
//    reach the largest of the waves' bounds go to a list in LDS, where each finds its
//    rank by comparison with the others. A wave has at most K lanes whose maximum
//    reaches the bound, so the list's length has a bound too.
//  * beam_join_kernel, a workgroup per request: the rows' sums, and the same choice
//    among the chunks' lists by their 64-bit scores.
//
// The order is total: larger first, then the lower beam, then the lower token; within
// a row by the logits themselves. Results do not depend on the order of the list's
// atomics. Sums of exponentials are fp32 within a lane and 64-bit across lanes, scores
// 64-bit until they are stored: beams' scores lie close together, and a rounding
// there would change which tokens are chosen.
#include <climits>

#include "l2c_common.h"
#include "../../include/l2c.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / L2C_WAVE;
constexpr int kMaxBeams = L2C_MAX_BEAMS;

typedef unsigned long long u64;

// What a chunk leaves in the workspace, followed by `beams` candidates.
struct ChunkStat {
  double sum;  // of exp(x - maximum); NaN if the chunk holds a NaN or +Inf
  float maximum;
  int unused;
};
struct Candidate {
  float logit;
  int token;  // -1: none
};
__host__ __device__ __forceinline__ size_t chunk_bytes(int beams) {
  return sizeof(ChunkStat) + sizeof(Candidate) * static_cast<size_t>(beams);
}

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

// The largest T that at least k of the wave's 64 values reach: the k-th largest.
template <typename T>
__device__ __forceinline__ T wave_kth(T v, int k) {
  T bound = 0;
  for (int bit = 8 * sizeof(T) - 1; bit >= 0; --bit) {
    const T next = bound | (static_cast<T>(1) << bit);
    if (__popcll(__ballot(v >= next)) >= k) bound = next;
  }
  return bound;
}

// 64-bit order of a chunk's values: the logit, then the lower place first.
__device__ __forceinline__ u64 ordered(unsigned key, unsigned place) {
  return (static_cast<u64>(key) << 32) | (UINT_MAX - place);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, L2C_WAVE);
  return v;
}

// V float4 a lane; `chunks` chunks of kThreads * 4 V logits a row.
template <int V>
__global__ __launch_bounds__(kThreads) void beam_chunks_kernel(unsigned char *__restrict__ workspace,
                                                               const float *__restrict__ logits,
                                                               const int *__restrict__ tokens, int eos, int vocab,
                                                               int beams, int chunks) {
  extern __shared__ u64 list[];  // at most kWaves * beams lanes' 4 V values
  __shared__ u64 bounds[kWaves];
  __shared__ unsigned tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ int length;
  const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
  if (eos >= 0 && tokens[row] == eos) return;  // ended: its logits do not count
  const int t = threadIdx.x, lane = t % L2C_WAVE, wave = t / L2C_WAVE;
  const int first = chunk * (kThreads * 4 * V);
  const int n = min(kThreads * 4 * V, vocab - first);
  const float *x = logits + static_cast<size_t>(row) * vocab + first;
  float4 q[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const int j = 4 * (t + c * kThreads);
    if (j < n) q[c] = l2c::ld_chunk(x, j, n);
  }
  if (t == 0) length = 0;
  float v[4 * V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const int j = 4 * (t + c * kThreads);
    const float4 w = j < n ? l2c::whole_chunk(q[c], j, n, -INFINITY) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    v[4 * c] = w.x, v[4 * c + 1] = w.y, v[4 * c + 2] = w.z, v[4 * c + 3] = w.w;
  }
  // The lane's first maximum.
  auto place = [&](int i) __attribute__((always_inline)) { return 4 * (t + i / 4 * kThreads) + i % 4; };
  auto key = [&](int i) __attribute__((always_inline)) { return place(i) < n ? key_of(v[i]) : 0u; };
  unsigned best = 0, best_place = UINT_MAX;
#pragma unroll
  for (int i = 0; i < 4 * V; ++i) {
    const unsigned k = key(i);
    if (k > best) best = k, best_place = place(i);
  }
  const unsigned bound = wave_kth(best, beams);
  unsigned bound_place = UINT_MAX;
  const u64 tied = __ballot(best == bound && bound != 0);
  const int wanted = beams - __popcll(__ballot(best > bound));
  if (__popcll(tied) > wanted) {  // of the lanes whose maxima tie, those with the lowest places
    bound_place = UINT_MAX - wave_kth(best == bound ? UINT_MAX - best_place : 0u, wanted);
  }
  unsigned top = best;
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), offset, L2C_WAVE)));
  if (lane == 0) {
    bounds[wave] = ordered(bound, bound_place);
    tops[wave] = top;
  }
  __syncthreads();
  u64 least = bounds[0];
  unsigned most = tops[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    least = max(least, bounds[w]);
    most = max(most, tops[w]);
  }
  // All -Inf or NaN: no finite maximum to subtract.
  const float maximum = most ? number_of(most) : -INFINITY;
  const float shift = maximum == -INFINITY ? 0.0f : maximum;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4 * V; ++i) sum += expf(v[i] - shift);
  const double total = wave_sum(static_cast<double>(sum));
  if (lane == 0) sums[wave] = total;
  if (ordered(best, best_place) >= least) {
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) {
      const unsigned k = key(i);
      if (k != 0 && ordered(k, place(i)) >= least) list[atomicAdd(&length, 1)] = ordered(k, place(i));
    }
  }
  __syncthreads();
  unsigned char *entry = workspace + (static_cast<size_t>(row) * chunks + chunk) * chunk_bytes(beams);
  Candidate *out = reinterpret_cast<Candidate *>(entry + sizeof(ChunkStat));
  const int m = length;
  for (int e = t; e < m; e += kThreads) {
    const u64 mine = list[e];
    int rank = 0;
    for (int o = 0; o < m; ++o) rank += list[o] > mine;
    if (rank < beams)
      out[rank] = {number_of(static_cast<unsigned>(mine >> 32)), first + static_cast<int>(UINT_MAX - static_cast<unsigned>(mine))};
  }
  for (int e = m + t; e < beams; e += kThreads) out[e] = {-INFINITY, -1};
  if (t == 0) {
    double all = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all += sums[w];
    *reinterpret_cast<ChunkStat *>(entry) = {all, maximum, 0};
  }
}

constexpr int kJoinList = 2048;

// A candidate's place in the request: beam, then token.
__device__ __forceinline__ u64 place_of(int beam, int token) {
  return (static_cast<u64>(beam) << 32) | static_cast<unsigned>(token);
}

__global__ __launch_bounds__(kThreads) void beam_join_kernel(float *scores_out, int *tokens_out, int *parents,
                                                             int *generated, const unsigned char *workspace,
                                                             const float *scores, const int *tokens, int eos,
                                                             int beams, int chunks, int steps, int step) {
  // A beam's scores are base + (logit - top), in this order: logits of the lowest value
  // would take the rest of the sum with them. NaN: no candidates.
  __shared__ double base[kMaxBeams];
  __shared__ float tops[kMaxBeams];
  __shared__ bool ended[kMaxBeams];
  __shared__ u64 list_key[kJoinList], list_place[kJoinList];
  __shared__ u64 slots[kWaves], place_slots[kWaves];
  __shared__ int length;
  const int t = threadIdx.x, lane = t % L2C_WAVE, wave = t / L2C_WAVE;
  const int first = blockIdx.x * beams;
  const size_t bytes = chunk_bytes(beams);
  auto stat = [&](int beam, int chunk) __attribute__((always_inline)) {
    return reinterpret_cast<const ChunkStat *>(workspace + (static_cast<size_t>(first + beam) * chunks + chunk) * bytes);
  };
  if (t == 0) length = 0;
  for (int k = wave; k < beams; k += kWaves) {
    const float score = scores[first + k];
    const bool end = eos >= 0 && tokens[first + k] == eos;
    const bool live = score >= -FLT_MAX && score <= FLT_MAX;
    double b = score;
    float m = 0.0f;
    if (!end && live) {
      m = -INFINITY;
      for (int c = lane; c < chunks; c += L2C_WAVE) m = fmaxf(m, stat(k, c)->maximum);
      m = l2c::wave_max(m);
      double sum = 0.0;
      for (int c = lane; c < chunks; c += L2C_WAVE) {
        const ChunkStat s = *stat(k, c);
        // A chunk of -Inf has sum 0; NaN stays NaN.
        sum += s.maximum == -INFINITY ? s.sum * 0.0 : s.sum * exp(static_cast<double>(s.maximum) - static_cast<double>(m));
      }
      sum = wave_sum(sum);
      b -= log(sum);
    }
    // Of a row of -Inf the sum is 0 and b +Inf, of one with NaN or +Inf it is NaN.
    if (lane == 0) {
      tops[k] = m;
      base[k] = live && b >= -DBL_MAX && b <= DBL_MAX ? b : __longlong_as_double(0x7ff8000000000000LL);
      ended[k] = end;
    }
  }
  __syncthreads();
  const int lists = beams * chunks;
  // Score key and place of candidate e of list l; key 0 where there is none.
  auto candidate = [&](int l, int e, u64 *place) __attribute__((always_inline)) -> u64 {
    const int beam = l / chunks, chunk = l - beam * chunks;
    if (ended[beam]) {
      *place = place_of(beam, eos);
      return chunk == 0 && e == 0 ? key_of(base[beam]) : 0ULL;
    }
    const Candidate c = reinterpret_cast<const Candidate *>(stat(beam, chunk) + 1)[e];
    *place = place_of(beam, c.token);
    return c.token >= 0 && c.logit > -INFINITY ? key_of(base[beam] + (static_cast<double>(c.logit) - tops[beam])) : 0ULL;
  };
  auto before = [](u64 key, u64 place, u64 other, u64 other_place) __attribute__((always_inline)) {
    return key > other || (key == other && place < other_place);
  };
  auto write = [&](int rank, u64 key, u64 place) __attribute__((always_inline)) {
    const int to = first + rank;
    const int token = key ? static_cast<int>(place) : -1;
    scores_out[to] = key ? static_cast<float>(number_of(key)) : -INFINITY;
    tokens_out[to] = token;
    parents[to] = key ? static_cast<int>(place >> 32) : -1;
    if (generated) generated[static_cast<size_t>(to) * steps + step] = token;
  };

  // The lists' heads are their largest: the k-th largest of the lanes' best heads is a
  // bound that at least `beams` candidates reach. Equal keys all pass.
  u64 best = 0;
  for (int l = t; l < lists; l += kThreads) {
    u64 place;
    best = max(best, candidate(l, 0, &place));
  }
  const u64 bound = wave_kth(best, beams);
  if (lane == 0) slots[wave] = bound;
  __syncthreads();
  u64 least = slots[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) least = max(least, slots[w]);
  least = max(least, static_cast<u64>(1));
  if (best >= least) {
    for (int l = t; l < lists; l += kThreads) {
      for (int e = 0; e < beams; ++e) {
        u64 place;
        const u64 key = candidate(l, e, &place);
        if (key < least) break;  // so are the rest of the list
        const int at = atomicAdd(&length, 1);
        if (at < kJoinList) list_key[at] = key, list_place[at] = place;
      }
    }
  }
  __syncthreads();
  const int m = length;
  if (m <= kJoinList) {
    for (int e = t; e < m; e += kThreads) {
      const u64 key = list_key[e], place = list_place[e];
      int rank = 0;
      for (int o = 0; o < m; ++o) rank += before(list_key[o], list_place[o], key, place);
      if (rank < beams) write(rank, key, place);
    }
    for (int e = m + t; e < beams; e += kThreads) write(e, 0, 0);
    return;
  }
  // More than the list holds: one beam after another, each the best after the last.
  u64 last = ~0ULL, last_place = 0;
  bool any = false;
  for (int r = 0; r < beams; ++r) {
    u64 top = 0, top_place = ~0ULL;
    for (int l = t; l < lists; l += kThreads) {
      for (int e = 0; e < beams; ++e) {
        u64 place;
        const u64 key = candidate(l, e, &place);
        if (key == 0) break;
        if (any && !before(last, last_place, key, place)) continue;
        if (before(key, place, top, top_place)) top = key, top_place = place;
      }
    }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) {
      const u64 k = __shfl_xor(top, offset, L2C_WAVE), p = __shfl_xor(top_place, offset, L2C_WAVE);
      if (before(k, p, top, top_place)) top = k, top_place = p;
    }
    __syncthreads();  // the slots of the round before are read
    if (lane == 0) slots[wave] = top, place_slots[wave] = top_place;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (before(slots[w], place_slots[w], top, top_place)) top = slots[w], top_place = place_slots[w];
    if (t == 0) write(r, top, top_place);
    last = top, last_place = top_place, any = true;
  }
}

using ChunkKernel = void (*)(unsigned char *, const float *, const int *, int, int, int, int);

struct ChunkConfig {
  ChunkKernel fn;
  int values, chunks;  // values a lane, chunks a row
};

ChunkConfig chunk_config(int vocab, int beams, int batch) {
  (void)beams, (void)batch;
  const int values = 8;
  return {beam_chunks_kernel<2>, values, (vocab - 1) / (kThreads * values) + 1};
}

}  // namespace

extern "C" size_t l2c_decoder_beam_workspace_bytes(int vocab, int beams, int batch) {
  if (vocab <= 0 || beams <= 0 || beams > kMaxBeams || batch <= 0) return 0;
  return static_cast<size_t>(batch) * beams * chunk_config(vocab, beams, batch).chunks * chunk_bytes(beams);
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
  const size_t list = sizeof(u64) * kWaves * static_cast<size_t>(beams) * c.values;
  hipLaunchKernelGGL(c.fn, dim3(static_cast<unsigned>(grid)), dim3(kThreads), list, stream, w, logits, tokens, eos,
                     vocab, beams, c.chunks);
  L2C_LAUNCH_CHECK();
  hipLaunchKernelGGL(beam_join_kernel, dim3(static_cast<unsigned>(batch)), dim3(kThreads), 0, stream, scores_out,
                     tokens_out, parents, generated, w, scores, tokens, eos, beams, c.chunks, steps, step);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

// ---------------------------------------------------------------------------
// States that follow their beams.
//
// out[g][b][k] = in[g][b][parents[b][k]]: a lane moves one column of 16 bytes, or one
// byte of what is left of a piece, of all beams of a request. It has loaded all of them
// when it stores the first, so `out` may be `in`: no other lane touches its column. In
// place, a beam that is its own parent costs nothing.

namespace {

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// from[k]: the row that row k becomes, -1 where it stays.
template <int BEAMS, typename T>
__device__ __forceinline__ void move_column(unsigned char *out, const unsigned char *in, const int (&from)[BEAMS],
                                            long long row_stride) {
  T v[BEAMS];
#pragma unroll
  for (int k = 0; k < BEAMS; ++k)
    if (from[k] >= 0) v[k] = *reinterpret_cast<const T *>(in + from[k] * row_stride);
#pragma unroll
  for (int k = 0; k < BEAMS; ++k)
    if (from[k] >= 0) *reinterpret_cast<T *>(out + k * row_stride) = v[k];
}

template <int BEAMS>
__global__ __launch_bounds__(kThreads) void beam_reorder_kernel(unsigned char *out, const unsigned char *in,
                                                                const int *__restrict__ parents, int beams, int batch,
                                                                unsigned columns, unsigned wide, unsigned all,
                                                                unsigned blocks, long long group_stride,
                                                                long long row_stride, long long piece_stride) {
  const unsigned state = blockIdx.x / blocks, part = blockIdx.x - state * blocks;
  const int group = state / batch, request = state - group * batch;
  const unsigned i = part * kThreads + threadIdx.x;
  if (i >= all) return;
  const unsigned piece = i / columns, c = i - piece * columns;
  const long long at = group * group_stride + static_cast<long long>(request) * beams * row_stride +
                       piece * piece_stride + (c < wide ? 16LL * c : 16LL * wide + (c - wide));
  const bool in_place = out == in;
  int from[BEAMS];
#pragma unroll
  for (int k = 0; k < BEAMS; ++k) {
    const int p = k < beams ? parents[static_cast<size_t>(request) * beams + k] : -1;
    from[k] = p < beams && !(in_place && p == k) ? p : -1;
  }
  if (c < wide) move_column<BEAMS, u32x4_any>(out + at, in + at, from, row_stride);
  else move_column<BEAMS, unsigned char>(out + at, in + at, from, row_stride);
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
  const long long blocks = (static_cast<long long>(all) + kThreads - 1) / kThreads;
  const wide_t grid = static_cast<wide_t>(blocks) * groups * batch;
  if (grid > INT_MAX || !l2c::launchable(static_cast<long long>(grid), kThreads)) return hipErrorInvalidValue;
  auto fn = beams <= 4 ? beam_reorder_kernel<4> : beams <= 8 ? beam_reorder_kernel<8>
            : beams <= 16 ? beam_reorder_kernel<16> : beam_reorder_kernel<32>;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, static_cast<unsigned char *>(out),
                     static_cast<const unsigned char *>(in), parents, beams, batch, static_cast<unsigned>(columns),
                     static_cast<unsigned>(piece_bytes / 16), static_cast<unsigned>(all),
                     static_cast<unsigned>(blocks), group_stride, row_stride, piece_stride);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

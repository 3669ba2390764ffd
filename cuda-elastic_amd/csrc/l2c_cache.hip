// The pages of a cache: new tokens' keys and values written into them, the step of the
// tables that name them, and the copies of pages that two sequences would write.
#include "l2c_cache.h"
#include "l2c_formats.h"

namespace {

using l2c::Sequences;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// append

constexpr int kAppendThreads = 256;

__device__ __forceinline__ float low_half(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_half(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// Keys, then values of a row's heads, then the next row's: an item each, by G lanes with eight values a lane,
// kItems items one after the other by the same lanes, all of them on their way before the first is looked at.
// Bound by memory; where a row goes is found once for the workgroup, meanwhile. 8192 rows of 8 x 128 into e4m3 pages
// 12.0-14.7 us (3.1 TB/s), 39 with an item a lane and every lane's own search; 64 rows into bf16 pages 2.4-2.7.
template <int G, int kItems, bool E4M3>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(void *keys, void *values, float *key_scales,
                                                                float *value_scales, const uint16_t *k,
                                                                long long k_stride, const uint16_t *v,
                                                                long long v_stride, Sequences s, int kv_heads,
                                                                int width, l2c::Quotient31 by_each) {
  constexpr int kTogether = kAppendThreads / G, kBlock = kTogether * kItems;
  __shared__ long long places[kBlock + 1];  // of the block's rows: in the cache's rows of head 0; -1: nowhere
  const int t = threadIdx.x, lane = t % G;
  const int each = 2 * kv_heads, all = each * s.rows, first = blockIdx.x * kBlock, first_row = by_each(first);
  // k and v may end where the sequences' rows do.
  const int begin = s.starts ? s.starts[0] : 0, end = s.starts ? min(s.starts[s.sequences], s.rows) : s.rows;
  u32x4 x[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int item = first + i * kTogether + t / G;
    x[i] = u32x4{0, 0, 0, 0};
    if (item >= all || 8 * lane >= width) continue;
    const int row = by_each(item), of = item - row * each;
    if (row < begin || row >= end) continue;
    const bool value = of >= kv_heads;
    const uint16_t *const from = value ? v + row * v_stride + static_cast<long long>(of - kv_heads) * width
                                       : k + row * k_stride + static_cast<long long>(of) * width;
    x[i] = *reinterpret_cast<const u32x4 *>(from + 8 * lane);
  }
  const int rows = by_each(min(first + kBlock, all) - 1) - first_row + 1;  // at most kBlock, two of which may be parts
  if (t < rows) {
    long long place = -1;
    int sequence, position;
    if (s.find(first_row + t, sequence, position) && position >= 0 && position < s.capacity()) {
      const int index = s.by_page(position), page = s.page(sequence, index);
      if (s.is_page(page))
        place = static_cast<long long>(page) * kv_heads * s.page_size + (position - index * s.page_size);
    }
    places[t] = place;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int item = first + i * kTogether + t / G;
    const int row = by_each(item), of = item - row * each;
    const long long place = item < all ? places[row - first_row] : -1;
    const bool value = of >= kv_heads, mine = place >= 0 && 8 * lane < width;
    const size_t to = place + static_cast<size_t>(value ? of - kv_heads : of) * s.page_size;
    if constexpr (!E4M3) {
      uint16_t *const cache = static_cast<uint16_t *>(value ? values : keys);
      if (mine) *reinterpret_cast<u32x4 *>(cache + to * width + 8 * lane) = x[i];
    } else {
      unsigned largest = 0;  // of the magnitudes' patterns, which order as the numbers do, NaN above all
#pragma unroll
      for (int e = 0; e < 4; ++e) largest = max(largest, max(x[i][e] << 16 & 0x7fff0000u, x[i][e] & 0x7fff0000u));
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) largest = max(largest, __shfl_xor(largest, o, L2C_WAVE));
      const bool finite = largest < 0x7f800000u;
      const float amax = __uint_as_float(largest);
      const float scale = !finite ? __uint_as_float(0x7fc00000u) : amax > 0.0f ? amax / 448.0f : 1.0f;
      u32x2 code = {0, 0};
      if (finite && l2c::fp8_has_short_quotient(scale)) {
        const float y = 1.0f / scale;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned low = x[i][2 * e], high = x[i][2 * e + 1];
          int c = __builtin_amdgcn_cvt_pk_fp8_f32(l2c::fp8_short_quotient(low_half(low), scale, y),
                                                  l2c::fp8_short_quotient(high_half(low), scale, y), 0, false);
          c = __builtin_amdgcn_cvt_pk_fp8_f32(l2c::fp8_short_quotient(low_half(high), scale, y),
                                              l2c::fp8_short_quotient(high_half(high), scale, y), c, true);
          const unsigned u = static_cast<unsigned>(c);
          const unsigned nonzero = ((u & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u;  // zeros are +0
          code[e] = u & (nonzero | 0x7f7f7f7fu);
        }
      } else if (finite) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned pair =
              l2c::e4m3_code(low_half(x[i][e]) / scale) | l2c::e4m3_code(high_half(x[i][e]) / scale) << 8;
          code[e / 2] |= pair << 16 * (e % 2);
        }
      }
      if (mine) {
        *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(value ? values : keys) + to * width + 8 * lane) = code;
        if (lane == 0) (value ? value_scales : key_scales)[to] = scale;
      }
    }
  }
}

using AppendKernel = void (*)(void *, void *, float *, float *, const uint16_t *, long long, const uint16_t *,
                              long long, Sequences, int, int, l2c::Quotient31);
template <int G>
AppendKernel append_of(bool many, bool e4m3) {
  return many ? (e4m3 ? append_kernel<G, 4, true> : append_kernel<G, 4, false>)
              : (e4m3 ? append_kernel<G, 1, true> : append_kernel<G, 1, false>);
}

// ---------------------------------------------------------------------------
// advance

constexpr int kAdvanceThreads = 1024;

struct Step {
  int *tables_out, *lengths_out, *uses, *copies, *shortage;
  const int *tables, *lengths, *parents, *starts, *held;
  int beams, sequences, pages, max_pages, page_size, window;

  __device__ __forceinline__ int pages_of(long long positions) const {  // may be more than max_pages
    return static_cast<int>((positions + page_size - 1) / page_size);
  }
  // Its parent (-1: none), the parent's length and the new tokens of a sequence.
  __device__ __forceinline__ int parent(int r, int &length, int &n) const {
    int p = r;
    if (parents) {
      const int k = parents[r];
      p = k >= 0 && k < beams ? r - r % beams + k : -1;
    }
    length = p < 0 ? 0 : max(0, lengths[p]);
    n = p < 0 ? 0 : starts ? static_cast<int>(max(0LL, static_cast<long long>(starts[r + 1]) - starts[r])) : 1;
    n = min(n, INT_MAX - length);
    return p;
  }
};

__device__ __forceinline__ int now(const int *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put(int *p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The sum over the workgroup's kAdvanceThreads lanes before this one; `all` over all of them.
template <class T>
__device__ __forceinline__ T scan_before(T v, T *slots, T &all) {
  constexpr int kWaves = kAdvanceThreads / L2C_WAVE;
  const int lane = threadIdx.x % L2C_WAVE, wave = threadIdx.x / L2C_WAVE;
  T upto = v;
#pragma unroll
  for (int o = 1; o < L2C_WAVE; o <<= 1) {
    const T before = __shfl_up(upto, o, L2C_WAVE);
    if (lane >= o) upto += before;
  }
  __syncthreads();  // the slots may still be read from the call before
  if (lane == L2C_WAVE - 1) slots[wave] = upto;
  __syncthreads();
  T base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) base += slots[w];
    all += slots[w];
  }
  return base + upto - v;
}

// A workgroup a sequence: its parent's entries; and the uses, where they are counted in place, from 0.
template <bool USES>
__global__ __launch_bounds__(256) void advance_tables_kernel(Step s) {
  const int r = blockIdx.x;
  if constexpr (USES)
    for (long long i = static_cast<long long>(r) * blockDim.x + threadIdx.x; i < s.pages;
         i += static_cast<long long>(gridDim.x) * blockDim.x)
      s.uses[i] = 0;
  int length, n;
  const int p = s.parent(r, length, n);
  const int have = min(s.pages_of(length), s.max_pages);
  const int dropped = s.window ? max(0, length - s.window + 1) / s.page_size : 0;  // entries behind the window
  int *const to = s.tables_out + static_cast<size_t>(r) * s.max_pages;
  const int *const from = s.tables + static_cast<size_t>(max(p, 0)) * s.max_pages;
  for (int i = threadIdx.x; i < s.max_pages; i += blockDim.x) to[i] = i < have && i >= dropped ? from[i] : -1;
}

__global__ __launch_bounds__(256) void advance_count_kernel(Step s) {
  const int r = blockIdx.x;
  int length, n;
  s.parent(r, length, n);
  const int have = min(s.pages_of(length), s.max_pages);
  const int *const table = s.tables_out + static_cast<size_t>(r) * s.max_pages;
  for (int i = threadIdx.x; i < have; i += blockDim.x)
    if (static_cast<unsigned>(table[i]) < static_cast<unsigned>(s.pages)) atomicAdd(&s.uses[table[i]], 1);
}

// One workgroup: which pages are replaced, and the new pages for all sequences. A
// sequence that writes into a page takes itself off its uses; what is left are those who do not
// write. Where nobody is, the lowest sequence leaves its number less the number of
// sequences, a negative one, by which it finds that it keeps the page. Sums and minima of
// integers: the order of the atomics does not show. 512 sequences over 13433 pages take the three kernels 34.8 us;
// the next one, with the tables', does so in 21.
__global__ __launch_bounds__(kAdvanceThreads) void advance_assign_kernel(Step s) {
  __shared__ long long slots[kAdvanceThreads / L2C_WAVE];
  const int t = threadIdx.x;
  // Entries that sequence r has and needs; the page that it writes into, or -1.
  auto written = [&](int r, int &first, int &last) {
    int length, n;
    s.parent(r, length, n);
    first = s.pages_of(length), last = s.pages_of(static_cast<long long>(length) + n);
    if (n == 0 || length % s.page_size == 0 || first > s.max_pages) return -1;
    const int page = s.tables_out[static_cast<size_t>(r) * s.max_pages + first - 1];
    return static_cast<unsigned>(page) < static_cast<unsigned>(s.pages) ? page : -1;
  };
  int first, last;
  for (int r = t; r < s.sequences; r += kAdvanceThreads) {
    const int page = written(r, first, last);
    if (page >= 0) atomicSub(&s.uses[page], 1);
  }
  __syncthreads();
  for (int r = t; r < s.sequences; r += kAdvanceThreads) {
    const int page = written(r, first, last);
    if (page >= 0 && now(&s.uses[page]) <= 0 && !(s.held && s.held[page])) atomicMin(&s.uses[page], r - s.sequences);
  }
  __syncthreads();
  // copies is scratch until the end: the page that is replaced, or -1, and how many new pages the
  // sequences before need (no more than INT_MAX, which no page's number reaches).
  long long total = 0, beyond = 0;
  for (int from = 0; from < s.sequences; from += kAdvanceThreads) {
    const int r = from + t;
    int replaced = -1;
    long long need = 0, lost = 0, all;
    if (r < s.sequences) {
      const int page = written(r, first, last);
      if (page >= 0 && now(&s.uses[page]) != r - s.sequences) replaced = page;
      const int upto = min(last, s.max_pages);
      need = max(0, upto - first) + (replaced >= 0);
      lost = last - max(first, upto);
    }
    const long long before = total + scan_before<long long>(need, slots, all);
    if (r < s.sequences) {
      s.copies[2LL * r] = replaced;
      s.copies[2LL * r + 1] = static_cast<int>(min(before, static_cast<long long>(INT_MAX)));
    }
    total += all;
    scan_before<long long>(lost, slots, all);
    beyond += all;
  }
  __syncthreads();
  for (int r = t; r < s.sequences; r += kAdvanceThreads) {
    const int page = written(r, first, last);
    if (page >= 0 && now(&s.uses[page]) == r - s.sequences) put(&s.uses[page], 1);  // it keeps the page
  }
  __syncthreads();
  // Free pages in order, each to the sequence that its rank falls to.
  long long given = 0;
  for (long long from = 0; from < s.pages && given < total; from += kAdvanceThreads) {
    const int page = static_cast<int>(min(from + t, static_cast<long long>(INT_MAX)));
    const bool free = page < s.pages && now(&s.uses[page]) == 0 && !(s.held && s.held[page]);
    long long all;
    const long long rank = given + scan_before<long long>(free, slots, all);
    if (free && rank < total) {
      int low = 0, high = s.sequences - 1;  // the last sequence whose first rank is at most this one
      while (low < high) {
        const int middle = high - (high - low) / 2;
        if (s.copies[2LL * middle + 1] <= rank) low = middle;
        else high = middle - 1;
      }
      const int replaced = s.copies[2LL * low] >= 0;
      int length, n;
      s.parent(low, length, n);
      const int entry = s.pages_of(length) - replaced + static_cast<int>(rank - s.copies[2LL * low + 1]);
      s.tables_out[static_cast<size_t>(low) * s.max_pages + entry] = page;
      put(&s.uses[page], 1);
    }
    given += all;
  }
  __syncthreads();
  for (int r = t; r < s.sequences; r += kAdvanceThreads) {
    int length, n;
    s.parent(r, length, n);
    const int replaced = s.copies[2LL * r];
    if (replaced >= 0) {
      int *const entry = s.tables_out + static_cast<size_t>(r) * s.max_pages + s.pages_of(length) - 1;
      const bool none = s.copies[2LL * r + 1] >= given;
      if (none) *entry = -1;
      s.copies[2LL * r] = none ? -1 : replaced;
      s.copies[2LL * r + 1] = none ? -1 : *entry;
    } else {
      s.copies[2LL * r + 1] = -1;
    }
    s.lengths_out[r] = length + n;
  }
  if (t == 0) *s.shortage = static_cast<int>(min(max(total - given, 0LL) + beyond, static_cast<long long>(INT_MAX)));
}

// The same for up to 1024 sequences and as many pages as LDS has counters for, in one workgroup with a lane a
// sequence: the steps below wait for LDS instead of memory. COPY: the tables, too, where they are small
// enough for one workgroup to be the sooner done. 32 sequences over 312 pages take 5.6 us, lengths and parents 1, the
// tables 0.6, who writes 1.4, free pages 2.4; 512 over 13433 pages, whose 132000 entries one CU reads, 18: 1.4,
// 6.5, 1.5 and 5.5. (Equal entries of sequences below each other counted together took 21 in all.)
constexpr int kLdsPages = 32768, kLdsSequences = kAdvanceThreads, kCopyEntries = 8192, kLdsEntries = 1 << 18;

typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(4)));

template <bool COPY>
__global__ __launch_bounds__(kAdvanceThreads) void advance_lds_kernel(Step s) {
  __shared__ int uses[kLdsPages];
  __shared__ int parent[kLdsSequences], have[kLdsSequences], dropped[kLdsSequences];
  __shared__ int base[kLdsSequences], entry[kLdsSequences], fresh[kLdsSequences];
  constexpr int kWaves = kAdvanceThreads / L2C_WAVE;
  __shared__ int slots[kWaves], ranks[kLdsPages / L2C_WAVE];
  __shared__ unsigned long long beyond;
  const int t = threadIdx.x, lane = t % L2C_WAVE, wave = __builtin_amdgcn_readfirstlane(t / L2C_WAVE);
  const bool is = t < s.sequences;
  int length = 0, n = 0, first = 0, last = 0, page = -1;
  if (is) {
    const int p = s.parent(t, length, n);
    first = s.pages_of(length), last = s.pages_of(static_cast<long long>(length) + n);
    // The page that the sequence writes into, or -1.
    if (n > 0 && length % s.page_size != 0 && first <= s.max_pages)
      page = s.tables[static_cast<size_t>(p) * s.max_pages + first - 1];
    parent[t] = max(p, 0), have[t] = min(first, s.max_pages);
    dropped[t] = s.window ? max(0, length - s.window + 1) / s.page_size : 0;
  }
  for (int i = t; i < s.pages; i += kAdvanceThreads) uses[i] = 0;
  if (t == 0) beyond = 0;
  __syncthreads();
  auto count = [&](int e) __attribute__((always_inline)) {
    if (static_cast<unsigned>(e) < static_cast<unsigned>(s.pages)) atomicAdd(&uses[e], 1);
  };
  if constexpr (COPY) {
    // A wave a sequence, four of them at a time.
    constexpr int kEach = 4;
    for (int from = wave; from < s.sequences; from += kEach * kWaves)
      for (int i = lane; i < s.max_pages; i += L2C_WAVE) {
        int e[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          const int r = from + u * kWaves;
          e[u] = -1;
          if (r < s.sequences && i >= dropped[r] && i < have[r])
            e[u] = s.tables[static_cast<size_t>(parent[r]) * s.max_pages + i];
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          const int r = from + u * kWaves;
          count(e[u]);
          if (r < s.sequences) s.tables_out[static_cast<size_t>(r) * s.max_pages + i] = e[u];
        }
      }
  } else {
    // The tables as one array, in which all that is no sequence's is -1.
    constexpr int kEach = 8;
    const int all = s.sequences * s.max_pages, whole = all / 4;
    for (int from = t; from < whole; from += kEach * kAdvanceThreads) {
      i32x4_any e[kEach];
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int i = from + u * kAdvanceThreads;
        e[u] = i32x4_any{-1, -1, -1, -1};
        if (i < whole) e[u] = *reinterpret_cast<const i32x4_any *>(s.tables_out + 4 * i);
      }
#pragma unroll
      for (int u = 0; u < kEach; ++u)
#pragma unroll
        for (int m = 0; m < 4; ++m) count(e[u][m]);
    }
    if (t < all % 4) count(s.tables_out[4 * whole + t]);
  }
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(s.pages)) page = -1;
  const bool held = page >= 0 && s.held && s.held[page];
  __syncthreads();
  if (page >= 0) atomicSub(&uses[page], 1);
  __syncthreads();
  if (page >= 0 && uses[page] <= 0 && !held) atomicMin(&uses[page], t - s.sequences);
  __syncthreads();
  const bool keeps = page >= 0 && uses[page] == t - s.sequences, replaced = page >= 0 && !keeps;
  const int upto = min(last, s.max_pages);
  if (is && last > max(first, upto)) atomicAdd(&beyond, static_cast<unsigned long long>(last - max(first, upto)));
  int total;  // no more than the tables' entries, and a page that each sequence replaces
  // Its barriers part the reads of uses above from what follows.
  const int before = scan_before(is ? max(0, upto - first) + replaced : 0, slots, total);
  if (keeps) uses[page] = 1;
  if (is) {
    base[t] = before;
    entry[t] = first - replaced;
    fresh[t] = -1;
  }
  __syncthreads();
  // Free pages in order, each to the sequence that its rank falls to. A wave's 64 of the i-th 1024 are lane i's mask,
  // and all of those are ranked by one sum.
  static_assert(kLdsPages / kAdvanceThreads <= L2C_WAVE, "a lane each");
  const int rounds = (s.pages + kAdvanceThreads - 1) / kAdvanceThreads, masks = rounds * kWaves;
  unsigned low_mask = 0, high_mask = 0;
#pragma unroll 4
  for (int i = 0; i < rounds; ++i) {
    const int of = i * kAdvanceThreads + t;
    const unsigned long long free = __ballot(of < s.pages && uses[of] == 0 && !(s.held && s.held[of]));
    if (lane == i) low_mask = static_cast<unsigned>(free), high_mask = static_cast<unsigned>(free >> 32);
  }
  if (lane < rounds) ranks[lane * kWaves + wave] = __popc(low_mask) + __popc(high_mask);
  __syncthreads();
  int given;
  const int before_mask = scan_before(t < masks ? ranks[t] : 0, slots, given);
  if (t < masks) ranks[t] = before_mask;
  __syncthreads();
  const int rank_of = lane < rounds ? ranks[lane * kWaves + wave] : 0;
  for (int i = 0; i < rounds; ++i) {
    const unsigned long long free =
        static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_readlane(high_mask, i))) << 32 |
        static_cast<unsigned>(__builtin_amdgcn_readlane(low_mask, i));
    const int first_rank = __builtin_amdgcn_readlane(rank_of, i);
    if (first_rank >= total) break;
    const int rank = first_rank + __popcll(free & ((1ull << lane) - 1));
    if ((free >> lane & 1) && rank < total) {
      int low = 0, high = s.sequences - 1;  // the last sequence whose first rank is at most this one
      while (low < high) {
        const int middle = high - (high - low) / 2;
        if (base[middle] <= rank) low = middle;
        else high = middle - 1;
      }
      const int of = i * kAdvanceThreads + t, at = rank - base[low];
      s.tables_out[static_cast<size_t>(low) * s.max_pages + entry[low] + at] = of;
      if (at == 0) fresh[low] = of;
      uses[of] = 1;
    }
  }
  __syncthreads();
  if (is) {
    const bool copied = replaced && fresh[t] >= 0;
    if (replaced && !copied) s.tables_out[static_cast<size_t>(t) * s.max_pages + first - 1] = -1;
    s.copies[2 * t] = copied ? page : -1;
    s.copies[2 * t + 1] = copied ? fresh[t] : -1;
    s.lengths_out[t] = length + n;
  }
  for (int i = t; i < s.pages; i += kAdvanceThreads) s.uses[i] = uses[i];
  constexpr unsigned long long kMost = INT_MAX;
  if (t == 0) *s.shortage = static_cast<int>(min(max(total - given, 0) + beyond, kMost));
}

// ---------------------------------------------------------------------------
// copy

constexpr int kCopyThreads = 256;

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// Part `blockIdx.x % parts` of pair blockIdx.x / parts in group blockIdx.y: columns of 16 bytes, and of
// one byte for what is left of the page. Bound by memory: about 160 pairs of 4 x 8 KB (10 MB read and written) 4.2
// us, a few 1 to 2.6.
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(unsigned char *cache, const int *__restrict__ copies,
                                                            int pages, unsigned parts, unsigned wide, unsigned columns,
                                                            long long group_stride, long long page_stride) {
  const unsigned pair = blockIdx.x / parts, part = blockIdx.x - pair * parts;
  const int from = copies[2 * static_cast<size_t>(pair)], to = copies[2 * static_cast<size_t>(pair) + 1];
  if (static_cast<unsigned>(from) >= static_cast<unsigned>(pages) ||
      static_cast<unsigned>(to) >= static_cast<unsigned>(pages) || from == to)
    return;
  const unsigned c = part * kCopyThreads + threadIdx.x;
  if (c >= columns) return;
  cache += blockIdx.y * group_stride;
  const unsigned char *const src = cache + from * page_stride;
  unsigned char *const dst = cache + to * page_stride;
  if (c < wide) *reinterpret_cast<u32x4_any *>(dst + 16LL * c) = *reinterpret_cast<const u32x4_any *>(src + 16LL * c);
  else dst[16LL * wide + (c - wide)] = src[16LL * wide + (c - wide)];
}

}  // namespace

extern "C" int l2c_cache_append(void *keys, void *values, float *key_scales, float *value_scales, int cache_type,
                                const uint16_t *k, long long k_stride, const uint16_t *v, long long v_stride,
                                const int *tables, const int *lengths, const int *starts, int sequences, int rows,
                                int kv_heads, int width, int page_size, int pages, int max_pages, hipStream_t stream) {
  if (!l2c::cache_sizes(cache_type, sequences, rows, kv_heads, width, page_size, pages, max_pages))
    return hipErrorInvalidValue;
  const long long row = static_cast<long long>(kv_heads) * width;
  if (k_stride < row || v_stride < row || k_stride % 8 != 0 || v_stride % 8 != 0) return hipErrorInvalidValue;
  if (sequences == 0 || rows == 0 || pages == 0 || max_pages == 0) return hipSuccess;
  if (!l2c::cache_arguments(cache_type, keys, values, key_scales, value_scales, tables, lengths, starts, sequences,
                            rows, pages, max_pages) ||
      !k || !v || !l2c_aligned16(k) || !l2c_aligned16(v))
    return hipErrorInvalidValue;
  const int lanes = width <= 64 ? 8 : width <= 128 ? 16 : 32;
  // Four items a lane where that leaves some workgroups for every CU.
  const long long items = 2LL * kv_heads * rows;
  const bool many = items * lanes >= 4LL * 4 * 256 * kAppendThreads;
  const long long block = kAppendThreads / lanes * (many ? 4 : 1), blocks = (items + block - 1) / block;
  if (items > INT_MAX - kAppendThreads || !l2c::launchable(blocks, kAppendThreads)) return hipErrorInvalidValue;
  const l2c::Sequences s =
      l2c::sequences_of(tables, lengths, starts, sequences, rows, max_pages, page_size, pages);
  const AppendKernel fn = lanes == 8    ? append_of<8>(many, cache_type == L2C_E4M3)
                          : lanes == 16 ? append_of<16>(many, cache_type == L2C_E4M3)
                                        : append_of<32>(many, cache_type == L2C_E4M3);
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0, stream, keys, values, key_scales,
                     value_scales, k, k_stride, v, v_stride, s, kv_heads, width, l2c::Quotient31(2 * kv_heads));
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

extern "C" int l2c_cache_advance(int *tables_out, int *lengths_out, int *uses, int *copies, int *shortage,
                                 const int *tables, const int *lengths, const int *parents, int beams,
                                 const int *starts, const int *held, int sequences, int page_size, int pages,
                                 int max_pages, int window, hipStream_t stream) {
  if (sequences < 0 || page_size <= 0 || pages < 0 || max_pages < 0 || window < 0 ||
      static_cast<long long>(max_pages) * page_size > l2c::kMostPositions ||
      (parents && (beams <= 0 || sequences % beams != 0)))
    return hipErrorInvalidValue;
  if (sequences == 0) return hipSuccess;
  if (!lengths_out || !copies || !shortage || !lengths || (pages > 0 && !uses) ||
      (max_pages > 0 && (!tables_out || !tables)) || (parents && (tables_out == tables || lengths_out == lengths)) ||
      !l2c::launchable(sequences, 256))
    return hipErrorInvalidValue;
  const Step s = {tables_out, lengths_out, uses, copies, shortage, tables, lengths, parents, starts, held,
                  beams, sequences, pages, max_pages, page_size, window};
  const long long entries = static_cast<long long>(sequences) * max_pages;
  if (sequences <= kLdsSequences && pages <= kLdsPages && entries <= kLdsEntries) {
    const bool copy = entries <= kCopyEntries;
    if (!copy) {
      hipLaunchKernelGGL(advance_tables_kernel<false>, dim3(sequences), dim3(256), 0, stream, s);
      L2C_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(copy ? advance_lds_kernel<true> : advance_lds_kernel<false>, dim3(1), dim3(kAdvanceThreads), 0,
                       stream, s);
    L2C_LAUNCH_CHECK();
    return hipSuccess;
  }
  hipLaunchKernelGGL(advance_tables_kernel<true>, dim3(sequences), dim3(256), 0, stream, s);
  L2C_LAUNCH_CHECK();
  hipLaunchKernelGGL(advance_count_kernel, dim3(sequences), dim3(256), 0, stream, s);
  L2C_LAUNCH_CHECK();
  hipLaunchKernelGGL(advance_assign_kernel, dim3(1), dim3(kAdvanceThreads), 0, stream, s);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

extern "C" int l2c_cache_copy(void *cache, const int *copies, int count, int pages, int groups, long long group_stride,
                              long long page_stride, long long page_bytes, hipStream_t stream) {
  if (count < 0 || pages < 0 || groups < 0 || page_bytes < 0) return hipErrorInvalidValue;
  if (count == 0 || pages == 0 || groups == 0 || page_bytes == 0) return hipSuccess;
  if (!cache || !copies) return hipErrorInvalidValue;
  // Pages and groups follow each other without overlap, within 63 bits.
  typedef __int128 wide_t;
  const wide_t group = static_cast<wide_t>(pages - 1) * page_stride + page_bytes;
  const wide_t span = static_cast<wide_t>(groups - 1) * group_stride + group;
  if ((pages > 1 && page_stride < page_bytes) || (groups > 1 && group_stride < group) || span > LLONG_MAX)
    return hipErrorInvalidValue;
  const long long wide = page_bytes / 16, columns = wide + page_bytes % 16;
  if (columns > INT_MAX) return hipErrorInvalidValue;
  const long long parts = (columns + kCopyThreads - 1) / kCopyThreads;
  // As many pairs and groups a launch as HIP takes; no more than some hundred launches for it.
  constexpr long long kGridY = 65535, kMostBlocks = 0xffffffffLL / kCopyThreads, kMostWork = 1LL << 31;
  const long long pairs = min(static_cast<long long>(count), kMostBlocks / parts);
  if (pairs == 0) return hipErrorInvalidValue;
  const long long deep = min(kGridY, kMostBlocks / (parts * pairs));
  if ((pairs < count || deep < kGridY) && parts * count > kMostWork / groups) return hipErrorInvalidValue;
  for (long long group = 0; group < groups; group += deep)
    for (long long pair = 0; pair < count; pair += pairs) {
      const dim3 grid(static_cast<unsigned>(parts * min(pairs, count - pair)),
                      static_cast<unsigned>(min(deep, groups - group)));
      hipLaunchKernelGGL(copy_kernel, grid, dim3(kCopyThreads), 0, stream,
                         static_cast<unsigned char *>(cache) + group * group_stride, copies + 2 * pair, pages,
                         static_cast<unsigned>(parts), static_cast<unsigned>(wide), static_cast<unsigned>(columns),
                         group_stride, page_stride);
      L2C_LAUNCH_CHECK();
    }
  return hipSuccess;
}

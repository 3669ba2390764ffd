// Attention of new tokens over a cache in pages (include/l2c.h has the formula).
//
// The rows of a tile are (token, query head of one key head) pairs, packed token by token: all of
// them read the same keys and values, once. One pass over the positions, with the running maximum m
// and sum l of a softmax in base 2: with S = scale log2(e) q.k and p = 2^(S - m), a larger maximum m'
// multiplies l and the sum of p v by 2^(m - m').
//
// Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T: a lane of the matrix
// instructions' results then has one query and several positions, so that maxima and sums run
// within lanes, and p is in the lanes and the order in which the second product wants it as an
// operand; only V has to be transposed, which the LDS does as it is read.
#include <type_traits>

#include "l2c_cache.h"

namespace {

using l2c::Sequences;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / L2C_WAVE;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kSlack = 8.0f;

__device__ const u32x4 zero_row[L2C_MAX_HEAD / 8] = {};  // of a position without a page

struct Attention {
  uint16_t *out;
  const uint16_t *q;
  const void *keys, *values;
  const float *key_scales, *value_scales;
  float *part_values;  // [row][head][split][width]
  float2 *part_sums;   // [row][head][split]: maximum and sum
  long long out_stride, q_stride;
  Sequences s;
  l2c::Quotient31 by_group;
  int heads, kv_heads, group, width, window, splits, slots, least;
  unsigned long long page_rows;  // of all heads
  float scale;                   // times log2(e)
};

// ---------------------------------------------------------------------------
// Which rows and positions a workgroup has.

struct Tile {
  int sequence, first, count;  // packed rows first .. first + count - 1 of the sequence's new tokens
  int start;                   // row of its first new token
  long long before;            // position of that
  int from, end;               // positions that any row of the tile sees
  int begin;                   // the last multiple of the step up to the first of them
  int chunk, parts;            // positions a part, parts that are not empty (at least 1)

  __device__ __forceinline__ int position(const Attention &a, int packed) const {  // -1: none
    const long long p = before + a.by_group(packed);
    return p < -1 ? -1 : p > INT_MAX ? INT_MAX : static_cast<int>(p);
  }
  __device__ __forceinline__ int row(const Attention &a, int packed) const { return start + a.by_group(packed); }
  __device__ __forceinline__ int head(const Attention &a, int kv, int packed) const {
    return kv * a.group + (packed - a.by_group(packed) * a.group);
  }
};

// The parts of a tile's positions: no shorter than a.least, in whole STEPs from the first one's.
template <int STEP>
__device__ __forceinline__ void divide(const Attention &a, Tile &t) {
  const int last = t.position(a, t.first + t.count - 1), low = t.position(a, t.first);
  t.end = min(last, a.s.capacity() - 1) + 1;
  t.from = a.window ? max(0, low - a.window + 1) : 0;
  t.begin = t.from / STEP * STEP;
  const int n = max(0, t.end - t.begin);
  const int each = (n + a.splits - 1) / a.splits;
  t.chunk = max((each + STEP - 1) / STEP * STEP, a.least);
  t.parts = max(1, (n + t.chunk - 1) / t.chunk);
}

// Tile `slot` of all. With starts sequence s has the slots from starts[s] group / M + s on, enough of
// them for its rows: some are empty, but where they begin needs no sum over the sequences before.
template <int M>
__device__ __forceinline__ bool tile_of(const Attention &a, int slot, Tile &t) {
  int n;
  if (!a.s.starts) {
    const int each = (a.group + M - 1) / M;
    t.sequence = slot / each;
    t.first = (slot - t.sequence * each) * M;
    t.start = t.sequence;
    t.before = static_cast<long long>(a.s.lengths[t.sequence]) - 1;
    n = a.group;
  } else {
    // The last sequence whose slots begin at or before this one: the lanes look at 64 at a time.
    const int lane = threadIdx.x % L2C_WAVE;
    int low = 0, count = a.s.sequences;
    while (true) {
      const int each = (count + L2C_WAVE - 1) / L2C_WAVE, s = low + lane * each;
      bool reached = false;
      if (lane * each < count)
        reached = static_cast<long long>(a.s.starts[s]) * a.group / M + s <= slot;
      const int reaches = __popcll(__ballot(reached));
      if (reaches > 1) low += (reaches - 1) * each;
      if (each == 1) break;
      count = min(each, a.s.sequences - low);
    }
    t.sequence = __builtin_amdgcn_readfirstlane(low);
    const int from = a.s.starts[t.sequence], to = a.s.starts[t.sequence + 1];
    const long long tile = slot - (static_cast<long long>(from) * a.group / M + t.sequence);
    // Of starts that are not in order any answer will do, within the arrays.
    if (from < 0 || to > a.s.rows || from >= to || tile < 0) return false;
    const long long packed = static_cast<long long>(to - from) * a.group;
    if (packed > INT_MAX || tile * M >= packed) return false;
    n = static_cast<int>(packed);
    t.first = static_cast<int>(tile) * M;
    t.start = from;
    t.before = static_cast<long long>(a.s.lengths[t.sequence]) - (to - from);
  }
  t.count = min(M, n - t.first);
  return true;
}

// The same with the tiles in the order of what they have to do, the most first: that of their sequences'
// lengths, and of a sequence its last tile first. For up to 64 sequences, a lane each; the tiles of many are
// in the order of the sequences, from the last. (Of three chunks of 750 to 1000 tokens over 3100 to 5000
// positions, 680 workgroups for 512 places, the longest began last.)
template <int M>
__device__ __forceinline__ bool longest_tile_of(const Attention &a, int slot, Tile &t) {
  if (!a.s.starts || a.s.sequences > L2C_WAVE) return tile_of<M>(a, a.slots - 1 - slot, t);
  const int s = threadIdx.x % L2C_WAVE;
  int from = 0, packed = 0, length = 0, tiles = 0;
  if (s < a.s.sequences) {
    from = a.s.starts[s];
    const int to = a.s.starts[s + 1];
    length = a.s.lengths[s];
    // Of starts that are not in order any answer will do, within the arrays.
    if (from >= 0 && to <= a.s.rows && from < to) packed = (to - from) * a.group, tiles = (packed + M - 1) / M;
  }
  int before = 0;  // tiles of longer sequences
  for (int o = 0; o < a.s.sequences; ++o) {
    const int other = __builtin_amdgcn_readlane(length, o), its = __builtin_amdgcn_readlane(tiles, o);
    before += other > length || (other == length && o < s) ? its : 0;
  }
  const unsigned long long here = __ballot(slot >= before && slot < before + tiles);
  if (here == 0) return false;
  const int lane = __ffsll(here) - 1;
  t.sequence = lane;
  t.start = __builtin_amdgcn_readlane(from, lane);
  packed = __builtin_amdgcn_readlane(packed, lane);
  t.before = static_cast<long long>(__builtin_amdgcn_readlane(length, lane)) - packed / a.group;
  t.first = (__builtin_amdgcn_readlane(tiles, lane) - 1 - (slot - __builtin_amdgcn_readlane(before, lane))) * M;
  t.count = min(M, packed - t.first);
  return true;
}

// ---------------------------------------------------------------------------
// Pieces.

__device__ __forceinline__ unsigned pack2(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}

// A weight as the sum of two bf16 numbers: its upper 16 bits, which are no larger, and the bf16 of what they leave, to
// 2^-15 of it together. 2^-20 of the weight is added to the second: it has the weight's sign even where the first is
// the whole of it, so that both times an infinity are the same infinity. BOUNDED: of a weight that is no infinity.
__device__ __forceinline__ float upper(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ unsigned pack_upper(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
template <bool BOUNDED>
__device__ __forceinline__ float lower(float v) {
  const float left = v - upper(v);  // NaN of an infinity, for which any other number does
  return fmaf(v, 0x1p-20f, BOUNDED ? left : fmaxf(left, -FLT_MAX));
}

// Eight e4m3 codes as bf16, exactly.
__device__ __forceinline__ u32x4 widen(u32x2 c) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.0f, false));
    v[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.0f, true));
  }
  return v;
}

template <bool E4M3>
using Raw = std::conditional_t<E4M3, u32x2, u32x4>;

// Eight cached values as they lie there, and as bf16.
template <bool E4M3>
__device__ __forceinline__ Raw<E4M3> load_raw(const void *cache, size_t at) {
  if constexpr (E4M3) return *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(cache) + at);
  else return *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(cache) + at);
}
__device__ __forceinline__ u32x4 as_bf16(u32x2 c) { return widen(c); }
__device__ __forceinline__ u32x4 as_bf16(u32x4 c) { return c; }

__device__ __forceinline__ bool not_finite(u32x4 v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}
__device__ __forceinline__ bool not_finite(float v) { return !(fabsf(v) <= FLT_MAX); }
// 0 in the place of those that are not.
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((v[i] & 0x7f80u) == 0x7f80u) v[i] &= 0xffff0000u;
    if ((v[i] & 0x7f800000u) == 0x7f800000u) v[i] &= 0xffffu;
  }
  return v;
}

// Four cached values from an index on, a multiple of four, as they are without a scale.
template <bool E4M3>
__device__ __forceinline__ f32x4 load4(const void *cache, size_t at) {
  if constexpr (E4M3) {
    const unsigned c = *reinterpret_cast<const unsigned *>(static_cast<const uint8_t *>(cache) + at);
    const bf16x2 low = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false);
    const bf16x2 high = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true);
    return f32x4{static_cast<float>(low[0]), static_cast<float>(low[1]), static_cast<float>(high[0]),
                 static_cast<float>(high[1])};
  } else {
    const u32x2 v = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(cache) + at);
    return f32x4{__uint_as_float(v[0] << 16), __uint_as_float(v[0] & 0xffff0000u), __uint_as_float(v[1] << 16),
                 __uint_as_float(v[1] & 0xffff0000u)};
  }
}

// Which of 32 positions in a row a row sees: those with a page, up to the `to`-th, after the `from`-th.
__device__ __forceinline__ unsigned seen_of_32(unsigned there, int to, int from) {
  const unsigned upto = to < 0 ? 0u : to >= 31 ? ~0u : (2u << to) - 1u;
  const unsigned behind = from < 0 ? 0u : from >= 31 ? ~0u : (2u << from) - 1u;
  return there & upto & ~behind;
}

// Values across lanes without a trip through LDS: of both lanes that differ in bit 5, or bit 4.
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_rows(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_rows(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }

// What is stored for `head` of `row`: the result, or one part of it.
__device__ __forceinline__ size_t part_of(const Attention &a, int row, int head, int split) {
  return (static_cast<size_t>(row) * a.heads + head) * a.splits + split;
}
__device__ __forceinline__ float inverse(float total) { return total == 0.0f ? 0.0f : 1.0f / total; }

// Four values of a row's head, from column d on.
__device__ __forceinline__ void store4(const Attention &a, bool whole, int row, int head, int split, int d, f32x4 v) {
  if (whole) {
    const u32x2 packed = {pack2(v[0], v[1]), pack2(v[2], v[3])};
    *reinterpret_cast<u32x2 *>(a.out + row * a.out_stride + static_cast<size_t>(head) * a.width + d) = packed;
  } else {
    *reinterpret_cast<f32x4 *>(a.part_values + part_of(a, row, head, split) * a.width + d) = v;
  }
}

__device__ __forceinline__ float dot8(u32x4 x, u32x4 y, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), sum);
    sum = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), sum);
  }
  return sum;
}

// Values that are not finite, in steps of positions that some rows of a tile see and others do not: in the product they
// would be NaN times the weight 0 of those, so their places have 0 there, and afterwards the rows that see them get
// them here. A wave goes through its steps of KEYS positions from `base` on; add(row, j) for each position j that has
// such a value, or, SCALED, such a scale, and its row in the cache. After all steps, since the registers for it are
// free then: one infinity in 4096 over 16384 positions 1030 us, 960 without; computed beside the products it spilled
// others, 1740.
template <int KEYS, bool E4M3, bool SCALED, class Add>
__device__ __forceinline__ void odd_positions(const Attention &a, const Tile &t, int kv, int base, int stride, int end,
                                              int every, int nobody, Add add) {
  const int lane = threadIdx.x % L2C_WAVE;
  for (; base < end; base += stride) {
    if (base + KEYS - 1 <= every && base > nobody) continue;
    const int j = base + lane;
    bool is = false;
    size_t at = 0;
    if (lane < KEYS && j >= t.from && j < end) {
      const int index = a.s.by_page(j), page = a.s.page(t.sequence, index);
      if (a.s.is_page(page)) {
        at = (static_cast<size_t>(page) * a.kv_heads + kv) * a.s.page_size + (j - index * a.s.page_size);
        if constexpr (SCALED) is = not_finite(a.value_scales[at]);
        for (int d = 0; d < a.width; d += 8) is |= not_finite(as_bf16(load_raw<E4M3>(a.values, at * a.width + d)));
      }
    }
    const unsigned low = static_cast<unsigned>(at), high = static_cast<unsigned>(at >> 32);
    for (unsigned long long odd = __ballot(is); odd; odd &= odd - 1) {
      const int key = __builtin_ctzll(odd);
      const unsigned long long above = static_cast<unsigned>(__builtin_amdgcn_readlane(high, key));
      add(static_cast<size_t>(above << 32 | static_cast<unsigned>(__builtin_amdgcn_readlane(low, key))), base + key);
    }
  }
}

typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

// Four keys of a column: lanes l of 16 point to keys l / 4 and columns 4 (l % 4), and get column l.
__device__ __forceinline__ u32x2 read_column(const uint16_t *at) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (lds_i16x4 *)(const __attribute__((address_space(3))) uint16_t *)at));
}

// ---------------------------------------------------------------------------
// Tiles of up to 16 rows: a step of decoding. Bound by the cache's bytes. The four waves
// of a workgroup go through positions of their own, 32 at a time, and join at the end. Keys go from
// memory to the matrix instructions' operands (16 x 16 x 32: a lane has eight values of one
// key), values through LDS of the wave's own, so that nothing waits for another wave.

constexpr int kNarrow = 16, kNarrowStep = 32;

// Where 16 bytes (`chunk`) of row `key` lie in a wave's values in LDS. Lanes that write together have sixteen keys
// and one chunk, lanes that read together the same 32 bytes of eight keys: chunks are exchanged so that
// neither meet in a bank.
template <int D>
__device__ __forceinline__ int value_place(int key, int chunk) {
  return key * D + 8 * (chunk ^ ((D == 64 ? key >> 1 & 3 : key & 7) << 1 | (key >> 3 & 1)));
}

// kChunks: of 32 columns, of which a lane has eight; those from kSure on may end before. A row has D columns in LDS.
// PAIRS: of e4m3 pages a lane has sixteen columns in a row for two chunks, so that it loads 16 bytes at a time, too (4
// x 131072 in e4m3 158 us, 5.2 TB/s; when eight took 215, that was as long as without any arithmetic; rows of an odd
// number of eights are loaded so). 64 x 4096 in bf16 takes 153 us, 4.9 TB/s; 16 x 5 of 2500, 80 wide, 18.7, of which
// the kernel 14.5 and the join 4.2. Three waves a SIMD up to 128 columns (64 x 4 over 1000 in bf16 82 us, 90 with two),
// four up to 64.
//
// The weights are two bf16 numbers each, and the second product is taken of both: the matrix units have the time (busy
// 4 to 7% of it with one number, 6 to 12 with two). With one and with two numbers, us: 153.7 and 153.3 (64 x 4096),
// 117.6 and 111.4 (64 x 4096 in e4m3), 18.3 and 18.7 (16 x 5 of 2500), 10.8 and 11.0 (1 x 2048), 30.6 and 32.7 (16 x 8
// of 3000, 64 wide, in e4m3). Rounded to one, a weight would be off by up to 2^-8 of it.
template <int kChunks, bool E4M3, bool PAIRS>
__global__ __launch_bounds__(kThreads, kChunks > 4 ? 1 : kChunks == 2 ? 4 : 3) void narrow_kernel(Attention a) {
  static_assert(!PAIRS || kChunks % 2 == 0, "two chunks a load");
  constexpr int kSure = PAIRS ? kChunks - 2 : kChunks == 2 ? 0 : kChunks <= 4 ? kChunks - 1 : kChunks - 2;
  constexpr int D = kChunks <= 2 ? 64 : kChunks <= 4 ? 128 : 256;
  constexpr int kTiles = 2 * kChunks;  // of columns
  constexpr int kApart = 68;       // floats from row to row of the join
  constexpr int kValues = D == 64 ? 2 * kNarrow * kApart : kNarrowStep * D;
  __shared__ __attribute__((aligned(16))) uint16_t values[kWaves][kValues];
  __shared__ float tops[kWaves][kNarrow], sums[kWaves][kNarrow];
  const int lane = threadIdx.x % L2C_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int n = lane % 16, g = lane / 16;
  int block = blockIdx.x;
  const int kv = block % a.kv_heads;
  block /= a.kv_heads;
  const int split = block % a.splits;
  Tile t;
  if (!tile_of<kNarrow>(a, block / a.splits, t)) return;
  divide<kNarrowStep>(a, t);
  if (split >= t.parts) return;
  const int begin = t.begin + split * t.chunk, end = min(t.end, begin + t.chunk);
  const bool mine = n < t.count;
  const int packed = t.first + (mine ? n : 0);
  const int row = t.row(a, packed), head = t.head(a, kv, packed);
  const int position = mine ? t.position(a, packed) : -1;
  const int lowest = a.window ? max(-1, position - a.window) : -1;  // it sees those above
  const int every = t.position(a, t.first);                // all rows see positions up to this one
  const unsigned long long head_rows = static_cast<unsigned long long>(kv) * a.s.page_size;
  const int nobody = a.window ? t.position(a, t.first + t.count - 1) - a.window : -1;  // and those above this one

  // The scale's sign goes to the queries, and 0 is the least number instead, so that the largest of the products
  // is the largest score, and -Inf stays that.
  const float scale = fmaxf(fabsf(a.scale), FLT_MIN);
  auto column = [&](int c) __attribute__((always_inline)) {  // the lane's first of a chunk
    return PAIRS ? 64 * (c / 2) + 16 * g + 8 * (c % 2) : 32 * c + 8 * g;
  };
  bf16x8 q[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int d = column(c);
    u32x4 v = {0, 0, 0, 0};
    if (mine && d < a.width)
      v = *reinterpret_cast<const u32x4 *>(a.q + row * a.q_stride + static_cast<size_t>(head) * a.width + d);
    if (a.scale < 0.0f) v ^= 0x80008000u;
    q[c] = __builtin_bit_cast(bf16x8, v);
  }

  // The pages of a step's keys n and 16 + n.
  auto look_up = [&](int (&page)[2], int base) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = base + 16 * u + n;
      page[u] = j < end ? a.s.page(t.sequence, a.s.by_page(j)) : -1;
    }
  };
  // Where a key's row lies.
  auto row_of = [&](int page, int j) __attribute__((always_inline)) {
    return static_cast<unsigned long long>(static_cast<unsigned>(page)) * a.page_rows + head_rows +
           static_cast<unsigned>(j - a.s.by_page(j) * a.s.page_size);
  };
  Raw<E4M3> k[2][kChunks], v[2][kChunks];
  f32x4 key_scale[2], value_scale[2];  // of keys 4 g + i, which the lane has scores of
  unsigned there;                      // keys with a page that some row sees
  const bool fours = a.s.page_size % 4 == 0;  // four keys from a multiple of four on lie in one page
  // The lane's part of a chunk is inside the row.
  auto inside = [&](int c) __attribute__((always_inline)) { return c < kSure || column(c) < a.width; };
  auto load = [&](const int (&page)[2], int base) __attribute__((always_inline)) {
    const bool seen[2] = {a.s.is_page(page[0]) && base + n >= t.from, a.s.is_page(page[1]) && base + 16 + n >= t.from};
    there = (static_cast<unsigned>(__ballot(seen[0])) & 0xffffu) | static_cast<unsigned>(__ballot(seen[1])) << 16;
    typedef std::conditional_t<E4M3, uint8_t, uint16_t> Element;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool is = seen[u];
      const unsigned long long of = row_of(page[u], base + 16 * u + n), at = of * a.width;
      // Of a key without a page zeros; past the row's end its beginning, which becomes zeros, or ends in columns
      // that nobody stores.
      const Element *const none = reinterpret_cast<const Element *>(zero_row);
      const Element *const key = is ? static_cast<const Element *>(a.keys) + at : none;
      const Element *const value = is ? static_cast<const Element *>(a.values) + at : none;
#pragma unroll
      for (int c = 0; c < kChunks; c += PAIRS ? 2 : 1) {
        const int from = inside(c) ? column(c) : 0;
        if constexpr (PAIRS) {
          const u32x4 x = *reinterpret_cast<const u32x4 *>(key + from);
          const u32x4 y = *reinterpret_cast<const u32x4 *>(value + from);
          k[u][c] = u32x2{x[0], x[1]}, k[u][c + 1] = u32x2{x[2], x[3]};
          v[u][c] = u32x2{y[0], y[1]}, v[u][c + 1] = u32x2{y[2], y[3]};
        } else {
          k[u][c] = *reinterpret_cast<const Raw<E4M3> *>(key + from);
          v[u][c] = *reinterpret_cast<const Raw<E4M3> *>(value + from);
        }
      }
      if constexpr (E4M3) {
        const float *const zero = reinterpret_cast<const float *>(zero_row);
        if (fours) {
          const int page_of_four = __shfl(page[u], 4 * g, L2C_WAVE);
          const unsigned long long four = row_of(page_of_four, base + 16 * u + 4 * g);
          const bool are = a.s.is_page(page_of_four);
          key_scale[u] = *reinterpret_cast<const f32x4_any *>(are ? a.key_scales + four : zero);
          value_scale[u] = *reinterpret_cast<const f32x4_any *>(are ? a.value_scales + four : zero);
        } else {
          const float x = *(is ? a.key_scales + of : zero), y = *(is ? a.value_scales + of : zero);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            key_scale[u][i] = __shfl(x, 4 * g + i, L2C_WAVE);
            value_scale[u][i] = __shfl(y, 4 * g + i, L2C_WAVE);
          }
        }
      }
    }
  };

  constexpr int kStride = kWaves * kNarrowStep;
  f32x4 acc[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float top = -INFINITY, total = 0.0f;  // of the products, without the scale
  bool odd = false;                     // there were values for odd_positions()
  uint16_t *const mine_values = values[wave];
  // Where the lane writes its first chunk of key n, and reads keys 4 g + n / 4 of the first tile of columns.
  int to_place = value_place<D>(n, PAIRS ? 2 * g : g);
  int from_place = value_place<D>(4 * g + n / 4, n % 4 / 2) + 4 * (n % 2);
  int base = begin + wave * kNarrowStep;
  int page[2];
  look_up(page, base);
  load(page, base);
  look_up(page, base + kStride);
  for (; base < end; base += kStride) {
    // Products of keys 4 g + i of both halves with query n.
    f32x4 s[2], factor[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        u32x4 x = as_bf16(k[u][c]);
        if (!inside(c)) x = u32x4{0, 0, 0, 0};  // q's zeros alone would make NaN of an infinity
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), q[c], s[u], 0, 0, 0);
      }
      if constexpr (E4M3) s[u] *= key_scale[u], factor[u] = value_scale[u];
    }
    const bool mixed = base + kNarrowStep - 1 > every || base <= nobody;
    if (mixed || there != 0xffffffffu) {
      const unsigned seen = seen_of_32(there, position - base, lowest - base);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(seen >> (16 * u + 4 * g + i) & 1)) {
            s[u][i] = -INFINITY;
            if constexpr (E4M3) factor[u][i] = 0.0f;  // a scale beside those that the row sees may be anything
          }
    }
    // Values into LDS; where some rows see them and others do not, 0 in the place of those that are not finite.
    bool bad = false;
    // The places differ by bits of their own from chunk to chunk: found anew in every step, not kept in registers.
    asm volatile("" : "+v"(to_place));
    auto place = [&](int u, int c) __attribute__((always_inline)) {
      const int chunk = PAIRS ? 8 * (c / 2) + c % 2 : 4 * c;
      return reinterpret_cast<u32x4 *>(mine_values + (to_place ^ 8 * chunk) + 16 * D * u);
    };
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const u32x4 w = as_bf16(v[u][c]);
        if (mixed) bad |= not_finite(w);
        *place(u, c) = w;
      }
    if (mixed && __ballot(bad)) {
      odd = true;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          *place(u, c) = finite_part(as_bf16(v[u][c]));
    }
    // The next step's, before anything waits for this one's.
    load(page, base + kStride);
    look_up(page, base + 2 * kStride);
    float most = top;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, s[u][i]);
    most = max_halves(max_rows(most));
    // Sums stay relative to an older maximum until a new one is more than 2^kSlack times as large. Weights are
    // 2^-kSlack of the softmax's, so that none is above 1 and large values do not overflow.
    if (__ballot((most - top) * scale > kSlack)) {
      const float again = top == -INFINITY ? 0.0f : exp2_of((top - most) * scale);
      total *= again;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) acc[i] *= again;
      top = most;
    }
    const float shift = top == -INFINITY ? 0.0f : fmaf(top, scale, kSlack);
    u32x4 p, rest;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float e[4], left[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = exp2_of(fmaf(s[u][i], scale, -shift));
        total += e[i];
        if constexpr (E4M3) e[i] *= factor[u][i];
        left[i] = lower<!E4M3>(e[i]);
      }
      p[2 * u] = pack_upper(e[0], e[1]), p[2 * u + 1] = pack_upper(e[2], e[3]);
      rest[2 * u] = pack2(left[0], left[1]), rest[2 * u + 1] = pack2(left[2], left[3]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" : "+v"(from_place));
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const uint16_t *const from = mine_values + (from_place ^ 16 * i);
      const u32x2 low = read_column(from), high = read_column(from + 16 * D);
      const u32x4 w = {low[0], low[1], high[0], high[1]};
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, p),
                                                       acc[i], 0, 0, 0);
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, rest),
                                                       acc[i], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  if (top > -INFINITY) top = fmaf(top, scale, kSlack);  // what its sums are relative to
  if (odd)
    odd_positions<kNarrowStep, E4M3, false>(
        a, t, kv, begin + wave * kNarrowStep, kStride, end, every, nobody, [&](size_t at, int j) {
          float score = 0.0f;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            if (inside(c))
              score = dot8(as_bf16(load_raw<E4M3>(a.keys, at * a.width + column(c))),
                           __builtin_bit_cast(u32x4, q[c]), score);
          score = sum_halves(sum_rows(score));
          if constexpr (E4M3) score *= a.key_scales[at];
          float weight = exp2_of(fmaf(score, scale, top > -INFINITY ? -top : 0.0f));
          if constexpr (E4M3) weight *= a.value_scales[at];
          const bool sees = j <= position && j > lowest;
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            const int d = 16 * i + 4 * g;
            const f32x4 x = load4<E4M3>(a.values, at * a.width + (d < a.width ? d : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] += sees && not_finite(x[e]) ? weight * x[e] : 0.0f;
          }
        });
  total = sum_halves(sum_rows(total));
  if (g == 0) tops[wave][n] = top, sums[wave][n] = total;
  __syncthreads();
  float most = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) most = fmaxf(most, tops[w][n]);
  const float shift = most == -INFINITY ? 0.0f : most;
  float all = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += sums[w][n] * exp2_of(tops[w][n] - shift);
  const bool whole = t.parts == 1;
  const float by = exp2_of(top - shift) * (whole ? inverse(all) : 1.0f);
  // The waves' sums by way of LDS, 64 columns at a time.
  float *const shared = reinterpret_cast<float *>(&values[0][0]);
#pragma unroll
  for (int part = 0; part < (kTiles + 3) / 4; ++part) {
    if (part > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * part + i < kTiles)
        *reinterpret_cast<f32x4 *>(shared + (wave * kNarrow + n) * kApart + 16 * i + 4 * g) = acc[4 * part + i] * by;
    __syncthreads();
    // 16 rows of 64 columns by 256 lanes.
    const int r = threadIdx.x / 16, c = 4 * (threadIdx.x % 16), d = 64 * part + c;
    if (r < t.count && d < a.width) {
      f32x4 sum = *reinterpret_cast<const f32x4 *>(shared + r * kApart + c);
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
        sum += *reinterpret_cast<const f32x4 *>(shared + (w * kNarrow + r) * kApart + c);
      store4(a, whole, t.row(a, t.first + r), t.head(a, kv, t.first + r), split, d, sum);
    }
  }
  if (!whole && wave == 0 && g == 0 && mine) a.part_sums[part_of(a, row, head, split)] = make_float2(most, all);
}

// ---------------------------------------------------------------------------
// Tiles of 32 rows a wave: chunks of a prompt. Bound by the matrix and the vector units, and by LDS, which each wave
// reads whole tiles from. The workgroup's keys and values, 64 positions at a time, lie in LDS, two tiles of them: while
// one is read, the next is on its way. bf16 pages go to LDS without registers between, rows that are not there from a
// row of zeros; e4m3 pages through registers, where they become bf16 (a chunk each of 2000 over up to 4000 positions of
// 8 sequences 648 us, 548 in bf16; two tiles in LDS here, too, 676: they cost registers). Of more than 128 columns a
// tile of 64 positions needs all 512 registers and 128 KB, and is still better than one of 32 (200 over 10000
// positions, 256 wide, 116 us and 130; 192 wide, 1000 over 4000 of 4, 139 and 157). Four waves share a tile, so that
// two workgroups fit a CU, or eight, for which half as much is loaded (a chunk of 4096 over 16384 positions 880 to 940
// us, 982 with four; three of 1000 over 5000 209 and 223), where 128 columns make that worth it and the tiles are
// enough (four chunks of 300 over 2000 57 us with four, 64 with eight; 64 columns the same with both). Four waves of
// more than 128 columns need the registers of eight.
//
// The weights are rounded to bf16, by up to 2^-8 of each, as operands of the second product: another product for what
// the rounding leaves, as tiles of 16 rows have it, takes 1215 us for 883 (4096 over 16384) and 278 for 210 (three of
// 1000 over 5000), since the matrix units are busy half of the time here.

constexpr int kManyWaves = 8, kWide = 32 * kWaves, kWideMany = 32 * kManyWaves;
constexpr int kSchedValu = 0x002, kSchedMfma = 0x008, kSchedDsRead = 0x100;  // sched_group_barrier classes

typedef __attribute__((address_space(1))) const void global_ptr;
typedef __attribute__((address_space(3))) void lds_ptr;

// kTiles: tiles of 32 columns, of which there are some; a row has D columns in LDS.
template <int kTiles, int kTileWaves, bool E4M3>
__global__ __launch_bounds__(kTileWaves * L2C_WAVE,
                             kTiles <= 4 && kTileWaves == kWaves ? 2 : 1) void wide_kernel(Attention a) {
  constexpr int kLaneCount = kTileWaves * L2C_WAVE;
  constexpr int D = kTiles <= 2 ? 64 : kTiles <= 4 ? 128 : 256;
  constexpr int kKeys = 64;
  constexpr int kLanes = D / 8;               // that load a row
  constexpr int kRows = kLaneCount / kLanes;    // rows loaded together
  constexpr int kPasses = kKeys / kRows;
  constexpr int kTogether = kRows / kTileWaves;   // of them by one wave
  constexpr int kSteps = 2 * kTiles, kParts = kKeys / 32;
  // Two of each, with names of their own: of one array's halves the compiler would wait for the loads into one
  // before it reads the other.
  constexpr int kSecond = E4M3 ? 8 : kKeys * D;
  __shared__ __attribute__((aligned(16))) uint16_t keys_0[kKeys * D], keys_1[kSecond], values_0[kKeys * D],
      values_1[kSecond];
  __shared__ __attribute__((aligned(16))) float key_scales[kKeys], value_scales[kKeys];
  __shared__ int odd_step;  // the last step in which a wave found values that are not finite
  const int lane = threadIdx.x % L2C_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int n = lane % 32, h = lane / 32;
  int block = blockIdx.x;
  const int kv = block % a.kv_heads;
  block /= a.kv_heads;
  const int split = block % a.splits;
  Tile t;
  if (!longest_tile_of<32 * kTileWaves>(a, block / a.splits, t)) return;
  divide<kKeys>(a, t);
  if (split >= t.parts) return;
  const int begin = t.begin + split * t.chunk, end = min(t.end, begin + t.chunk);
  const int first = 32 * wave;                       // of the wave's rows
  const int count = max(0, min(32, t.count - first));  // of them
  const bool mine = n < count;
  const int packed = t.first + (mine ? first + n : 0);
  const int row = t.row(a, packed), head = t.head(a, kv, packed);
  const int position = mine ? t.position(a, packed) : -1;
  const int lowest = a.window ? max(-1, position - a.window) : -1;
  const int every = t.position(a, t.first);  // all rows of the tile see positions up to this one
  const int nobody = a.window ? t.position(a, t.first + t.count - 1) - a.window : -1;
  // Of the wave: all rows see positions in (whole_from, whole_to], none those outside [some_from, some_to].
  const int whole_to = count > 0 ? t.position(a, t.first + first) : -1;
  const int some_to = count > 0 ? t.position(a, t.first + first + count - 1) : -1;
  const int whole_from = a.window ? some_to - a.window : -1, some_from = a.window ? whole_to - a.window + 1 : 0;
  if (threadIdx.x == 0) odd_step = -1;
  __syncthreads();

  // The scale's sign goes to the queries, and 0 is the least number instead, so that the largest of the products
  // is the largest score, and -Inf stays that.
  const float scale = fmaxf(fabsf(a.scale), FLT_MIN);
  bf16x8 q[kSteps];
#pragma unroll
  for (int c = 0; c < kSteps; ++c) {
    const int d = 16 * c + 8 * h;
    u32x4 v = {0, 0, 0, 0};
    if (mine && d < a.width)
      v = *reinterpret_cast<const u32x4 *>(a.q + row * a.q_stride + static_cast<size_t>(head) * a.width + d);
    if (a.scale < 0.0f) v ^= 0x80008000u;
    q[c] = __builtin_bit_cast(bf16x8, v);
  }

  // A tile's pages, a key a lane.
  auto look_up = [&](int base) __attribute__((always_inline)) {
    const int j = base + lane;
    return j >= t.from && j < end ? a.s.page(t.sequence, a.s.by_page(j)) : -1;
  };
  auto row_of = [&](int page, int j) __attribute__((always_inline)) {
    return (static_cast<size_t>(static_cast<unsigned>(page)) * a.kv_heads + kv) * a.s.page_size +
           (j - a.s.by_page(j) * a.s.page_size);
  };
  // Lanes that read a chunk of eight (sixteen) keys together: each in other banks.
  auto key_swap = [](int key) __attribute__((always_inline)) { return D == 64 ? key >> 1 & 7 : key & 15; };
  // Lanes that read four keys of 32 columns together, the same.
  auto value_swap = [](int key) __attribute__((always_inline)) {
    return D == 64 ? (key >> 1 & 1) << 2 : (key & 3) << 2;
  };
  auto value_place = [&](int key, int chunk) __attribute__((always_inline)) {
    return key * D + 8 * (chunk ^ value_swap(key));
  };
  const int load_row = threadIdx.x / kLanes, load_chunk = threadIdx.x % kLanes;
  Raw<E4M3> k[kPasses], v[kPasses];
  float key_scale = 0.0f, value_scale = 0.0f;
  // Begins to load a tile, `there` of which have a page: into LDS, or registers.
  static_assert(kKeys == L2C_WAVE, "a key a lane");
  const bool together = a.s.page_size % kTogether == 0;  // a wave's rows lie in one page
  const unsigned row_bytes = 2u * static_cast<unsigned>(a.width);
  const unsigned long long page_bytes = a.page_rows * row_bytes;
  const unsigned long long head_bytes = static_cast<unsigned long long>(kv) * a.s.page_size * row_bytes;
  auto load = [&](int pages, unsigned long long there, int base, uint16_t *to_keys, uint16_t *to_values)
                  __attribute__((always_inline)) {
    if constexpr (E4M3) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = i * kRows + load_row, page = __shfl(pages, r, L2C_WAVE);
        k[i] = v[i] = Raw<E4M3>{};
        if (a.s.is_page(page) && 8 * load_chunk < a.width) {
          const size_t at = row_of(page, base + r) * a.width + 8 * load_chunk;
          k[i] = load_raw<E4M3>(a.keys, at);
          v[i] = load_raw<E4M3>(a.values, at);
        }
      }
      key_scale = value_scale = 0.0f;
      if (a.s.is_page(pages)) {
        const size_t at = row_of(pages, base + lane);
        key_scale = a.key_scales[at], value_scale = a.value_scales[at];
      }
    } else {
      // Where the lane's key lies; then a lane's 16 bytes go to LDS after those of the lane before.
      const int j = base + lane;
      const unsigned long long page = static_cast<unsigned>(pages), of_page = j - a.s.by_page(j) * a.s.page_size;
      const unsigned long long offset = page * page_bytes + head_bytes + of_page * row_bytes;
      const unsigned low = static_cast<unsigned>(offset), high = static_cast<unsigned>(offset >> 32);
      const bool whole = together && there == ~0ull;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = i * kRows + load_row, first_row = i * kRows + wave * kTogether;
        const unsigned key_at = 16u * (load_chunk ^ key_swap(r)), value_at = 16u * (load_chunk ^ value_swap(r));
        const unsigned char *from_key, *from_value;
        if (whole) {
          const unsigned long long at =
              static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_readlane(high, first_row))) << 32 |
              static_cast<unsigned>(__builtin_amdgcn_readlane(low, first_row));
          const unsigned row_at = (load_row % kTogether) * row_bytes;
          from_key = static_cast<const unsigned char *>(a.keys) + at + (row_at + key_at);
          from_value = static_cast<const unsigned char *>(a.values) + at + (row_at + value_at);
        } else {
          const unsigned long long above = static_cast<unsigned>(__shfl(high, r, L2C_WAVE));
          const unsigned long long at = above << 32 | static_cast<unsigned>(__shfl(low, r, L2C_WAVE));
          const bool is = there >> r & 1;
          from_key = is ? static_cast<const unsigned char *>(a.keys) + at + key_at
                        : reinterpret_cast<const unsigned char *>(zero_row);
          from_value = is ? static_cast<const unsigned char *>(a.values) + at + value_at
                          : reinterpret_cast<const unsigned char *>(zero_row);
        }
        if (a.width != D) {  // columns past the row's
          if (key_at >= row_bytes) from_key = reinterpret_cast<const unsigned char *>(zero_row);
          if (value_at >= row_bytes) from_value = reinterpret_cast<const unsigned char *>(zero_row);
        }
        const int place = i * kRows * D + wave * 8 * L2C_WAVE;
        __builtin_amdgcn_global_load_lds((global_ptr *)from_key, (lds_ptr *)(to_keys + place), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((global_ptr *)from_value, (lds_ptr *)(to_values + place), 16, 0, 0);
      }
    }
  };

  f32x16 acc[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
  float top = -INFINITY, total = 0.0f;  // of the products, without the scale
  bool odd = false;                     // there were values for odd_positions()
  int pages = look_up(begin);
  unsigned long long next_there = __ballot(a.s.is_page(pages));
  load(pages, next_there, begin, keys_0, values_0);
  pages = look_up(begin + kKeys);
  auto step = [&](int base, uint16_t *keys, uint16_t *values, uint16_t *next_keys, uint16_t *next_values)
      __attribute__((always_inline)) {
    const unsigned long long there = next_there;
    const bool mixed = base + kKeys - 1 > every || base <= nobody;
    bool bad = false;
    if constexpr (E4M3) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = i * kRows + load_row;
        const u32x4 kk = as_bf16(k[i]), vv = as_bf16(v[i]);
        if (mixed) bad |= not_finite(vv);
        *reinterpret_cast<u32x4 *>(keys + r * D + 8 * (load_chunk ^ key_swap(r))) = kk;
        *reinterpret_cast<u32x4 *>(values + r * D + 8 * (load_chunk ^ value_swap(r))) = vv;
      }
      const bool odd_scale = mixed && not_finite(value_scale);
      if (__ballot(odd_scale)) odd = true;
      if (wave == 0) key_scales[lane] = key_scale, value_scales[lane] = odd_scale ? 0.0f : value_scale;
      if (mixed && __ballot(bad) && lane == 0) odd_step = base;
      __syncthreads();
    } else {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (mixed) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
          bad |= not_finite(*reinterpret_cast<const u32x4 *>(values + 8 * (i * kLaneCount + threadIdx.x)));
        if (__ballot(bad) && lane == 0) odd_step = base;
        __syncthreads();
      }
    }
    // Where some rows see values and others do not, 0 in the place of those that are not finite.
    if (mixed && __builtin_amdgcn_readfirstlane(odd_step) == base) {
      odd = true;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        u32x4 *const at = reinterpret_cast<u32x4 *>(values + 8 * (i * kLaneCount + threadIdx.x));
        *at = finite_part(*at);
      }
      __syncthreads();
    }
    next_there = __ballot(a.s.is_page(pages));
    load(pages, next_there, base + kKeys, next_keys, next_values);
    pages = look_up(base + 2 * kKeys);
    if (base > some_to || base + kKeys - 1 < some_from) return;
    // Scores of positions 32 u + 8 (i / 4) + 4 h + i % 4, of query n. Keys are read four operands ahead, in
    // this order and no other: left to itself the compiler reads one, waits, and multiplies.
    f32x16 s[kParts];
    constexpr int kAhead = 4, kGroups = kParts * kSteps / kAhead;
    u32x4 operand[2][kAhead];
    auto read_keys = [&](u32x4 (&to)[kAhead], int group) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int u = (group * kAhead + e) / kSteps, c = (group * kAhead + e) % kSteps;
        to[e] =
            *reinterpret_cast<const u32x4 *>(keys + (32 * u + n) * D + 8 * ((2 * c + h) ^ key_swap(32 * u + n)));
      }
    };
    read_keys(operand[0], 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int group = 0; group < kGroups; ++group) {
      if (group + 1 < kGroups) read_keys(operand[(group + 1) % 2], group + 1);
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int u = (group * kAhead + e) / kSteps, c = (group * kAhead + e) % kSteps;
        f32x16 before = s[u];
        if (c == 0)
#pragma unroll
          for (int i = 0; i < 16; ++i) before[i] = 0.0f;
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, operand[group % 2][e]), q[c], before,
                                                       0, 0, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kSchedDsRead, kAhead, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, kAhead, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (E4M3) {
#pragma unroll
      for (int u = 0; u < kParts; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = *reinterpret_cast<const f32x4 *>(&key_scales[32 * u + 8 * i + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][4 * i + e] *= x[e];
        }
    }
    if (base + kKeys - 1 > whole_to || base <= whole_from || there != ~0ull) {
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        const unsigned seen = seen_of_32(static_cast<unsigned>(there >> (32 * u)), position - base - 32 * u,
                                         lowest - base - 32 * u) >>
                              (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(seen >> (8 * (i / 4) + i % 4) & 1)) s[u][i] = -INFINITY;
      }
    }
    float most = top;
#pragma unroll
    for (int u = 0; u < kParts; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, s[u][i]);
    most = max_halves(most);
    // Sums stay relative to an older maximum until a new one is more than 2^kSlack times as large. Weights are
    // 2^-kSlack of the softmax's, so that none is above 1 and large values do not overflow.
    if (__ballot((most - top) * scale > kSlack)) {
      const float again = top == -INFINITY ? 0.0f : exp2_of((top - most) * scale);
      total *= again;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        // The sums of more than 128 columns lie in accumulation registers, and leave them here alone: where the
        // compiler chose, they were copied to others and back on every step (256 wide, 200 over 10000: 130 us, 155).
        if constexpr (kTiles > 4) asm volatile("" : "+a"(acc[i]));
        acc[i] *= again;
        if constexpr (kTiles > 4) asm volatile("" : "+a"(acc[i]));
      }
      top = most;
    }
    const float shift = top == -INFINITY ? 0.0f : fmaf(top, scale, kSlack);
    // 16 positions at a time: while the matrix unit has their product, the next ones' weights are computed and
    // their values read.
    u32x4 weight[2], column[2][kTiles];
    auto weigh = [&](u32x4 &to, int group) __attribute__((always_inline)) {
      const int u = group / 2;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const int at = 8 * (group % 2) + i;
        f32x4 x = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (E4M3) x = *reinterpret_cast<const f32x4 *>(&value_scales[32 * u + 2 * at + 4 * h]);
        float e[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          e[m] = exp2_of(fmaf(s[u][at + m], scale, -shift));
          total += e[m];
          if constexpr (E4M3) e[m] *= x[m];
        }
        to[i / 2] = pack2(e[0], e[1]);
        to[i / 2 + 1] = pack2(e[2], e[3]);
      }
    };
    auto read_values = [&](u32x4 (&to)[kTiles], int group) __attribute__((always_inline)) {
      const int key = 16 * group + 4 * h + (n % 16) / 4;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const int d = 32 * i + 16 * (n / 16) + 4 * (n % 4);
        const u32x2 low = read_column(values + value_place(key, d / 8) + d % 8);
        const u32x2 high = read_column(values + value_place(key + 8, d / 8) + d % 8);
        to[i] = u32x4{low[0], low[1], high[0], high[1]};
      }
    };
    read_values(column[0], 0);
    weigh(weight[0], 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int group = 0; group < 2 * kParts; ++group) {
      const bool more = group + 1 < 2 * kParts;
      if (more) {
        read_values(column[(group + 1) % 2], group + 1);
        weigh(weight[(group + 1) % 2], group + 1);
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, column[group % 2][i]),
                                                         __builtin_bit_cast(bf16x8, weight[group % 2]), acc[i],
                                                         0, 0, 0);
      if (more) {
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2 * kTiles, 0);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kSchedValu, 28 / kTiles, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (E4M3) {
    for (int base = begin; base < end; base += kKeys) {
      step(base, keys_0, values_0, nullptr, nullptr);
      __syncthreads();
    }
  } else {
    for (int base = begin; base < end; base += 2 * kKeys) {
      step(base, keys_0, values_0, keys_1, values_1);
      if (base + kKeys >= end) break;
      step(base + kKeys, keys_1, values_1, keys_0, values_0);
    }
  }
  // The last tile's load, of no positions, may still be writing zeros to LDS.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  if (odd)
    odd_positions<kKeys, E4M3, E4M3>(a, t, kv, begin, kKeys, end, every, nobody, [&](size_t at, int j) {
      const bool sees = j <= position && j > lowest;
      if (!__ballot(sees)) return;
      float score = 0.0f;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        const int d = 16 * c + 8 * h;
        if (d < a.width)
          score = dot8(as_bf16(load_raw<E4M3>(a.keys, at * a.width + d)), __builtin_bit_cast(u32x4, q[c]), score);
      }
      score = sum_halves(score);
      if constexpr (E4M3) score *= a.key_scales[at];
      float weight = exp2_of(fmaf(score, scale, top == -INFINITY ? 0.0f : -fmaf(top, scale, kSlack)));
      bool whole_row = false;
      if constexpr (E4M3) {
        const float value_scale = a.value_scales[at];
        whole_row = not_finite(value_scale);
        weight *= value_scale;
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int d = 32 * i + 8 * m + 4 * h;
          const f32x4 x = load4<E4M3>(a.values, at * a.width + (d < a.width ? d : 0));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[i][4 * m + e] += sees && (whole_row || not_finite(x[e])) ? weight * x[e] : 0.0f;
        }
    });
  total = sum_halves(total);
  const bool whole = t.parts == 1;
  const float by = whole ? inverse(total) : 1.0f;
  if (!mine) return;
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int d = 32 * i + 8 * m + 4 * h;
      if (d >= a.width) continue;
      const f32x4 o = {acc[i][4 * m] * by, acc[i][4 * m + 1] * by, acc[i][4 * m + 2] * by, acc[i][4 * m + 3] * by};
      store4(a, whole, row, head, split, d, o);
    }
  if (!whole && h == 0)
    a.part_sums[part_of(a, row, head, split)] = make_float2(top == -INFINITY ? top : fmaf(top, scale, kSlack), total);
}

// ---------------------------------------------------------------------------
// The parts of tiles that were divided. A wave a row and head, or, of many parts, a workgroup, whose halves of
// waves have every eighth part: one wave went through 64 of them in 28 us (4 x 32 rows and heads).
constexpr int kFewParts = 8;

template <int M, int STEP, bool MANY>
__global__ __launch_bounds__(kThreads) void join_kernel(Attention a) {
  constexpr int kBlock = 128;  // columns of a half wave
  __shared__ __attribute__((aligned(16))) float shared[MANY ? kWaves * kBlock : 4];
  const int lane = threadIdx.x % L2C_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / L2C_WAVE);
  const int item = MANY ? blockIdx.x : __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + wave);
  if (item >= a.s.rows * a.heads) return;
  const int row = item / a.heads, head = item - row * a.heads;
  int sequence, position;
  if (!a.s.find(row, sequence, position)) return;
  Tile t;
  t.sequence = sequence;
  t.start = a.s.starts ? a.s.starts[sequence] : row;
  const int to = a.s.starts ? a.s.starts[sequence + 1] : row + 1;
  t.before = static_cast<long long>(a.s.lengths[sequence]) - (to - t.start);
  const int kv = head / a.group, packed = (row - t.start) * a.group + (head - kv * a.group);
  t.first = packed / M * M;
  t.count = min(M, (to - t.start) * a.group - t.first);
  divide<STEP>(a, t);
  if (t.parts == 1) return;  // whole already
  const size_t first = part_of(a, row, head, 0);
  // At most 64 parts: a lane each.
  const float2 sums = lane < t.parts ? a.part_sums[first + lane] : make_float2(-INFINITY, 0.0f);
  const float most = l2c::wave_max(sums.x);
  const float weight = lane < t.parts ? exp2_of(sums.x - (most == -INFINITY ? 0.0f : most)) : 0.0f;
  const float by = inverse(l2c::wave_sum(sums.y * weight));
  const float *const values = a.part_values + first * a.width;
  constexpr int kLanes = kBlock / 4, kStride = MANY ? 2 * kWaves : 2;
  const int half = (MANY ? 2 * wave : 0) + lane / kLanes, column = 4 * (lane % kLanes);
  for (int block = 0; block < a.width; block += kBlock) {
    const int d = block + column;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = 0; i < t.parts; i += kStride) {
      const int part = i + half;
      const float w = __shfl(weight, part & (L2C_WAVE - 1), L2C_WAVE);
      if (part < t.parts && d < a.width)
        sum += *reinterpret_cast<const f32x4 *>(values + static_cast<size_t>(part) * a.width + d) * w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = sum_halves(sum[e]);
    if constexpr (MANY) {
      if (block > 0) __syncthreads();
      if (lane < kLanes) *reinterpret_cast<f32x4 *>(shared + wave * kBlock + column) = sum;
      __syncthreads();
      if (wave > 0 || lane >= kLanes) continue;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4 *>(shared + w * kBlock + column);
    }
    if (lane < kLanes && d < a.width) store4(a, true, row, head, 0, d, sum * by);
  }
}

// ---------------------------------------------------------------------------

constexpr int kMaxSplits = 64;

struct Plan {
  int rows;  // of a tile: kNarrow, kWide or kWideMany
  long long slots;
  int splits, least;  // the least positions of a part: a multiple of the kernels' steps
};

// Tiles of 16 rows where the sequences have no more on average, whose weights are the more precise, or, of e4m3 pages,
// up to 24, and of 64 columns up to 48, else of 128, or of 256. In tiles of 16 and of 128 rows, us: single tokens 11.1
// and 15.1 (1 x 2048), 153 and 145 (64 x 4096), 158 and 294 (4 x 131072 in e4m3), 18.7 and 30 (16 x 5 of 2500); of 8
// rows for each of 8 key heads in bf16 58 and 52 (64 x 1000), 47 and 42 (16 x 3000), and of 24 rows 70 and 52, 62 and
// 43; in e4m3 of 24 rows 52 and 49, 44 and 55, of 32 rows 58 and 50, 48 and 57; of 64 columns in e4m3 of 32 rows 33 and
// 39, 31 and 43, of 48 rows 46 and 40, 38 and 46, of 64 rows 47 and 40, 44 and 48: where the rule ends the one is as
// often the sooner as the other. It goes by the average of a call, so a chunk among many single tokens is cut into
// small tiles, and single tokens beside a large chunk have a large tile each (1 of 1000 over 5000 and 3 of 1 over
// 131072: 2770 us in one call, 119 and 300 in two).
//
// Positions are divided until there are some workgroups for every CU, but not into parts that are mostly beginnings and
// ends: 256 positions, or, where that leaves CUs idle, 128 (16 x 5 of 2500 in tiles of 10 heads, when it took longer in
// all: 19.9 us with 256, 21.0 with 128). Of larger tiles the join has as much to write and read as a part of 256
// positions takes, so the more tiles there are, the longer their parts (700 over 700 positions of 3 sequences, 152
// tiles: 30 us in parts of 256, 24 undivided; 700 over 5000 of 4, 240 tiles: 80 in two parts, 110 undivided). A CU
// has room for two workgroups of four waves of up to 128 columns, and one of wider ones (200 over 10000, 256 wide:
// 116 us with 256 workgroups, 130 with 512). With a window, a tile sees no more positions than that and its tokens.
Plan plan(int sequences, int rows, int heads, int kv_heads, int width, int page_size, int max_pages, int window,
          bool starts, bool e4m3) {
  const int group = heads / kv_heads;
  const long long packed = static_cast<long long>(rows) * group;
  Plan p;
  const bool narrow = packed <= (!e4m3 ? 16LL : width <= 64 ? 48LL : 24LL) * sequences;
  const bool many = width > 96 && width <= 128 && packed / kWideMany * kv_heads > 256;
  const int m = p.rows = narrow ? kNarrow : many ? kWideMany : kWide;
  p.slots = starts ? packed / m + sequences : static_cast<long long>(sequences) * ((group + m - 1) / m);
  const long long tiles = p.slots * kv_heads, wanted = narrow ? 2048 : width > 128 ? 256 : 512;
  const long long least = narrow ? (tiles < 128 ? 128 : 256) : max(256LL, min(tiles, 512LL) / 8 * 64);
  long long positions = static_cast<long long>(max_pages) * page_size;
  if (window > 0) positions = min(positions, window + 2LL * m);
  long long splits = wanted / tiles;
  splits = min(splits, (positions + least - 1) / least);
  splits = min(splits, (1LL << 17) / (static_cast<long long>(rows) * heads));
  p.least = static_cast<int>(least);
  p.splits = static_cast<int>(max(1LL, min(splits, static_cast<long long>(kMaxSplits))));
  return p;
}

bool sizes(int sequences, int rows, int heads, int kv_heads, int width, int page_size, int pages, int max_pages) {
  return l2c::cache_sizes(L2C_BF16, sequences, rows, kv_heads, width, page_size, pages, max_pages) && heads > 0 &&
         heads <= 65535 && heads % kv_heads == 0;
}

using Kernel = void (*)(Attention);
template <bool E4M3>
Kernel kernel(int rows, int width) {
  if (rows == kNarrow) {
    if (E4M3 && width % 16 == 0)
      return width <= 64    ? narrow_kernel<2, E4M3, E4M3>
             : width <= 128 ? narrow_kernel<4, E4M3, E4M3>
             : width <= 192 ? narrow_kernel<6, E4M3, E4M3>
                            : narrow_kernel<8, E4M3, E4M3>;
    return width <= 64    ? narrow_kernel<2, E4M3, false>
           : width <= 96  ? narrow_kernel<3, E4M3, false>
           : width <= 128 ? narrow_kernel<4, E4M3, false>
           : width <= 192 ? narrow_kernel<6, E4M3, false>
                          : narrow_kernel<8, E4M3, false>;
  }
  return width <= 64         ? wide_kernel<2, kWaves, E4M3>
         : width <= 96       ? wide_kernel<3, kWaves, E4M3>
         : rows == kWideMany ? wide_kernel<4, kManyWaves, E4M3>
         : width <= 128      ? wide_kernel<4, kWaves, E4M3>
         : width <= 192      ? wide_kernel<6, kWaves, E4M3>
                             : wide_kernel<8, kWaves, E4M3>;
}

// Tiles of 256 rows are more than 256 and not divided.
Kernel join(const Plan &p, int width, bool many) {
  if (p.rows == kNarrow)
    return many ? join_kernel<kNarrow, kNarrowStep, true> : join_kernel<kNarrow, kNarrowStep, false>;
  return many ? join_kernel<kWide, 64, true> : join_kernel<kWide, 64, false>;
}

size_t part_bytes(const Plan &p, int rows, int heads, int width) {
  return p.splits == 1 ? 0 : static_cast<size_t>(rows) * heads * p.splits * (width + 2) * sizeof(float);
}

}  // namespace

extern "C" size_t l2c_cache_attention_workspace_bytes(int sequences, int rows, int heads, int kv_heads, int width,
                                                      int page_size, int max_pages) {
  if (!sizes(sequences, rows, heads, kv_heads, width, page_size, 0, max_pages) || sequences == 0 || rows == 0) return 0;
  // The most that a call with starts or without, of either type's pages, needs: the fewer slots, the more parts.
  size_t most = 0;
  for (const bool starts : {true, false})
    for (const bool e4m3 : {true, false})
      if (starts || rows == sequences)
        most = max(most, part_bytes(plan(sequences, rows, heads, kv_heads, width, page_size, max_pages, 0, starts,
                                         e4m3),
                                    rows, heads, width));
  return most;
}

extern "C" int l2c_cache_attention(uint16_t *out, long long out_stride, const uint16_t *q, long long q_stride,
                                   const void *keys, const void *values, const float *key_scales,
                                   const float *value_scales, int cache_type, const int *tables, const int *lengths,
                                   const int *starts, int sequences, int rows, int heads, int kv_heads, int width,
                                   int page_size, int pages, int max_pages, int window, float scale, void *workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  scale *= kLog2e;
  if (!sizes(sequences, rows, heads, kv_heads, width, page_size, pages, max_pages) || window < 0 ||
      !(fabsf(scale) <= FLT_MAX) || (cache_type != L2C_BF16 && cache_type != L2C_E4M3))
    return hipErrorInvalidValue;
  const long long row = static_cast<long long>(heads) * width;
  if (q_stride < row || out_stride < row || q_stride % 8 != 0 || out_stride % 8 != 0) return hipErrorInvalidValue;
  if (sequences == 0 || rows == 0) return hipSuccess;
  const size_t need =
      l2c_cache_attention_workspace_bytes(sequences, rows, heads, kv_heads, width, page_size, max_pages);
  if (!l2c::cache_arguments(cache_type, keys, values, key_scales, value_scales, tables, lengths, starts, sequences,
                            rows, pages, max_pages) ||
      !q || !out || !l2c_aligned16(q) || !l2c_aligned16(out) || workspace_bytes < need ||
      (need > 0 && (!workspace || !l2c_aligned16(workspace))))
    return hipErrorInvalidValue;
  const Plan p = plan(sequences, rows, heads, kv_heads, width, page_size, max_pages, window, starts != nullptr,
                      cache_type == L2C_E4M3);
  const long long grid = p.slots * kv_heads * p.splits;
  const int threads = p.rows == kWideMany ? kManyWaves * L2C_WAVE : kThreads;
  if (static_cast<long long>(rows) * heads > INT_MAX || p.slots > INT_MAX || grid > INT_MAX ||
      !l2c::launchable(grid, threads))
    return hipErrorInvalidValue;
  float *const parts = static_cast<float *>(workspace);
  const size_t items = static_cast<size_t>(rows) * heads * p.splits;
  Attention a = {};
  a.out = out, a.q = q, a.keys = keys, a.values = values, a.key_scales = key_scales, a.value_scales = value_scales;
  a.part_values = parts, a.part_sums = reinterpret_cast<float2 *>(parts + (p.splits > 1 ? items * width : 0));
  a.out_stride = out_stride, a.q_stride = q_stride;
  a.page_rows = static_cast<unsigned long long>(kv_heads) * page_size;
  a.s = l2c::sequences_of(tables, lengths, starts, sequences, rows, max_pages, page_size, pages);
  a.group = heads / kv_heads, a.by_group = l2c::Quotient31(a.group);
  a.heads = heads, a.kv_heads = kv_heads, a.width = width, a.window = window;
  a.splits = p.splits, a.slots = static_cast<int>(p.slots), a.least = p.least, a.scale = scale;
  const Kernel fn = cache_type == L2C_E4M3 ? kernel<true>(p.rows, width) : kernel<false>(p.rows, width);
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, stream, a);
  L2C_LAUNCH_CHECK();
  if (p.splits == 1) return hipSuccess;
  const bool many = p.splits > kFewParts;
  const long long pairs = static_cast<long long>(rows) * heads;
  const unsigned joins = static_cast<unsigned>(many ? pairs : (pairs + kWaves - 1) / kWaves);
  hipLaunchKernelGGL(join(p, width, many), dim3(joins), dim3(kThreads), 0, stream, a);
  L2C_LAUNCH_CHECK();
  return hipSuccess;
}

// What the kernels of the paged cache (l2c_cache.hip, l2c_attention.hip) share: which
// sequence a new token belongs to, and where in the pages a position lies.
#pragma once

#include <climits>

#include "l2c_common.h"
#include "../../include/l2c.h"

namespace l2c {

// n / by for 0 <= n < 2^31 without a division: with s = ceil(log2 by) and m =
// floor(2^32 (2^s - by) / by) + 1, (mulhi(m, n) + n) >> s (T. Granlund and P. Montgomery,
// Division by invariant integers using multiplication, 1994).
struct Quotient31 {
  unsigned by, m, s;
  Quotient31() = default;
  explicit Quotient31(int divisor) : by(static_cast<unsigned>(divisor)), s(0) {
    while ((1ull << s) < by) ++s;
    m = static_cast<unsigned>(((1ull << 32) * ((1ull << s) - by)) / by + 1);
  }
  __device__ __forceinline__ int operator()(int n) const {
    const unsigned u = static_cast<unsigned>(n);
    return static_cast<int>((__umulhi(m, u) + u) >> s);
  }
};

// Positions that tables may have room for: with some to spare below 2^31, loops may step past the last.
constexpr long long kMostPositions = 0x7fff0000LL;

struct Sequences {
  const int *tables, *lengths, *starts;
  int sequences, rows, max_pages, page_size, pages;
  Quotient31 by_page;

  // Positions that can have a page.
  __device__ __forceinline__ int capacity() const { return max_pages * page_size; }
  // The page number of a position in [0, capacity()), which may be none.
  __device__ __forceinline__ int page(int sequence, int index) const {
    return tables[static_cast<size_t>(sequence) * max_pages + index];
  }
  __device__ __forceinline__ bool is_page(int page) const {
    return static_cast<unsigned>(page) < static_cast<unsigned>(pages);
  }
  // The sequence that a row is a new token of, and its position; false for rows of no sequence. Of
  // starts that are not in order any answer will do, within the arrays.
  __device__ __forceinline__ bool find(int row, int &sequence, int &position) const {
    if (!starts) {
      sequence = row;
      position = lengths[row] - 1;
      return true;
    }
    int low = 0, high = sequences + 1;  // how many of the starts are at most row
    while (low < high) {
      const int middle = low + (high - low) / 2;
      if (starts[middle] <= row) low = middle + 1;
      else high = middle;
    }
    sequence = low - 1;
    if (sequence < 0 || sequence >= sequences) return false;
    // In 64 bits: lengths and starts may be anything.
    const long long p = static_cast<long long>(lengths[sequence]) - (static_cast<long long>(starts[low]) - row);
    position = p < -1 || p > INT_MAX ? -1 : static_cast<int>(p);
    return true;
  }
};

// The arguments that append and attention have in common; false where they are refused. Arrays of no pages, and tables
// of no columns, are nowhere.
inline bool cache_arguments(int cache_type, const void *keys, const void *values, const float *key_scales,
                            const float *value_scales, const int *tables, const int *lengths, const int *starts,
                            int sequences, int rows, int pages, int max_pages) {
  return (pages == 0 || ((cache_type == L2C_BF16 || (key_scales && value_scales)) && keys && values)) &&
         l2c_aligned16(keys) && l2c_aligned16(values) && (max_pages == 0 || tables) && lengths &&
         (starts || rows == sequences);
}
inline bool cache_sizes(int cache_type, int sequences, int rows, int kv_heads, int width, int page_size, int pages,
                        int max_pages) {
  return (cache_type == L2C_BF16 || cache_type == L2C_E4M3) && sequences >= 0 && rows >= 0 && kv_heads > 0 &&
         kv_heads <= 65535 && width > 0 && width <= L2C_MAX_HEAD && width % 8 == 0 && page_size > 0 && pages >= 0 &&
         max_pages >= 0 && static_cast<long long>(max_pages) * page_size <= kMostPositions;
}
inline Sequences sequences_of(const int *tables, const int *lengths, const int *starts, int sequences, int rows,
                              int max_pages, int page_size, int pages) {
  return {tables, lengths, starts, sequences, rows, max_pages, page_size, pages, Quotient31(page_size)};
}

}  // namespace l2c

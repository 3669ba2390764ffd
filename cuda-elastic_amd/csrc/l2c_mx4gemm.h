// The kernels behind l2c_matmul_mxfp4, and what they cost.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace l2c {

// out, X codes, X scales, W codes, W scales, batch, rows, blocks of 32 values a row.
using Mx4Kernel = void (*)(float *, const uint8_t *, const uint8_t *, const uint8_t *, const uint8_t *, int, int, int);

// One kernel: its tile (batch rows x weight rows), its lanes, the fewest blocks a row that
// it takes, and its time in ns: `launch`, and for each of the tiles that a CU takes in
// turn `tile` and `k` a value of the length.
struct Mx4Tile {
  Mx4Kernel fn;
  int bm, bn, threads, min_blocks;
  double launch, tile, k;
};

// l2c_mx4gemm_rows.hip, l2c_mx4gemm_slices.hip and l2c_mx4gemm_tiles.hip.
constexpr int kMx4SliceTiles = 3, kMx4LdsTiles = 5;
extern const Mx4Tile mx4_row_tile, mx4_slice_tiles[kMx4SliceTiles], mx4_lds_tiles[kMx4LdsTiles];

}  // namespace l2c

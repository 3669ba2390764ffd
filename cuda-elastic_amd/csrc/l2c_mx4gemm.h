// The kernels behind l2c_matmul_mxfp4, called after its argument checks (batch and
// rows above 0, `blocks` = cols / 32). Each launches and returns true where its shape is
// one of its own; the caller reads the launch's error.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

bool l2c_mx4_tiles(float *out, const uint8_t *X, const uint8_t *Xs, const uint8_t *W, const uint8_t *Ws, int batch,
                   int blocks, int rows, hipStream_t stream);

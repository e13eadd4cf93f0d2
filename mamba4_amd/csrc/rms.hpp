// Shapes and arguments of the root-mean-square norm's kernels, shared by the host entry
// points and rms.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace rn {

typedef unsigned short bf16_t;

constexpr int THREADS = 256;        // of a block, or the lanes of a row where those are more
constexpr int MAX_CHANNELS = 32768;
constexpr int SLOTS = 1024;         // scales of a block's rows at a time

// x, y, dy, dx in one type, the residual, sum, dsum, dresidual in one (x's, without a
// residual), all [M,C].
struct Rms {
  const void *x, *residual;         // residual: or NULL
  const float* weight;              // [C], or NULL
  long M;
  int C;
  float eps;
  void *y, *sum;                    // y of e4m3: bytes; sum: or NULL
  float* inverse;                   // [M] (forward: or NULL)
  // e4m3: channels of a scale, scales of a row, and lanes of a wave that share one.
  float* scale;
  int block, blocks, group;
  // Backward: x is the sum.
  const void *dy, *dsum;            // dsum: or NULL
  void *dx, *dresidual;             // or NULL
  float* part;                      // [blocks][C] sums of dweight, or NULL
  int lanes, rows;                  // threads of a row, rows of a block at a time
};

}  // namespace rn

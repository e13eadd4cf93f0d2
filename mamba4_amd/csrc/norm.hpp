// Shapes and arguments of the group norm's kernels, shared by the host entry
// points and norm.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace gn {

typedef unsigned short bf16_t;

constexpr int ROW_THREADS = 512;   // largest block of the row kernels
constexpr int POS_THREADS = 512;   // block of the position kernels
enum Activation { NONE = 0, SILU = 1, GELU = 2 };
// What a launch over positions does: partial sums, what follows from them (a part of
// the positions a block), or both (whole samples).
enum Phase { SUMS = 0, APPLY = 1, BOTH = 2 };

// x, gate, dy, y, dx, dgate: [M, L, C] with G groups of D = C / G channels.
struct Norm {
  const void *x, *gate, *dy;
  const float *weight, *bias;  // [C], or NULL
  void *y, *dx, *dgate;        // dx, dgate: NULL if not wanted (dgate also without a gate)
  float* part;                 // column sums' partials [rows][2][C], or NULL
  long M;
  int L, C, G, D;
  float eps;
  int act;
  // Row kernels: lanes of a group, rows of a block at a time, groups of a block.
  int lanes, rows, groups;
  // Position kernels: parts of the positions, vectors of a group, groups of a block,
  // parts of a group (more vectors than a block's threads), rows at a time.
  int parts, vecs, span, subs;
  float* sums;                 // [M][parts][subs][G][4] partial statistics
  float* stats;                // [M][G][2] mean, 1 / deviation (forward: or NULL)
};

}  // namespace gn

// Shapes and arguments of the selective scan's kernels, shared by the host entry
// points and selscan.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace ss {

typedef unsigned short bf16_t;

constexpr int TILE = 16;    // tokens of a tile: the lanes of a row hold a tile's b and c
// Tokens between the states that the forward keeps (of NG groups of 16 states): a tile, or
// half of one where the backward could not hold a tile's states in registers.
constexpr int kept_tokens(int NG) { return NG == 1 ? TILE : TILE / 2; }
constexpr int WAVES = 4;    // waves of a block, of 16 channels each
constexpr int BLOCK_CHANNELS = 16 * WAVES;
constexpr int STEP_THREADS = 256;

struct Rows {
  const void* p;
  long batch, token;
};

struct Scan {
  Rows x, delta, gate, b, c;
  long bg, cg;                    // group strides of b and c
  const float *a, *skip, *bias;   // [D,N], [D], [D] (skip, bias: or NULL)
  const int* lengths;             // [B], or NULL
  int B, T, D, G, Dg, N;          // Dg = D / G
  int softplus, gated;            // (gate: x's rows, where there is none)
  int whole_n;                    // float32 states are read in pieces of four
  int blocks;                     // blocks of a group's channels
  int seg, NS;                    // tokens of a segment, segments
  int skipped;                    // first segments that a launch leaves out
  int folded;                     // whether a segment joins those before it by itself
  const float* initial;           // [B,D,N], or NULL (NS == 1: the start state)
  // Of the segments ([B,NS,D,N] and [B,NS,D]): what each adds to the state (forward)
  // or its cotangent (backward) from zero, then, carried, what each starts from; and
  // the sums of its steps.
  float *ends, *sums;
  float* kept;                    // [B,tiles,D,N] states before each tile, or NULL
  void* out;                      // [B,T,D]
  float* state;                   // [B,D,N]
  // Backward.
  const void* dout;               // [B,T,D]
  const float* dstate;            // [B,D,N], or NULL
  void *dx, *ddelta, *dgate;      // [B,T,D] (dgate: or NULL)
  float* dinitial;                // [B,D,N], or NULL
  float* part_bc;                 // [blocks][B,T,G][2][N]
  float* part_a;                  // [B,NS][D,N], or NULL
  float* part_d;                  // [B,NS][2][D]: of skip and bias
};

// The sums of the backward's parts.
struct Join {
  const float *part_bc, *part_a, *part_d;
  unsigned bc_blocks;             // blocks of the launch that join b's and c's
  int blocks;                     // of channels
  long rows;                      // batch rows and segments
  int B, T, D, G, N;
  const int* lengths;
  void *db, *dc;
  float *da, *dskip, *dbias;      // or NULL
};

struct Step {
  Rows x, delta, gate, b, c;      // (token strides unused)
  long bg, cg;
  const float *a, *skip, *bias;
  const unsigned char* active;    // [B], or NULL
  const float* state;
  float* new_state;
  void* out;
  long B;
  int D, Dg, N, softplus;
  int whole_n, whole_bc;          // states and a, b and c are read in pieces of four
  int span;                       // 2^span threads hold a channel's states
  int blocks;                     // of all channels
};

}  // namespace ss

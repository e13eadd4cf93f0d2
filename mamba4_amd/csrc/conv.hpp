// Shapes and arguments of the short causal convolution's kernels, shared by the host
// entry points and conv.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace cv {

typedef unsigned short bf16_t;

constexpr int THREADS = 256;
constexpr int MAX_TAPS = 8;
enum Activation { NONE = 0, SILU = 1 };

// x, y, dy, dx [B,T,D] (x with strides, the others dense); initial, state and their
// gradients [B,W-1,D], dense.
struct Conv {
  const void* x;
  long xb, xt;
  const float *weight, *bias;    // [D,W], [D] (or NULL)
  const void* initial;           // or NULL
  const int* lengths;            // [B], or NULL
  int B, T, D;
  int act;
  int run;                       // tokens that a thread walks
  int runs;                      // of a row
  int cols;                      // pieces of channels
  int lines;                     // runs of a block at a time (THREADS / columns of a block)
  void *y, *state;               // state: or NULL
  const void *dy, *dstate;       // dstate: or NULL
  void *dx, *dinitial;           // or NULL
  float* part;                   // [blocks along runs][W + 1][D] sums of dweight, dbias, or NULL
};

struct Step {
  const void* x;
  long xb;
  const float *weight, *bias;
  const unsigned char* active;   // [B], or NULL
  const void* state;
  void *new_state, *y;
  long B;
  int D, act, cols;
  int blocks;                    // of a row
};

}  // namespace cv

// Shapes and arguments of the decayed linear attention's kernels, shared by
// the host entry points and linattn.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace la {

constexpr int C = 64;        // tokens of a chunk
constexpr int TILE = 64;     // value columns of a block
constexpr int WAVES = 4;     // strips of 16 tokens in a chunk, each a wave's
constexpr int MAX_WIDTH = 128;
constexpr int GRAD_THREADS = 256;  // block of the decays' gradient
constexpr int STEP_THREADS = 256;  // block of the step's kernel

typedef unsigned short bf16_t;

// Rows [B,T,h,W] of one operand: unit stride along W, element strides along
// the others, `share` attention heads to each of its own; whole: 16-byte pieces.
struct Rows {
  const void* base;
  long sb, st, sh;
  int share, width, whole;
};

// States [B,H,.,.] float32 with element strides of the key and value axes
// (a transposed state swaps them); NULL: zeros, or not wanted.
struct States {
  float* base;
  int sn, sp;
};

// One linear attention over the tokens (in reverse, if rev): scores q.k,
// values v, state [n, p] with n the width of q and k and p that of v.
//   out_i = intra * sum_j D_ij (q_i.k_j) v_j + inter * E_i q_i^T S
//   S'    = D_L S + update * sum_j F_j k_j v_j^T
struct Role {
  Rows q, k, v;
  States initial, final;
  void* out;           // [B,T,H,p] contiguous
  int out_f32;         // out is float32 (else the operands' type)
  int rev;
  float intra, inter, update;
  Rows e;              // dots_i = (out_i less its term j = i) . e_i over the
                       // tile's columns, if dots
  float* dots;         // [tiles][B,H,T], or NULL
  int n, p, tiles;
  float* starts;       // [tiles][B*H][NS][NT * 4096] segments' start states (split runs,
                       // and with dots)
  float* decays;       // split runs: [tiles][B*H][NS]
};

struct Args {
  Role role[3];
  int roles, blocks;       // blocks of one (b, h): the roles' tiles together
  const float* g;          // log decays, element strides gb, gt (zero: per head)
  long gb, gt;
  const int* lengths;      // [B], or NULL
  int B, T, H, NC, NS;
  int seg, split;          // chunks of a segment; split: a segment a block
};

// d log_decay from the dots and the segments' start states of the roles of dQ
// and dK.
struct DecayGrad {
  const float *dots_q, *dots_k;      // [tiles][B,H,T]
  const float *starts_q, *starts_k;  // [tiles][B*H][NS][slot]
  int tiles, slot, seg, NS;
  const float* g;
  long gb, gt;
  const int* lengths;
  const float *state, *d_state;      // [B,H,n,p], or both NULL
  int n, p;
  float* d_g;                        // [B,T,H], or NULL
  double* head;                      // [B,H,NS] sums over the tokens, or NULL
  int B, T, H;
};

// Rows to be copied to rows of `padded` columns, [B,T,heads,padded], zeros past
// the width.
struct Pack {
  Rows from[4];
  void* to[4];
  int heads[4], padded[4];
  int B, T;
};

struct Step {
  const void *q, *k, *v;
  long qb, qh, kb, kh, vb, vh;
  int q_share, k_share, v_share;
  const float* g;
  long gb;
  const unsigned char* active;   // [B], or NULL
  const float* state;
  float* new_state;
  void* out;
  float scale;
  int B, H, N, P;
  int span;                      // 2^span threads hold a row of the state
};

}  // namespace la

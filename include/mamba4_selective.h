/*
 * mamba4_selective.h -- C ABI of the MI355X (gfx950) selective state space
 * layer's operators: the selective scan over prompts and training batches, its
 * gradient, and its step for single tokens; the short causal convolution before it,
 * likewise; the root-mean-square norm with the residual's addition, its gradient, and
 * its result in 8 bits (the library that also holds mamba4_memread.h).
 *
 * Plain pointers and sizes only; every buffer is on the device and owned by
 * the caller.  `stream` is a hipStream_t passed as void* (NULL = the null
 * stream).  No function allocates, frees or synchronises.  Return values are
 * those of mamba4_memread.h (M4MR_OK, M4MR_EINVAL with nothing launched,
 * M4MR_EHIP); m4mr_last_error() gives the message.
 */
#ifndef MAMBA4_SELECTIVE_H
#define MAMBA4_SELECTIVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Most states of a channel, and most taps of the convolution. */
#define M4SL_MAX_STATES 64
#define M4SL_MAX_TAPS 8

/*
 * Rows [B,T,...] with unit stride along the channels (or states) and strides in
 * elements along the others (the token stride is not read by the steps).
 */
typedef struct {
  const void* data;
  long batch_stride, token_stride;
} m4sl_rows;

/*
 * The selective scan: every channel d of D has N states,
 *   s_t = softplus(delta_t + delta_bias) if `softplus` is not zero, else
 *         delta_t + delta_bias
 *   h_t[n] = exp(s_t a[d,n]) h_{t-1}[n] + s_t b_t[g,n] x_t
 *   y_t = sum over n of c_t[g,n] h_t[n] + skip x_t,    out_t = y_t silu(gate_t)
 * x, delta, gate [B,T,D] and b, c [B,T,G,N] in float32, or bfloat16 if `bf16` is
 * not zero; G divides D and channel d reads group g = d / (D / G).  a [D,N],
 * skip [D], delta_bias [D] float32.  gate.data, skip, delta_bias: NULL for none.
 */
typedef struct {
  m4sl_rows x, delta, gate, b, c;
  long b_group_stride, c_group_stride;
  const float *a, *skip, *delta_bias;
  int B, T, D, G, N, bf16, softplus;
} m4sl_scan;

/* Floats of the states that the forward keeps for the backward: every 16 tokens, with more
 * than 16 states every 8. */
long m4sl_scan_kept_floats(const m4sl_scan* scan);

/*
 * initial [B,D,N] float32, or NULL for zeros.  lengths [B] int32, or NULL: tokens at
 * lengths[b] and after are absent (their rows are not read into any result, their
 * output is zero; lengths outside 0..T are clamped).  output [B,T,D] in x's type;
 * state [B,D,N] float32, after the last token.  kept: for the backward, or NULL.
 *
 * Steps, decays, states and sums are float32; each result is rounded once.  A long
 * sequence of a small batch is cut into segments whose states are formed first, so
 * that a row's result may depend on the batch size, by rounding.
 */
size_t m4sl_scan_workspace_bytes(const m4sl_scan* scan);
int m4sl_scan_forward(const m4sl_scan* scan, const float* initial, const int* lengths,
                      void* output, float* state, float* kept, void* workspace,
                      size_t workspace_bytes, void* stream);

/*
 * Its gradient, from the cotangents d_output [B,T,D] in x's type and d_state
 * [B,D,N] (NULL: zero) and what the forward kept.  Gradients: x, delta, gate
 * [B,T,D] and b, c [B,T,G,N] in the inputs' type, contiguous; a, skip, delta_bias
 * and initial float32.  gate, skip, delta_bias, initial and a: NULL if not wanted.
 * Sums over tokens, channels and states are float32 in a fixed order.
 */
typedef struct {
  void *x, *delta, *gate, *b, *c;
  float *a, *skip, *delta_bias, *initial;
} m4sl_scan_grads;
size_t m4sl_scan_backward_workspace_bytes(const m4sl_scan* scan);
int m4sl_scan_backward(const m4sl_scan* scan, const int* lengths, const void* d_output,
                       const float* d_state, const float* kept, const m4sl_scan_grads* grads,
                       void* workspace, size_t workspace_bytes, void* stream);

/*
 * One token (T is not read): state [B,D,N] float32 to new_state (which may be state
 * itself: in place) and output [B,D] in x's type.  active [B] bytes, or NULL: a row
 * whose byte is zero keeps its state and its output is zero.
 */
int m4sl_scan_step(const m4sl_scan* scan, const uint8_t* active, const float* state,
                   float* new_state, void* output, void* stream);

#define M4SL_NONE 0
#define M4SL_SILU 1

/*
 * Causal convolution of W taps over each channel:
 *   y_t = act(bias + sum over j < W of weight[d,j] x_{t-W+1+j})
 * x [B,T,D] in float32, or bfloat16 if `bf16` is not zero; weight [D,W], bias [D]
 * (or NULL) float32; W in 1..M4SL_MAX_TAPS.  initial [B,W-1,D] in x's type: the rows
 * before the first token, oldest first (NULL: zeros).  lengths as in the scan.
 * output [B,T,D] and state [B,W-1,D] (the last rows that are present, of `initial`
 * where they are fewer; NULL: not wanted) in x's type.
 */
int m4sl_conv_forward(const m4sl_rows* x, const float* weight, const float* bias,
                      const void* initial, const int* lengths, int bf16, int B, int T, int D,
                      int W, int activation, void* output, void* state, void* stream);

/*
 * Its gradient, from d_output [B,T,D] and d_state [B,W-1,D] (NULL: zero) in x's
 * type: d_x [B,T,D] and d_initial [B,W-1,D] in x's type, d_weight [D,W] and
 * d_bias [D] float32, each NULL if not wanted.  Sums are float32 in a fixed order.
 */
size_t m4sl_conv_backward_workspace_bytes(int B, int T, int D, int W);
int m4sl_conv_backward(const m4sl_rows* x, const float* weight, const float* bias,
                       const void* initial, const int* lengths, const void* d_output,
                       const void* d_state, int bf16, int B, int T, int D, int W,
                       int activation, void* d_x, void* d_initial, float* d_weight,
                       float* d_bias, void* workspace, size_t workspace_bytes, void* stream);

/*
 * One token: x [B,D] (rows; the token stride is not read), state [B,W-1,D] in x's
 * type to new_state (which may be state itself) and output [B,D].  active as in the
 * scan's step.
 */
int m4sl_conv_step(const m4sl_rows* x, const float* weight, const float* bias,
                   const uint8_t* active, int bf16, int B, int D, int W, int activation,
                   const void* state, void* new_state, void* output, void* stream);

/* Most channels of the norm. */
#define M4SL_MAX_NORM 32768

/*
 * Root-mean-square norm of the sum of x and the residual, both [M,C]:
 *   sum = x + residual, rounded to the residual's type;
 *   output = sum / sqrt(mean(sum^2) + eps) * weight, in x's type.
 * x float32, or bfloat16 if `x_bf16`, the residual and the sum likewise; weight float32
 * [C], or NULL for ones.  residual NULL: x itself is normalised (sum must be NULL).
 * inverse [M] float32: 1 / sqrt(mean + eps), for the gradient (NULL: not wanted).
 */
int m4sl_rms_forward(const void* x, int x_bf16, const void* residual, int residual_bf16,
                     const float* weight, long M, int C, float eps, void* output, void* sum,
                     float* inverse, void* stream);

/*
 * The same with the result in 8 bits (e4m3: 4 exponent bits, 3 mantissa bits, no
 * infinities): each `block` channels of a row (the last may be shorter) have a scale,
 * max |y| / 448 but at least 2^-126, and output = y / scale, rounded to nearest.
 * output [M,C] bytes, scale [M, ceil(C / block)] float32.  block: a power of two in
 * 32..512, or at least C for one scale a row.  A NaN in a block makes its scale and all its
 * values NaN.
 */
int m4sl_rms_e4m3(const void* x, int x_bf16, const void* residual, int residual_bf16,
                  const float* weight, long M, int C, float eps, int block, void* output,
                  float* scale, void* sum, void* stream);

/*
 * Its gradient (of m4sl_rms_forward), from `sum` (x itself where there was no
 * residual), the inverse, d_output [M,C] in x's type and d_sum [M,C] in the sum's type
 * (NULL: zero).  d_x in x's type and d_residual in the sum's (the same numbers), d_weight
 * float32 [C], each NULL if not wanted.
 */
size_t m4sl_rms_backward_workspace_bytes(long M, int C);
int m4sl_rms_backward(const void* sum, int sum_bf16, const float* weight, const float* inverse,
                      const void* d_output, int x_bf16, const void* d_sum, long M, int C,
                      void* d_x, void* d_residual, float* d_weight, void* workspace,
                      size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif

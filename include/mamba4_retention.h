/*
 * mamba4_retention.h -- C ABI of the MI355X (gfx950) retention layer's
 * operators: decayed linear attention over prompts and training batches, its
 * gradient, and its step for single tokens; group normalisation with an
 * activation or a gate; the scaled embedding lookup (the library that also
 * holds mamba4_memread.h).
 *
 * Plain pointers and sizes only; every buffer is on the device and owned by
 * the caller.  `stream` is a hipStream_t passed as void* (NULL = the null
 * stream).  No function allocates, frees or synchronises.  Return values are
 * those of mamba4_memread.h (M4MR_OK, M4MR_EINVAL with nothing launched,
 * M4MR_EHIP); m4mr_last_error() gives the message.
 */
#ifndef MAMBA4_RETENTION_H
#define MAMBA4_RETENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Largest key and value width of the linear attention. */
#define M4RT_MAX_WIDTH 128

/*
 * Rows [B,T,heads,width] with unit stride along the width and strides in
 * elements along the others (the token stride is not read by
 * m4rt_attention_step).  `heads` divides the attention's H: head h reads row
 * h / (H / heads).  The token stride is at least `width` and 64 of it less
 * than 2^31 bytes.
 */
typedef struct {
  const void* data;
  long batch_stride, token_stride, head_stride;
  int heads, width;
} m4rt_rows;

/* The queries, keys and values of a call, in this order. */
typedef struct {
  m4rt_rows q, k, v;
} m4rt_qkv;

/*
 * Linear attention with a decay for each head.
 *   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
 *
 * q, k [B,T,.,N], v [B,T,.,P] in float32, or bfloat16 if `bf16` is not zero;
 * N, P in 1..M4RT_MAX_WIDTH.  log_decay: float32, [B,T,H] if `per_token` is not
 * zero, else [H].  lengths [B] int32, or NULL: tokens at lengths[b] and after
 * are absent (their rows are not read into any result, their output is zero; lengths
 * outside 0..T are clamped).  initial [B,H,N,P] float32, or NULL for zeros.
 * output [B,T,H,P] in v's type; state [B,H,N,P] float32, after the last
 * token, or NULL.
 *
 * Sums, states and decays are held in float32 or more.  What is computed on the way
 * and multiplied again (the scores, the state, the weighted keys) enters the products
 * as three bfloat16 parts, all its bits, where the result is float32, and as two
 * where it is rounded to bfloat16.  A row's result does not depend on the batch
 * size (at the same T).  A log decay of -infinity (or any that
 * underflows) drops what came before exactly.  An infinity or NaN in a row that is
 * present reaches what the recurrence carries it to, as NaN or an infinity: a value its
 * column of the outputs from its token on, a key every column of them, a query its own
 * output.  Others keep their bits.  (Float32 numbers beyond 3.39e38, which round to an
 * infinite bfloat16, count as infinite.)
 */
size_t m4rt_attention_workspace_bytes(const m4rt_qkv* rows, int bf16, int B, int T, int H);
int m4rt_attention_forward(const m4rt_qkv* rows, int bf16, const float* log_decay, int per_token,
                           const int* lengths, const float* initial, float scale, int B, int T,
                           int H, void* output, float* state, void* workspace,
                           size_t workspace_bytes, void* stream);

/*
 * Its gradient, from the cotangents d_output [B,T,H,P] in the inputs' type and
 * d_state [B,H,N,P] (NULL: zero).  state: the forward's final state, required
 * where both d_state and d_log_decay are given.  d_q, d_k, d_v:
 * [B,T,heads,width] in the inputs' type, contiguous; d_log_decay float32,
 * [B,T,H] if per_token else [H], or NULL; d_initial [B,H,N,P], or NULL.
 * Gradients of shared heads are summed in float32 and rounded once.  `decays` of
 * the workspace's size: whether d_log_decay is wanted.  Infinities and NaN in q, k, v
 * and d_output reach d_q, d_k and d_v as the recurrences of these carry them, and any
 * of d_log_decay of their batch row and head.
 */
size_t m4rt_attention_backward_workspace_bytes(const m4rt_qkv* rows, const void* d_output,
                                               int bf16, int B, int T, int H, int decays);
int m4rt_attention_backward(const m4rt_qkv* rows, int bf16, const float* log_decay,
                            int per_token, const int* lengths, const float* initial, float scale,
                            int B, int T, int H, const void* d_output, const float* d_state,
                            const float* state, void* d_q, void* d_k, void* d_v, float* d_log_decay,
                            float* d_initial, void* workspace, size_t workspace_bytes,
                            void* stream);

/*
 * One token: state [B,H,N,P] float32 to new_state (which may be state itself:
 * in place) and output [B,H,P] in v's type.  log_decay [B,H] if per_token,
 * else [H].  active [B] bytes, or NULL: a row whose byte is zero keeps its
 * state and its output is zero.
 */
int m4rt_attention_step(const m4rt_qkv* rows, int bf16, const float* log_decay, int per_token,
                        const uint8_t* active, float scale, int B, int H, const float* state,
                        float* new_state, void* output, void* stream);

#define M4RT_NONE 0
#define M4RT_SILU 1
#define M4RT_GELU 2 /* z Phi(z), by the error function */

/*
 * Group normalisation, channels last: x [M,L,C] in float32, or bfloat16 if
 * `bf16` is not zero; G groups of C/G channels.  Over a sample's L positions and
 * a group's channels n = (x - mean) / sqrt(variance + eps);
 * z = n weight + bias (weight, bias float32 [C], or NULL: ones, zeros).
 * output [M,L,C] in x's type: act(z), or z act(gate) with a gate [M,L,C] in x's
 * type (NULL: none).  stats: [M][G][2] float32, mean and 1 / sqrt(variance +
 * eps), for the gradient (NULL: not wanted).  Statistics and sums are float32, the
 * variance about the mean.  A sample's bits do not depend on M.
 */
size_t m4rt_norm_workspace_bytes(long M, int L, int C, int G, int bf16, int backward);
int m4rt_norm_forward(const void* x, const float* weight, const float* bias, const void* gate,
                      int bf16, long M, int L, int C, int G, int activation, float eps,
                      void* output, float* stats, void* workspace, size_t workspace_bytes,
                      void* stream);

/*
 * Its gradient, from d_output [M,L,C] in x's type and the forward's stats: d_x and
 * d_gate (with a gate) in x's type, d_weight and d_bias float32 [C], each NULL if
 * not wanted.
 */
int m4rt_norm_backward(const void* x, const float* weight, const float* bias, const void* gate,
                       const void* d_output, const float* stats, int bf16, long M, int L, int C,
                       int G, int activation, float eps, void* d_x, float* d_weight,
                       float* d_bias, void* d_gate, void* workspace, size_t workspace_bytes,
                       void* stream);

/*
 * Embedding: output [n,width] = scale * table[ids[i]], float32 or bfloat16 each;
 * table [rows,width].  ids int32, or int64 if `ids_int64`.  An id outside
 * 0..rows-1 (-1 for padding, say) gives a row of zeros.
 */
int m4rt_embedding_forward(const void* ids, int ids_int64, const void* table, int table_bf16,
                           long n, int rows, int width, float scale, void* output,
                           int output_bf16, void* stream);

/*
 * Its gradient: d_table [rows,width] = scale * the sums of d_output's rows by
 * id, every row written (ids outside the table add to none).  Sums are float32 in a
 * fixed order and rounded once.
 */
size_t m4rt_embedding_workspace_bytes(long n, int rows, int width);
int m4rt_embedding_backward(const void* ids, int ids_int64, const void* d_output, int output_bf16,
                            long n, int rows, int width, float scale, void* d_table,
                            int table_bf16, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif

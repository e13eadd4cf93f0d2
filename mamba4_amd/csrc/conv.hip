// The short causal convolution over each channel, for gfx950:
//   z_t = bias + sum over j < W of w[j] x_{t-W+1+j},   y_t = act(z_t).
// Gradient, with dz = dy act'(z):
//   dx_s = sum over j of w[j] dz_{s+W-1-j},   dw[j] = sum over t of dz_t x_{t-W+1+j}.
// It moves data and computes little: a thread holds a piece of four channels (forward:
// eight, where they are bfloat16) and walks a run of tokens, several rows in flight at a
// time, with the last W - 1 rows (backward: and the last W - 1 dz) in registers, so that
// rows are read once but for the W - 1 at a run's edge.  The backward forms z again
// instead of keeping it.  (Pieces of eight bfloat16 channels leave it two waves a SIMD:
// B16 T1024 D1536 W4 77 us for 55; the forward takes 30 us with them and 35 with four.)
// Those 30 and 55 us are 3.4 and 2.8 TB/s of the rows read and written once, float32 B8 T1000
// D768 12 and 23 us 4.1 and 3.2: it waits for memory, with vector instructions in half of
// the cycles.
#include <hip/hip_runtime.h>

#include "conv.hpp"

namespace cv {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned pack(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}

// V channels as they are in memory.
template <typename In, int V>
struct Piece;
template <>
struct Piece<float, 4> {
  f4 r = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ float get(int i) const { return r[i]; }
  __device__ __forceinline__ void set(const float (&v)[4]) { r = f4{v[0], v[1], v[2], v[3]}; }
};
template <>
struct Piece<float, 1> {
  float r = 0.f;
  __device__ __forceinline__ float get(int) const { return r; }
  __device__ __forceinline__ void set(const float (&v)[1]) { r = v[0]; }
};
template <>
struct Piece<bf16_t, 8> {
  u4 r = {0, 0, 0, 0};
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    r = u4{pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7])};
  }
};
template <>
struct Piece<bf16_t, 4> {
  u2 r = {0, 0};
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[4]) {
    r = u2{pack(v[0], v[1]), pack(v[2], v[3])};
  }
};
template <>
struct Piece<bf16_t, 1> {
  bf16_t r = 0;
  __device__ __forceinline__ float get(int) const { return __uint_as_float((unsigned)r << 16); }
  __device__ __forceinline__ void set(const float (&v)[1]) { r = (bf16_t)pack(v[0], 0.f); }
};

template <typename In, int V>
__device__ __forceinline__ Piece<In, V> load(const void* p, long at) {
  return *reinterpret_cast<const Piece<In, V>*>(static_cast<const In*>(p) + at);
}
template <typename In, int V>
__device__ __forceinline__ void store(void* p, long at, const Piece<In, V>& v) {
  *reinterpret_cast<Piece<In, V>*>(static_cast<In*>(p) + at) = v;
}
template <typename In, int V>
__device__ __forceinline__ void widen(const Piece<In, V>& p, float (&v)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = p.get(k);
}

__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

// Row t of a sequence: of `initial` before the first token, zeros where absent.
template <typename In, int V, int W>
__device__ __forceinline__ Piece<In, V> row(const Conv& a, long b, int c, int t, int len) {
  Piece<In, V> r;
  if (t >= 0) {
    if (t < len) r = load<In, V>(a.x, b * a.xb + t * a.xt + c);
  } else if (a.initial && t >= 1 - W) {
    r = load<In, V>(a.initial, (b * (W - 1) + t + W - 1) * a.D + c);
  }
  return r;
}

// The taps of a piece's channels, V * W consecutive floats, and the biases.
template <int V, int W>
__device__ __forceinline__ void load_taps(const float* weight, const float* bias, int c,
                                          float (&w)[W][V], float (&bv)[V]) {
  const float* from = weight + (long)c * W;
  if constexpr (V >= 4) {
    f4 r[V / 4 * W], b[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4 * W; ++i) r[i] = reinterpret_cast<const f4*>(from)[i];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      b[i] = f4{0.f, 0.f, 0.f, 0.f};
      if (bias) b[i] = reinterpret_cast<const f4*>(bias + c)[i];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      bv[k] = b[k / 4][k % 4];
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][k] = r[(k * W + j) / 4][(k * W + j) % 4];
    }
  } else {
    bv[0] = bias ? bias[c] : 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][0] = from[j];
  }
}

// ------------------------------------------------------------ forward

template <typename In, int V, int W>
__global__ __launch_bounds__(THREADS) void conv_kernel(Conv a) {
  constexpr int U = 8;
  const long i = (long)blockIdx.x * THREADS + threadIdx.x;
  const long line = i / a.cols;
  const int c = (int)(i - line * a.cols) * V;
  const long b = line / a.runs;
  if (b >= a.B) return;
  const int run = (int)(line - b * a.runs);
  const int begin = run * a.run, end = min(a.T, begin + a.run);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  float w[W][V], bias[V], x[U + W - 1][V];
  load_taps<V, W>(a.weight, a.bias, c, w, bias);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) widen(row<In, V, W>(a, b, c, begin - W + 1 + j, len), x[j]);
  for (int t0 = begin; t0 < end; t0 += U) {
    Piece<In, V> next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = row<In, V, W>(a, b, c, t0 + u, min(len, end));
#pragma unroll
    for (int u = 0; u < U; ++u) widen(next[u], x[W - 1 + u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float y[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float z = bias[k];
#pragma unroll
        for (int j = 0; j < W; ++j) z = fmaf(w[j][k], x[u + j][k], z);
        if (a.act == SILU) z *= sigmoid(z);
        y[k] = t0 + u < len ? z : 0.f;
      }
      Piece<In, V> p;
      p.set(y);
      if (t0 + u < end) store<In, V>(a.y, (b * a.T + t0 + u) * a.D + c, p);
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) x[j][k] = x[U + j][k];
  }
  if (W > 1 && run == 0 && a.state)
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      store<In, V>(a.state, (b * (W - 1) + j) * a.D + c,
                   row<In, V, W>(a, b, c, len - W + 1 + j, len));
}

// ------------------------------------------------------------ backward

// A block keeps to its columns and walks lines (runs of rows), so that the sums of dw
// and the bias's gradient stay in registers.
template <typename In, int V, int W>
__global__ __launch_bounds__(THREADS) void conv_backward_kernel(Conv a) {
  constexpr int U = 4;
  __shared__ float fold[THREADS];
  const int wide = THREADS / a.lines;
  const int col = threadIdx.x % wide, lane = threadIdx.x / wide;
  const int c = (blockIdx.y * wide + col) * V;
  const bool on = c < a.D;
  float w[W][V], bias[V], dw[W][V], db[V];
  if (on) load_taps<V, W>(a.weight, a.bias, c, w, bias);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    db[k] = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][k] = 0.f;
  }
  const long lines = (long)a.B * a.runs;
  for (long line = (long)blockIdx.x * a.lines + lane; on && line < lines;
       line += (long)gridDim.x * a.lines) {
    const long b = line / a.runs;
    const int run = (int)(line - b * a.runs);
    const int begin = run * a.run, end = min(a.T, begin + a.run);
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    float x[U + W - 1][V], dz[U + W - 1][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      widen(row<In, V, W>(a, b, c, begin - W + 1 + j, len), x[j]);
#pragma unroll
      for (int k = 0; k < V; ++k) dz[j][k] = 0.f;
    }
    for (int t0 = begin; t0 < end + W - 1; t0 += U) {
      Piece<In, V> nx[U], ny[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u;
        nx[u] = row<In, V, W>(a, b, c, t, len);
        if (t < len) ny[u] = load<In, V>(a.dy, (b * a.T + t) * a.D + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u;
        widen(nx[u], x[W - 1 + u]);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float d = ny[u].get(k);
          if (a.act == SILU) {
            float z = bias[k];
#pragma unroll
            for (int j = 0; j < W; ++j) z = fmaf(w[j][k], x[u + j][k], z);
            const float s = sigmoid(z);
            d *= s * fmaf(z, 1.f - s, 1.f);
          }
          d = t < len ? d : 0.f;
          dz[W - 1 + u][k] = d;
        }
        // (The next run's tokens are its own to sum up.)
        if (t < end) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            db[k] += dz[W - 1 + u][k];
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j][k] = fmaf(dz[W - 1 + u][k], x[u + j][k], dw[j][k]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = t0 + u - W + 1;
        if (s >= end || (s < begin && s >= 0)) continue;
        float dx[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          dx[k] = 0.f;
#pragma unroll
          for (int j = 0; j < W; ++j) dx[k] = fmaf(w[j][k], dz[W - 1 + u - j][k], dx[k]);
        }
        if (a.dstate && s < len && s > len - W) {
          const Piece<In, V> more =
              load<In, V>(a.dstate, (b * (W - 1) + s - (len - W + 1)) * a.D + c);
#pragma unroll
          for (int k = 0; k < V; ++k) dx[k] += more.get(k);
        }
        Piece<In, V> p;
        p.set(dx);
        if (s >= 0) {
          if (a.dx) store<In, V>(a.dx, (b * a.T + s) * a.D + c, p);
        } else if (run == 0 && a.dinitial) {
          store<In, V>(a.dinitial, (b * (W - 1) + s + W - 1) * a.D + c, p);
        }
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          x[j][k] = x[U + j][k];
          dz[j][k] = dz[U + j][k];
        }
    }
  }
  if (!a.part) return;
  // The block's sums: its lines of one column in order.
#pragma unroll
  for (int j = 0; j <= W; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float mine = j < W ? dw[j < W ? j : 0][k] : db[k];
      float s = mine;
      if (a.lines > 1) {
        __syncthreads();
        fold[threadIdx.x] = mine;
        __syncthreads();
        if (lane == 0)
          for (int l = 1; l < a.lines; ++l) s += fold[l * wide + col];
      }
      if (lane == 0 && on) a.part[((long)blockIdx.x * (W + 1) + j) * a.D + c + k] = s;
    }
}

// Sums of the blocks' parts [rows][W + 1][D], in 16 slices of the rows joined in their
// order, to dweight [D,W] and dbias [D].  Latency: 4 us.
__global__ __launch_bounds__(1024) void conv_join_kernel(const float* part, int rows, int W,
                                                         int D, float* dweight, float* dbias) {
  __shared__ float fold[1024];
  const int col = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int d = blockIdx.x * 64 + col, j = blockIdx.y;
  const long stride = (long)(W + 1) * D;
  const int each = (rows + 15) / 16, last = min(rows, (slice + 1) * each);
  float s = 0.f;
  if (d < D)
    for (int r = slice * each; r < last; ++r) s += part[r * stride + (long)j * D + d];
  fold[threadIdx.x] = s;
  __syncthreads();
  if (slice || d >= D) return;
  for (int i = 1; i < 16; ++i) s += fold[i * 64 + col];
  if (j < W) {
    if (dweight) dweight[(long)d * W + j] = s;
  } else if (dbias) {
    dbias[d] = s;
  }
}

// ------------------------------------------------------------ one token

// Bound by memory; a thread takes ROWS batch rows, whose loads are in flight together, with
// the taps of its channels in registers (2,048 rows of 1536 bfloat16, W4: one row 25 us,
// four 10.4, 4.8 TB/s).
template <typename In, int V, int W, int ROWS>
__global__ __launch_bounds__(THREADS) void conv_step_kernel(Step a) {
  const int rows = blockIdx.x / a.blocks;
  const int i = (blockIdx.x - rows * a.blocks) * THREADS + threadIdx.x;
  if (i >= a.cols) return;
  const int c = i * V;
  const long first = (long)rows * ROWS;
  Piece<In, V> x[ROWS][W];
  bool on[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    const long b = first + m;
    on[m] = b < a.B && (!a.active || a.active[b]);
    if (!on[m] && (b >= a.B || a.new_state == a.state)) continue;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) x[m][j] = load<In, V>(a.state, (b * (W - 1) + j) * a.D + c);
    if (on[m]) x[m][W - 1] = load<In, V>(a.x, b * a.xb + c);
  }
  float w[W][V], bias[V];
  load_taps<V, W>(a.weight, a.bias, c, w, bias);
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    const long b = first + m;
    if (b >= a.B) return;
    float y[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float z = bias[k];
#pragma unroll
      for (int j = 0; j < W; ++j) z = fmaf(w[j][k], x[m][j].get(k), z);
      if (a.act == SILU) z *= sigmoid(z);
      y[k] = on[m] ? z : 0.f;
    }
    Piece<In, V> p;
    p.set(y);
    store<In, V>(a.y, b * a.D + c, p);
    if (on[m] || a.new_state != a.state)
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        store<In, V>(a.new_state, (b * (W - 1) + j) * a.D + c, on[m] ? x[m][j + 1] : x[m][j]);
  }
}

#define M4SL_CONV_TAPS(In, V, W)                                 \
  template __global__ void conv_kernel<In, V, W>(Conv);          \
  template __global__ void conv_backward_kernel<In, V, W>(Conv); \
  template __global__ void conv_step_kernel<In, V, W, 1>(Step);  \
  template __global__ void conv_step_kernel<In, V, W, 4>(Step);
#define M4SL_CONV_FORWARD(In, V, W) template __global__ void conv_kernel<In, V, W>(Conv);
#define M4SL_CONV(TAPS, In, V) \
  TAPS(In, V, 1)               \
  TAPS(In, V, 2)               \
  TAPS(In, V, 3)               \
  TAPS(In, V, 4)               \
  TAPS(In, V, 5)               \
  TAPS(In, V, 6)               \
  TAPS(In, V, 7)               \
  TAPS(In, V, 8)
M4SL_CONV(M4SL_CONV_TAPS, float, 4)
M4SL_CONV(M4SL_CONV_TAPS, float, 1)
M4SL_CONV(M4SL_CONV_TAPS, bf16_t, 4)
M4SL_CONV(M4SL_CONV_TAPS, bf16_t, 1)
M4SL_CONV(M4SL_CONV_FORWARD, bf16_t, 8)

}  // namespace cv

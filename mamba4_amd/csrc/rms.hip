// Root-mean-square norm of x + residual, for gfx950:
//   s = x + residual (rounded to the residual's type),  n = s / sqrt(mean(s^2) + eps),
//   y = n weight, in x's type or as 8-bit values with a scale for each block of channels.
// Gradient, with dn = dy weight:
//   ds = (dn - n mean(dn n)) / sqrt(mean(s^2) + eps) + dsum,  dweight = sum of dy n.
// It moves data and computes little: a row is read once, in 16-byte pieces of its
// narrowest type, and stays in the registers of its lanes (of one wave up to 1024
// channels) between the statistics and their use.  Blocks walk rows, so that the weights
// and the sums of dweight stay in registers too.  How a row is spread depends on C
// alone, so that its bits do not depend on how many rows there are.  16,384 rows of 768
// bfloat16 with a float32 residual: forward 28 us, 5.5 TB/s, gradient 42, 4.8; to 8 bits
// 4,096 channels with a bfloat16 residual: 92 us, 5.1 TB/s (a large copy's rate).
#include <hip/hip_runtime.h>

#include "rms.hpp"

namespace rn {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned pack(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}

// V values in memory: whole pieces (V = 8), or one element.
template <typename T, int V>
struct Piece;
template <>
struct Piece<float, 8> {
  f4 r[2];
  __device__ __forceinline__ void zero() { r[0] = r[1] = f4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ float get(int i) const { return r[i >> 2][i & 3]; }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    r[0] = f4{v[0], v[1], v[2], v[3]};
    r[1] = f4{v[4], v[5], v[6], v[7]};
  }
};
template <>
struct Piece<bf16_t, 8> {
  u4 r;
  __device__ __forceinline__ void zero() { r = u4{0, 0, 0, 0}; }
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    r = u4{pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7])};
  }
};
template <>
struct Piece<float, 1> {
  float r;
  __device__ __forceinline__ void zero() { r = 0.f; }
  __device__ __forceinline__ float get(int) const { return r; }
  __device__ __forceinline__ void set(const float (&v)[1]) { r = v[0]; }
};
template <>
struct Piece<bf16_t, 1> {
  bf16_t r;
  __device__ __forceinline__ void zero() { r = 0; }
  __device__ __forceinline__ float get(int) const { return __uint_as_float((unsigned)r << 16); }
  __device__ __forceinline__ void set(const float (&v)[1]) { r = (bf16_t)pack(v[0], 0.f); }
};

template <typename T, int V>
__device__ __forceinline__ Piece<T, V> load(const void* p, long at) {
  return *reinterpret_cast<const Piece<T, V>*>(static_cast<const T*>(p) + at);
}
template <typename T, int V>
__device__ __forceinline__ void store(void* p, long at, const float (&v)[V]) {
  Piece<T, V> w;
  w.set(v);
  *reinterpret_cast<Piece<T, V>*>(static_cast<T*>(p) + at) = w;
}

// A joined over the aligned 2^k lanes of a wave that share a row or a scale.
template <typename F>
__device__ __forceinline__ unsigned group_join(unsigned x, int lanes, F&& join) {
  const auto dpp = [](unsigned v, auto ctrl) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl(), 0xf, 0xf, true);
  };
  if (lanes > 1) x = join(x, dpp(x, [] { return 0xB1; }));   // quad_perm [1,0,3,2]
  if (lanes > 2) x = join(x, dpp(x, [] { return 0x4E; }));   // quad_perm [2,3,0,1]
  if (lanes > 4) x = join(x, dpp(x, [] { return 0x141; }));  // row_half_mirror
  if (lanes > 8) x = join(x, dpp(x, [] { return 0x140; }));  // row_mirror
  if (lanes > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = join(a[0], a[1]);
  }
  if (lanes > 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = join(a[0], a[1]);
  }
  return x;
}

__device__ __forceinline__ unsigned add_bits(unsigned a, unsigned b) {
  return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
// Of magnitudes, whose order as numbers is that of their bits, with NaN above infinity.
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }

// The sum over a row's lanes: within the wave, then over its waves in their order.
__device__ __forceinline__ float row_sum(float x, int lanes, float* fold) {
  x = __uint_as_float(group_join(__float_as_uint(x), lanes < 64 ? lanes : 64, add_bits));
  if (lanes <= 64) return x;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) fold[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < lanes / 64; ++w) s += fold[w];
  return s;
}

// Where a thread works: row rr of the block's, pieces lane, lane + lanes, ...
template <int V, int IT>
struct Place {
  int rr, lane;
  bool on[IT];
  __device__ __forceinline__ Place(const Rms& a) {
    rr = threadIdx.x / a.lanes;
    lane = threadIdx.x - rr * a.lanes;
#pragma unroll
    for (int i = 0; i < IT; ++i) on[i] = rr < a.rows && (i * a.lanes + lane) * V < a.C;
  }
  __device__ __forceinline__ int channel(const Rms& a, int i) const {
    return (i * a.lanes + lane) * V;
  }
};

template <int V, int IT>
__device__ __forceinline__ void load_weight(const Rms& a, const Place<V, IT>& p,
                                            float (&w)[IT][V]) {
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    Piece<float, V> v;
    v.zero();
    if (a.weight && p.on[i]) v = load<float, V>(a.weight, p.channel(a, i));
#pragma unroll
    for (int k = 0; k < V; ++k) w[i][k] = a.weight ? v.get(k) : 1.f;
  }
}

// ------------------------------------------------------------ forward

// E4M3: the result in 8 bits.  The largest magnitudes of a block of channels join in its
// lanes, then in LDS (a maximum: the order does not matter).
template <typename X, typename R, int V, int IT, bool E4M3>
__global__ __launch_bounds__(1024) void rms_kernel(Rms a) {
  __shared__ float fold[16];
  __shared__ unsigned slots[E4M3 ? SLOTS : 1];
  const Place<V, IT> p(a);
  float w[IT][V];
  load_weight(a, p, w);
  const float share = 1.f / a.C;
  const int slot = p.rr * a.blocks;
  for (long base = (long)blockIdx.x * a.rows; base < a.M; base += (long)gridDim.x * a.rows) {
    const long m = base + p.rr;
    const bool here = m < a.M;
    Piece<X, V> xv[IT];
    Piece<R, V> rv[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      xv[i].zero();
      rv[i].zero();
      if (here && p.on[i]) {
        const long at = m * a.C + p.channel(a, i);
        xv[i] = load<X, V>(a.x, at);
        if (a.residual) rv[i] = load<R, V>(a.residual, at);
      }
    }
    if (E4M3) {
      __syncthreads();
      for (int i = threadIdx.x; i < a.rows * a.blocks; i += blockDim.x) slots[i] = 0;
    }
    float s[IT][V], squares = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) s[i][k] = xv[i].get(k) + rv[i].get(k);
      if (a.residual) {
        // The sum is normalised as it is kept.
        Piece<R, V> kept;
        kept.set(s[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) s[i][k] = kept.get(k);
        if (a.sum && here && p.on[i])
          *reinterpret_cast<Piece<R, V>*>(static_cast<R*>(a.sum) + m * a.C + p.channel(a, i)) =
              kept;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) squares = fmaf(s[i][k], s[i][k], squares);
    }
    const float inverse =
        __builtin_amdgcn_rsqf(fmaf(row_sum(squares, a.lanes, fold), share, a.eps));
    if (a.inverse && here && p.lane == 0) a.inverse[m] = inverse;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) s[i][k] = s[i][k] * inverse * w[i][k];
    if constexpr (!E4M3) {
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (here && p.on[i]) store<X, V>(a.y, m * a.C + p.channel(a, i), s[i]);
    } else {
      if (a.lanes <= 64) __syncthreads();
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        unsigned most = 0;
#pragma unroll
        for (int k = 0; k < V; ++k)
          most = larger(most, __float_as_uint(s[i][k]) & 0x7fffffffu);
        most = group_join(p.on[i] ? most : 0, a.group, larger);
        if ((threadIdx.x & (a.group - 1)) == 0 && p.on[i])
          atomicMax(&slots[slot + p.channel(a, i) / a.block], most);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        if (!(here && p.on[i])) continue;
        const int c = p.channel(a, i), n = c / a.block;
        const float most = __uint_as_float(slots[slot + n]) * (1.f / 448.f);
        // (A NaN stays one.)
        const float scale = most < 1.17549435e-38f ? 1.17549435e-38f : most;
        const float inv = __builtin_amdgcn_rcpf(scale);
        if (c - n * a.block < V) a.scale[m * a.blocks + n] = scale;
        unsigned char* to = static_cast<unsigned char*>(a.y) + m * a.C + c;
        if constexpr (V == 8) {
          u2 q;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(s[i][4 * h] * inv, s[i][4 * h + 1] * inv, 0,
                                                    false);
            v = __builtin_amdgcn_cvt_pk_fp8_f32(s[i][4 * h + 2] * inv, s[i][4 * h + 3] * inv, v,
                                                true);
            q[h] = (unsigned)v;
          }
          *reinterpret_cast<u2*>(to) = q;
        } else {
          *to = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(s[i][0] * inv, 0.f, 0, false);
        }
      }
    }
  }
}

// ------------------------------------------------------------ backward

template <typename X, typename R, int V, int IT>
__global__ __launch_bounds__(1024) void rms_backward_kernel(Rms a) {
  __shared__ float fold[1024];
  const Place<V, IT> p(a);
  float w[IT][V], dw[IT][V];
  load_weight(a, p, w);
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = 0.f;
  const float share = 1.f / a.C;
  for (long base = (long)blockIdx.x * a.rows; base < a.M; base += (long)gridDim.x * a.rows) {
    const long m = base + p.rr;
    const bool here = m < a.M;
    Piece<R, V> sv[IT], ev[IT];
    Piece<X, V> dv[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      sv[i].zero();
      ev[i].zero();
      dv[i].zero();
      if (here && p.on[i]) {
        const long at = m * a.C + p.channel(a, i);
        sv[i] = load<R, V>(a.x, at);
        dv[i] = load<X, V>(a.dy, at);
        if (a.dsum) ev[i] = load<R, V>(a.dsum, at);
      }
    }
    const float inverse = here && p.rr < a.rows ? a.inverse[m] : 0.f;
    float n[IT][V], dn[IT][V], dot = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float dy = dv[i].get(k);
        n[i][k] = sv[i].get(k) * inverse;
        dn[i][k] = dy * w[i][k];
        dot = fmaf(dn[i][k], n[i][k], dot);
        dw[i][k] = fmaf(dy, n[i][k], dw[i][k]);
      }
    const float mean = row_sum(dot, a.lanes, fold) * share;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (!(here && p.on[i])) continue;
      float ds[V];
#pragma unroll
      for (int k = 0; k < V; ++k)
        ds[k] = fmaf(inverse, dn[i][k] - n[i][k] * mean, ev[i].get(k));
      const long at = m * a.C + p.channel(a, i);
      if (a.dx) store<X, V>(a.dx, at, ds);
      if (a.dresidual) store<R, V>(a.dresidual, at, ds);
    }
  }
  if (!a.part) return;
  // The block's sums: its rows' threads of one column in order.
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float s = dw[i][k];
      if (a.rows > 1) {
        __syncthreads();
        fold[threadIdx.x] = s;
        __syncthreads();
        if (p.rr == 0)
          for (int j = 1; j < a.rows; ++j) s += fold[j * a.lanes + p.lane];
      }
      if (p.rr == 0 && p.on[i]) a.part[(long)blockIdx.x * a.C + p.channel(a, i) + k] = s;
    }
}

// Sums of the blocks' parts [rows][C], in 16 slices of the rows joined in their order.
// Latency: 5 us (one slice 37).
__global__ __launch_bounds__(1024) void rms_join_kernel(const float* part, int rows, int C,
                                                        float* dweight) {
  __shared__ float fold[1024];
  const int col = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + col;
  const int each = (rows + 15) / 16, last = min(rows, (slice + 1) * each);
  float s = 0.f;
  if (c < C)
    for (int r = slice * each; r < last; ++r) s += part[(long)r * C + c];
  fold[threadIdx.x] = s;
  __syncthreads();
  if (slice || c >= C) return;
  for (int i = 1; i < 16; ++i) s += fold[i * 64 + col];
  dweight[c] = s;
}

#define M4SL_RMS_ONE(X, R, V, IT)                               \
  template __global__ void rms_kernel<X, R, V, IT, false>(Rms); \
  template __global__ void rms_kernel<X, R, V, IT, true>(Rms);  \
  template __global__ void rms_backward_kernel<X, R, V, IT>(Rms);
#define M4SL_RMS(X, R)      \
  M4SL_RMS_ONE(X, R, 8, 1)  \
  M4SL_RMS_ONE(X, R, 8, 2)  \
  M4SL_RMS_ONE(X, R, 8, 4)  \
  M4SL_RMS_ONE(X, R, 1, 1)  \
  M4SL_RMS_ONE(X, R, 1, 4)  \
  M4SL_RMS_ONE(X, R, 1, 8)  \
  M4SL_RMS_ONE(X, R, 1, 32)
M4SL_RMS(float, float)
M4SL_RMS(float, bf16_t)
M4SL_RMS(bf16_t, float)
M4SL_RMS(bf16_t, bf16_t)

}  // namespace rn

// Group normalisation with an activation or a gate, channels last, for gfx950.
//
// x [M, L, C], G groups of D = C / G channels; over a sample's L positions and a
// group's D channels
//   n = (x - mean) / sqrt(var + eps),  z = n weight + bias,
//   y = act(z),  or  y = z act(gate).
// Gradient, with dz = dy act'(z) (or dy act(gate), and dgate = dy z act'(gate))
// and dn = dz weight:
//   dx = (dn - mean(dn) - n mean(dn n)) / sqrt(var + eps),
//   dweight = sum of dz n, dbias = sum of dz over samples and positions.
// All of it moves data and computes little, so each kernel reads its arrays
// once in 16-byte pieces, keeps them in registers between the statistics and
// their use, and sums in float32 (variances about the mean, never as a
// difference of squares).
//
// One position (the heads of a token): a group is D consecutive elements, and
// lanes / of a wave hold it; a block keeps to its channels and walks rows, so
// the weights and the column sums of the gradient stay in registers.
// Several positions: blocks take ranges of positions; partial statistics
// (count, mean, sum of squares about it) are joined pairwise.
#include <hip/hip_runtime.h>

#include "norm.hpp"

namespace gn {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned pack(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}
__device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

template <typename T, int V>
struct Vec;
template <int V>
struct Vec<float, V> {
  typedef float raw __attribute__((ext_vector_type(V)));
  raw r;
  __device__ __forceinline__ void load(const void* p, long i) {
    r = *reinterpret_cast<const raw*>(static_cast<const float*>(p) + i);
  }
  __device__ __forceinline__ void zero() { r = raw(0.f); }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (V == 1) return r[0];
    else return r[i];
  }
  __device__ __forceinline__ static void store(void* p, long i, const float (&v)[V]) {
    raw r;
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = v[k];
    *reinterpret_cast<raw*>(static_cast<float*>(p) + i) = r;
  }
};
template <int V>
struct Vec<bf16_t, V> {
  typedef unsigned raw __attribute__((ext_vector_type(V / 2)));
  raw r;
  __device__ __forceinline__ void load(const void* p, long i) {
    r = *reinterpret_cast<const raw*>(static_cast<const bf16_t*>(p) + i);
  }
  __device__ __forceinline__ void zero() { r = raw(0u); }
  __device__ __forceinline__ float get(int i) const {
    return i & 1 ? high(r[i >> 1]) : low(r[i >> 1]);
  }
  __device__ __forceinline__ static void store(void* p, long i, const float (&v)[V]) {
    raw r;
#pragma unroll
    for (int k = 0; k < V / 2; ++k) r[k] = pack(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<raw*>(static_cast<bf16_t*>(p) + i) = r;
  }
};
template <>
struct Vec<bf16_t, 1> {
  bf16_t r;
  __device__ __forceinline__ void load(const void* p, long i) {
    r = static_cast<const bf16_t*>(p)[i];
  }
  __device__ __forceinline__ void zero() { r = 0; }
  __device__ __forceinline__ float get(int) const { return __uint_as_float((unsigned)r << 16); }
  __device__ __forceinline__ static void store(void* p, long i, const float (&v)[1]) {
    static_cast<bf16_t*>(p)[i] = (bf16_t)pack(v[0], 0.f);
  }
};

// Sum over the aligned 2^k lanes that share a group.
__device__ __forceinline__ float group_sum(float x, int lanes) {
  const auto dpp = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl(), 0xf, 0xf, true));
  };
  if (lanes > 1) x += dpp(x, [] { return 0xB1; });   // quad_perm [1,0,3,2]
  if (lanes > 2) x += dpp(x, [] { return 0x4E; });   // quad_perm [2,3,0,1]
  if (lanes > 4) x += dpp(x, [] { return 0x141; });  // row_half_mirror
  if (lanes > 8) x += dpp(x, [] { return 0x140; });  // row_mirror
  if (lanes > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if (lanes > 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return x;
}

__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

// An activation's value and derivative.
__device__ __forceinline__ float activate(float z, int act, float* slope) {
  if (act == SILU) {
    const float s = sigmoid(z);
    *slope = s * fmaf(z, 1.f - s, 1.f);
    return z * s;
  }
  if (act == GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678f * z);
    *slope = fmaf(z * 0.39894228f, __builtin_amdgcn_exp2f(-0.72134752f * z * z), cdf);
    return z * cdf;
  }
  *slope = 1.f;
  return z;
}

// The same of several values, with one choice of the activation.
template <int V>
__device__ __forceinline__ void activate(const float (&z)[V], int act, float (&y)[V],
                                         float (&slope)[V]) {
  if (act == SILU) {
#pragma unroll
    for (int k = 0; k < V; ++k) y[k] = activate(z[k], SILU, &slope[k]);
  } else if (act == GELU) {
#pragma unroll
    for (int k = 0; k < V; ++k) y[k] = activate(z[k], GELU, &slope[k]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) y[k] = activate(z[k], NONE, &slope[k]);
  }
}

// ---------------------------------------------------------------- one position

// Bound by memory: 16384 x 1536 bfloat16 with a gate 35 us forward (4.3 TB/s), 64
// backward (3.9), and 5 for the columns' sums.
template <typename In, int V, int IT, bool BWD>
__global__ __launch_bounds__(ROW_THREADS) void norm_rows_kernel(Norm a) {
  __shared__ float fold[BWD ? ROW_THREADS : 1];
  const int tid = threadIdx.x, across = a.groups * a.lanes;
  const int rr = tid / across, rem = tid - rr * across;
  const int local = rem / a.lanes, lane = rem - local * a.lanes;
  const int group = blockIdx.y * a.groups + local;
  const bool member = rr < a.rows && group < a.G;
  const int vecs = a.D / V;
  float w[IT][V], bias[IT][V], dw[IT][V], db[IT][V];
  bool on[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int v = i * a.lanes + lane;
    on[i] = member && v < vecs;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = group * a.D + v * V + k;
      w[i][k] = a.weight && on[i] ? a.weight[c] : 1.f;
      bias[i][k] = a.bias && on[i] ? a.bias[c] : 0.f;
      dw[i][k] = db[i][k] = 0.f;
    }
  }
  const float scale = 1.f / a.D;
  const long stride = (long)gridDim.x * a.rows;
  // The next row's pieces are on their way while a row is computed.
  Vec<In, V> xn[IT], gn[IT], dn_[IT];
  auto fetch = [&](long m) {
    const long at = m * a.C + group * a.D + lane * V;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      xn[i].zero();
      gn[i].zero();
      dn_[i].zero();
      if (m < a.M && on[i]) {
        xn[i].load(a.x, at + i * a.lanes * V);
        if (a.gate) gn[i].load(a.gate, at + i * a.lanes * V);
        if (BWD) dn_[i].load(a.dy, at + i * a.lanes * V);
      }
    }
  };
  fetch((long)blockIdx.x * a.rows + rr);
  for (long base = (long)blockIdx.x * a.rows; base < a.M; base += stride) {
    const long m = base + rr;
    const bool here = m < a.M;
    const long at = m * a.C + group * a.D + lane * V;
    Vec<In, V> xv[IT], gv[IT], dv[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      xv[i] = xn[i];
      gv[i] = gn[i];
      dv[i] = dn_[i];
    }
    fetch(m + stride);
    float n[IT][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        n[i][k] = xv[i].get(k);
        s += n[i][k];
      }
    const float mean = group_sum(s, a.lanes) * scale;
    // Again, for the mean's own rounding, which a small deviation about a large
    // mean feels.
    s = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        n[i][k] = on[i] ? n[i][k] - mean : 0.f;
        s += n[i][k];
      }
    const float rest = group_sum(s, a.lanes) * scale;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        n[i][k] = on[i] ? n[i][k] - rest : 0.f;
        s = fmaf(n[i][k], n[i][k], s);
      }
    const float inv = __builtin_amdgcn_rsqf(fmaf(group_sum(s, a.lanes), scale, a.eps));
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) n[i][k] *= inv;
    if constexpr (!BWD) {
      if (a.stats && here && member && lane == 0) {
        a.stats[(m * a.G + group) * 2] = mean + rest;
        a.stats[(m * a.G + group) * 2 + 1] = inv;
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        float z[V], u[V], y[V], slope[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          z[k] = fmaf(n[i][k], w[i][k], bias[i][k]);
          u[k] = a.gate ? gv[i].get(k) : z[k];
        }
        activate<V>(u, a.act, y, slope);
        if (a.gate) {
#pragma unroll
          for (int k = 0; k < V; ++k) y[k] *= z[k];
        }
        if (here && on[i]) Vec<In, V>::store(a.y, at + i * a.lanes * V, y);
      }
    } else {
      float dn[IT][V];
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        float z[V], u[V], y[V], slope[V], dz[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          z[k] = fmaf(n[i][k], w[i][k], bias[i][k]);
          u[k] = a.gate ? gv[i].get(k) : z[k];
        }
        activate<V>(u, a.act, y, slope);
        if (a.gate) {
          float dg[V];
#pragma unroll
          for (int k = 0; k < V; ++k) {
            dz[k] = dv[i].get(k) * y[k];
            dg[k] = dv[i].get(k) * z[k] * slope[k];
          }
          if (a.dgate && here && on[i])
            Vec<In, V>::store(a.dgate, at + i * a.lanes * V, dg);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) dz[k] = dv[i].get(k) * slope[k];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          dn[i][k] = dz[k] * w[i][k];
          s1 += dn[i][k];
          s2 = fmaf(dn[i][k], n[i][k], s2);
        }
        if (here) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            dw[i][k] = fmaf(dz[k], n[i][k], dw[i][k]);
            db[i][k] += dz[k];
          }
        }
      }
      s1 = group_sum(s1, a.lanes) * scale;
      s2 = group_sum(s2, a.lanes) * scale;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        float dx[V];
#pragma unroll
        for (int k = 0; k < V; ++k) dx[k] = inv * (dn[i][k] - s1 - n[i][k] * s2);
        if (a.dx && here && on[i]) Vec<In, V>::store(a.dx, at + i * a.lanes * V, dx);
      }
    }
  }
  if constexpr (BWD) {
    if (!a.part) return;
    // The block's column sums: its rows' threads of one column in order.
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int k = 0; k < 2 * V; ++k) {
        const float mine = k < V ? dw[i][k % V] : db[i][k % V];
        float s = mine;
        if (a.rows > 1) {
          __syncthreads();
          fold[tid] = mine;
          __syncthreads();
          if (rr == 0)
            for (int j = 1; j < a.rows; ++j) s += fold[j * across + rem];
        }
        if (rr == 0 && on[i]) {
          const int c = group * a.D + (i * a.lanes + lane) * V + k % V;
          a.part[((long)blockIdx.x * 2 + (k < V ? 0 : 1)) * a.C + c] = s;
        }
      }
  }
}

// Sums of `rows` partials [rows][2][C]: 16 columns a block, 64 threads of a
// column each every 64th row, joined in order.
__global__ __launch_bounds__(1024) void norm_columns_kernel(const float* part, int rows, int C,
                                                            float* dweight, float* dbias) {
  __shared__ float fold[64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  const int column = blockIdx.x * 16 + x;
  float s = 0.f;
  if (column < 2 * C) {
#pragma unroll 8
    for (int r = y; r < rows; r += 64) s += part[(long)r * 2 * C + column];
  }
  fold[y][x] = s;
  for (int h = 32; h > 0; h >>= 1) {
    __syncthreads();
    if (y < h) fold[y][x] += fold[y + h][x];
  }
  if (y == 0 && column < 2 * C) {
    if (column < C) {
      if (dweight) dweight[column] = fold[0][x];
    } else if (dbias) {
      dbias[column - C] = fold[0][x];
    }
  }
}

// ----------------------------------------------------------- several positions

// Statistics of some values: how many, their mean, the squares about it.
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float d = b.mean - a.mean, f = b.n / n;
  return Moments{n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
}
struct Pair {
  float a, b;
};
__device__ __forceinline__ Pair join(const Pair& x, const Pair& y) {
  return Pair{x.a + y.a, x.b + y.b};
}

// Joins the entries of each team (`team` threads, thread k of it) into its
// thread 0, in a fixed order; every thread receives the result.
template <typename T>
__device__ __forceinline__ T team_join(T mine, T* fold, int first, int k, int team, bool member) {
  const int at = first + k;
  __syncthreads();
  fold[threadIdx.x] = mine;
  __syncthreads();
  int s = 1;
  while (s < team) s <<= 1;
  for (s >>= 1; s > 0; s >>= 1) {
    if (member && k < s && k + s < team) fold[at] = join(fold[at], fold[at + s]);
    __syncthreads();
  }
  return fold[first];
}

// A block: positions of one sample, the channels of `span` groups (or a part
// of one).  Thread: one vector of channels and every rows-th position.  A group's
// threads are consecutive: thread = (group, row, vector).  Statistics are of `parts`
// ranges of the positions, joined in the same order whether a block takes one part
// (SUMS, then APPLY) or a whole sample (BOTH): a sample's bits do not depend on how
// many there are.  Blocks walk over the samples, blockIdx.y and every gridDim.y-th
// after it.  Bound by memory: 8 x
// 4000 x 512 float32 16 + 27 us forward, 25 + 33 backward (65 MB an array).
template <typename In, int V, bool BWD, int PHASE>
__global__ __launch_bounds__(POS_THREADS) void norm_positions_kernel(Norm a) {
  __shared__ Moments folded[POS_THREADS];
  Pair* pairs = reinterpret_cast<Pair*>(folded);
  const int tid = threadIdx.x;
  const int vecs = min(a.vecs, POS_THREADS), team = vecs * a.rows;
  const int local = tid / team, k = tid - local * team, first = local * team;
  const int rr = k / vecs, j = k - rr * vecs;
  const int unit = blockIdx.z * a.span + local;      // a group, or part of one
  const int group = unit / a.subs, sub = unit - group * a.subs;
  const int v = sub * POS_THREADS + j;
  const bool member = local < a.span && group < a.G;
  const bool on = member && v < a.vecs;
  const int per = (a.L + a.parts - 1) / a.parts;
  const int part0 = PHASE == BOTH ? 0 : blockIdx.x, part1 = PHASE == BOTH ? a.parts : part0 + 1;
  auto begin = [&](int part) { return (int)min((long)a.L, (long)part * per); };
  const int l0 = begin(part0), l1 = begin(part1);
  const long column = (long)group * a.D + v * V;
  const float count = (float)a.L * a.D;
  float w[V], bias[V], dw[V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = a.weight && on ? a.weight[column + i] : 1.f;
    bias[i] = a.bias && on ? a.bias[column + i] : 0.f;
    dw[i] = db[i] = 0.f;
  }
  constexpr int AHEAD = 4;
  for (long m = blockIdx.y; m < a.M; m += gridDim.y) {
    const long at = m * a.L * a.C + column;
    // Partial sums: [m][part][sub][group][4].
    auto slot = [&](int part, int s) {
      return a.sums + (((m * a.parts + part) * a.subs + s) * a.G + group) * 4;
    };
    float mean = 0.f, inv = 0.f;

    if constexpr (!BWD) {
      Moments mine{0.f, 0.f, 0.f};
      if constexpr (PHASE != APPLY) {
        for (int part = part0; part < part1; ++part) {
          const int end = begin(part + 1);
          mine = Moments{0.f, 0.f, 0.f};
          if (on)
            for (int l = begin(part) + rr; l < end; l += AHEAD * a.rows) {
              Vec<In, V> x[AHEAD];
              int have = 0;
#pragma unroll
              for (int i = 0; i < AHEAD; ++i) {
                x[i].zero();
                if (l + i * a.rows < end) {
                  x[i].load(a.x, at + (long)(l + i * a.rows) * a.C);
                  have = i + 1;
                }
              }
              float s = 0.f, q = 0.f;
#pragma unroll
              for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) s += x[i].get(e);
              const float c = s / (float)(have * V);
#pragma unroll
              for (int i = 0; i < AHEAD; ++i)
                if (i < have)
#pragma unroll
                  for (int e = 0; e < V; ++e) q = fmaf(x[i].get(e) - c, x[i].get(e) - c, q);
              mine = join(mine, Moments{(float)(have * V), c, q});
            }
          mine = team_join(mine, folded, first, k, team, member);
          if ((PHASE == SUMS || a.parts > 1) && member && k == 0) {
            float* s = slot(part, sub);
            s[0] = mine.n;
            s[1] = mine.mean;
            s[2] = mine.m2;
          }
        }
        if constexpr (PHASE == SUMS) continue;
      }
      if (PHASE == APPLY || a.parts > 1) {
        if (PHASE == BOTH) __syncthreads();  // the slots are written
        mine = Moments{0.f, 0.f, 0.f};
        if (member)
          for (int b = k; b < a.parts * a.subs; b += team) {
            const float* s = slot(b / a.subs, b % a.subs);
            mine = join(mine, Moments{s[0], s[1], s[2]});
          }
        mine = team_join(mine, folded, first, k, team, member);
      }
      mean = mine.mean;
      inv = 1.f / sqrtf(mine.m2 / count + a.eps);
      if (a.stats && member && k == 0 && sub == 0 && blockIdx.x == 0) {
        a.stats[(m * a.G + group) * 2] = mean;
        a.stats[(m * a.G + group) * 2 + 1] = inv;
      }
      if (on)
        for (int l = l0 + rr; l < l1; l += AHEAD * a.rows) {
          Vec<In, V> x[AHEAD], g[AHEAD];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i)
            if (l + i * a.rows < l1) {
              x[i].load(a.x, at + (long)(l + i * a.rows) * a.C);
              if (a.gate) g[i].load(a.gate, at + (long)(l + i * a.rows) * a.C);
            }
#pragma unroll
          for (int i = 0; i < AHEAD; ++i)
            if (l + i * a.rows < l1) {
              float z[V], u[V], y[V], slope[V];
#pragma unroll
              for (int e = 0; e < V; ++e) {
                z[e] = fmaf((x[i].get(e) - mean) * inv, w[e], bias[e]);
                u[e] = a.gate ? g[i].get(e) : z[e];
              }
              activate<V>(u, a.act, y, slope);
              if (a.gate) {
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] *= z[e];
              }
              Vec<In, V>::store(a.y, at + (long)(l + i * a.rows) * a.C, y);
            }
        }
    } else {
      if (member) {
        mean = a.stats[(m * a.G + group) * 2];
        inv = a.stats[(m * a.G + group) * 2 + 1];
      }
      Pair mine{0.f, 0.f};
      if constexpr (PHASE != APPLY) {
        for (int part = part0; part < part1; ++part) {
          const int end = begin(part + 1);
          mine = Pair{0.f, 0.f};
          float dws[V], dbs[V];  // of this part
#pragma unroll
          for (int e = 0; e < V; ++e) dws[e] = dbs[e] = 0.f;
          if (on)
            for (int l = begin(part) + rr; l < end; l += AHEAD * a.rows) {
              Vec<In, V> x[AHEAD], g[AHEAD], d[AHEAD];
#pragma unroll
              for (int i = 0; i < AHEAD; ++i)
                if (l + i * a.rows < end) {
                  const long p = at + (long)(l + i * a.rows) * a.C;
                  x[i].load(a.x, p);
                  d[i].load(a.dy, p);
                  if (a.gate) g[i].load(a.gate, p);
                }
#pragma unroll
              for (int i = 0; i < AHEAD; ++i)
                if (l + i * a.rows < end) {
                  float n[V], u[V], y[V], slope[V];
#pragma unroll
                  for (int e = 0; e < V; ++e) {
                    n[e] = (x[i].get(e) - mean) * inv;
                    u[e] = a.gate ? g[i].get(e) : fmaf(n[e], w[e], bias[e]);
                  }
                  activate<V>(u, a.act, y, slope);
#pragma unroll
                  for (int e = 0; e < V; ++e) {
                    const float dz = d[i].get(e) * (a.gate ? y[e] : slope[e]);
                    dws[e] = fmaf(dz, n[e], dws[e]);
                    dbs[e] += dz;
                  }
                }
            }
#pragma unroll
          for (int e = 0; e < V; ++e) {
            mine.a = fmaf(w[e], dbs[e], mine.a);
            mine.b = fmaf(w[e], dws[e], mine.b);
            dw[e] += dws[e];
            db[e] += dbs[e];
          }
          mine = team_join(mine, pairs, first, k, team, member);
          if ((PHASE == SUMS || a.parts > 1) && member && k == 0) {
            float* s = slot(part, sub);
            s[0] = mine.a;
            s[1] = mine.b;
          }
        }
        if constexpr (PHASE == SUMS) continue;
      }
      if (PHASE == APPLY || a.parts > 1) {
        if (PHASE == BOTH) __syncthreads();  // the slots are written
        mine = Pair{0.f, 0.f};
        if (member)
          for (int b = k; b < a.parts * a.subs; b += team) {
            const float* s = slot(b / a.subs, b % a.subs);
            mine = join(mine, Pair{s[0], s[1]});
          }
        mine = team_join(mine, pairs, first, k, team, member);
      }
      const float s1 = mine.a / count, s2 = mine.b / count;
      if (on)
        for (int l = l0 + rr; l < l1; l += AHEAD * a.rows) {
          Vec<In, V> x[AHEAD], g[AHEAD], d[AHEAD];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i)
            if (l + i * a.rows < l1) {
              const long p = at + (long)(l + i * a.rows) * a.C;
              x[i].load(a.x, p);
              d[i].load(a.dy, p);
              if (a.gate) g[i].load(a.gate, p);
            }
#pragma unroll
          for (int i = 0; i < AHEAD; ++i)
            if (l + i * a.rows < l1) {
              const long p = at + (long)(l + i * a.rows) * a.C;
              float n[V], z[V], u[V], y[V], slope[V], dx[V], dg[V];
#pragma unroll
              for (int e = 0; e < V; ++e) {
                n[e] = (x[i].get(e) - mean) * inv;
                z[e] = fmaf(n[e], w[e], bias[e]);
                u[e] = a.gate ? g[i].get(e) : z[e];
              }
              activate<V>(u, a.act, y, slope);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float dy = d[i].get(e), dz = dy * (a.gate ? y[e] : slope[e]);
                dg[e] = dy * z[e] * slope[e];
                dx[e] = inv * (dz * w[e] - s1 - n[e] * s2);
              }
              if (a.dx) Vec<In, V>::store(a.dx, p, dx);
              if (a.dgate) Vec<In, V>::store(a.dgate, p, dg);
            }
        }
    }
  }
  if constexpr (BWD && PHASE != APPLY) {
    if (!a.part) return;
    // The block's column sums: the rows of one vector in order.
#pragma unroll
    for (int e = 0; e < V; ++e) {
      __syncthreads();
      pairs[tid] = Pair{dw[e], db[e]};
      __syncthreads();
      if (on && rr == 0) {
        Pair s = pairs[tid];
        for (int i = 1; i < a.rows; ++i) s = join(s, pairs[tid + i * vecs]);
        float* p = a.part + ((long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.C + column + e;
        p[0] = s.a;
        p[a.C] = s.b;
      }
    }
  }
}

#define GN_ROWS(In, V, IT)                                         \
  template __global__ void norm_rows_kernel<In, V, IT, false>(Norm); \
  template __global__ void norm_rows_kernel<In, V, IT, true>(Norm);
#define GN_POSITIONS(In, V)                                              \
  template __global__ void norm_positions_kernel<In, V, false, SUMS>(Norm);  \
  template __global__ void norm_positions_kernel<In, V, false, APPLY>(Norm); \
  template __global__ void norm_positions_kernel<In, V, false, BOTH>(Norm);  \
  template __global__ void norm_positions_kernel<In, V, true, SUMS>(Norm);   \
  template __global__ void norm_positions_kernel<In, V, true, APPLY>(Norm);  \
  template __global__ void norm_positions_kernel<In, V, true, BOTH>(Norm);
#define GN_ALL(In, V) GN_ROWS(In, V, 1) GN_ROWS(In, V, 2) GN_ROWS(In, V, 4) GN_POSITIONS(In, V)
GN_ALL(float, 1)
GN_ALL(float, 2)
GN_ALL(float, 4)
GN_ALL(bf16_t, 1)
GN_ALL(bf16_t, 2)
GN_ALL(bf16_t, 4)
GN_ROWS(bf16_t, 8, 1)
GN_ROWS(bf16_t, 8, 2)
GN_POSITIONS(bf16_t, 8)

}  // namespace gn

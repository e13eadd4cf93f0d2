// The selective scan for gfx950: every channel d has N states with a decay each,
//   s = softplus(delta + bias) (or without),  h[n] <- exp(s a[d,n]) h[n] + s b[n] x,
//   y = sum over n of c[n] h[n] + skip x,     out = y silu(gate).
// Gradient, with dy = dout silu(gate) and g the cotangent of h after a token:
//   g <- g + c dy,  dc[n] = sum over d of dy h,  db[n] = sum over d of g s x,
//   flow = sum over n of g b,  rate[n] = g exp(s a) h_before,  g <- g exp(s a),
//   dx = s flow + skip dy,  ds = x flow + sum over n of rate a,  da = sum of rate s.
// The decays differ by channel and state, so that no product of matrices takes the
// place of the recurrence: it is walked, a few instructions a state and token, and
// the exponential (8.6 cycles a wave against 2.5 of a multiply-add with operands in
// vector registers) is most of them.
//
// A wave holds 16 channels: lane 16 q + ch has the states 4 q .. 4 q + 3 of channel ch
// (and of each further 16 states).  Tokens come in tiles of 16: lane k of row q holds
// b and c of token k for the row's states, and a multiply-add reads them by the row
// broadcast of its operand; what belongs to a channel (the step, s x, dy) goes through
// the wave's own LDS.  Sums over the states join the four rows of a wave once every
// four tokens.
#include <hip/hip_runtime.h>

#include "selscan.hpp"

namespace ss {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

// ------------------------------------------------------------ small functions

__device__ __forceinline__ unsigned pack(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}

// Four consecutive elements as they are in memory.
template <typename In>
struct Four;
template <>
struct Four<float> {
  f4 r;
  __device__ __forceinline__ float get(int i) const { return r[i]; }
  __device__ __forceinline__ void set(const float (&v)[4]) { r = f4{v[0], v[1], v[2], v[3]}; }
};
template <>
struct Four<bf16_t> {
  u2 r;
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[4]) {
    r = u2{pack(v[0], v[1]), pack(v[2], v[3])};
  }
};

// `count` (0..4) elements at p, zeros for the rest; whole: a piece is all or nothing
// and aligned.
template <typename In>
__device__ __forceinline__ Four<In> load4(const In* p, int count, bool whole) {
  Four<In> v;
  v.r = 0;
  if (whole) {
    if (count > 0) v = *reinterpret_cast<const Four<In>*>(p);
    return v;
  }
  if constexpr (sizeof(In) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) v.r[i] = p[i];
  } else {
    unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) w[i] = p[i];
    v.r = u2{w[0] | w[1] << 16, w[2] | w[3] << 16};
  }
  return v;
}

template <typename In>
__device__ __forceinline__ void store4(In* p, const float (&v)[4], int count, bool whole) {
  Four<In> f;
  f.set(v);
  if (whole) {
    if (count > 0) *reinterpret_cast<Four<In>*>(p) = f;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) {
      if constexpr (sizeof(In) == 4) p[i] = f.r[i];
      else p[i] = (bf16_t)(f.r[i >> 1] >> (16 * (i & 1)));
    }
}

// exp(-|v|), to float32's own precision: the product's rounding is put back.
__device__ __forceinline__ float exp_minus(float v) {
  const float a = -fabsf(v), p = a * LOG2E;
  const float low = fmaf(a, LOG2E, -p) + a * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(p);
  // (Far below the range the low part is no number any more.)
  return p < -200.f ? 0.f : fmaf(e, low * LN2, e);
}

// log(1 + exp(v)): u = 1 + e is rounded, and log(u) e / (u - 1) takes the rounding back
// (Kahan's form of log1p).
__device__ __forceinline__ float softplus(float v) {
  const float e = exp_minus(v), u = 1.f + e, d = u - 1.f;
  const float l = __builtin_amdgcn_logf(u) * LN2 * (e * __builtin_amdgcn_rcpf(d));
  return fmaxf(v, 0.f) + (d == 0.f ? e : l);
}

// 1 / (1 + exp(-v)), small values to their own precision.
__device__ __forceinline__ float sigmoid(float v) {
  const float e = exp_minus(v), r = __builtin_amdgcn_rcpf(1.f + e);
  return v < 0.f ? e * r : r;
}

// Lane K's value of each row of 16 lanes.
template <int K>
__device__ __forceinline__ float lane_of_row(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + K, 0xf, 0xf, true));
}

template <int CTRL, int BANKS = 0xf>
__device__ __forceinline__ float dpp(float old, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL,
                                                    0xf, BANKS, BANKS == 0xf));
}

// Sums over the four rows of a wave: row q has that of v[q].
__device__ __forceinline__ float join_rows(const float (&v)[4]) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0]), __float_as_uint(v[2]),
                                                  false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[1]), __float_as_uint(v[3]),
                                                  false, false);
  const float s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const float t = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  const auto c = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(t), false,
                                                  false);
  return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// x in banks KEEP (of four lanes each) of a row, y in the others.
template <int KEEP>
__device__ __forceinline__ float banks(float x, float y) {
  return dpp<0xE4, KEEP>(y, x);
}

// Sums over the 16 lanes of a row: bank b has that of v[b with its two bits swapped].
__device__ __forceinline__ float join_lanes(const float (&v)[4]) {
  const float s = banks<0x3>(v[0], v[1]) + dpp<0x128>(0.f, banks<0x3>(v[1], v[0]));
  const float t = banks<0x3>(v[2], v[3]) + dpp<0x128>(0.f, banks<0x3>(v[3], v[2]));
  float u = banks<0x5>(s, t) + dpp<0x141>(0.f, banks<0x5>(t, s));
  u += dpp<0xB1>(0.f, u);
  u += dpp<0x4E>(0.f, u);
  return u;
}

// Orders a wave's own LDS accesses (which the hardware keeps in order).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int K>
struct Index {
  static constexpr int value = K;
};
template <int K, int END, typename F>
__device__ __forceinline__ void unroll(F&& f) {
  if constexpr (K < END) {
    f(Index<K>{});
    unroll<K + 1, END>(f);
  }
}

// ------------------------------------------------------------ where a wave works

// As the recurrence runs: lane 16 q + ch.  As rows are read and written: lane
// 4 token + piece, of four channels.
struct Place {
  int lane, wave, q, ch, token, piece;
  int b, g, block, first;  // batch row, group, channel block, the wave's first channel of it
  int s, begin, end, len;  // segment, its tokens, the row's present tokens
  long row;                // batch row and segment
  int d;                   // the lane's channel, of all D
  bool on;                 // whether there is one
  int d4, count;           // the piece's first channel, and how many there are
};

__device__ __forceinline__ Place place(const Scan& a) {
  Place p;
  p.lane = threadIdx.x & 63;
  p.wave = threadIdx.x >> 6;
  p.q = p.lane >> 4;
  p.ch = p.lane & 15;
  p.token = p.lane >> 2;
  p.piece = (p.lane & 3) * 4;
  const int rest = blockIdx.x / a.blocks;
  p.block = blockIdx.x - rest * a.blocks;
  p.b = rest / a.G;
  p.g = rest - p.b * a.G;
  p.first = p.block * BLOCK_CHANNELS + p.wave * 16;
  p.s = blockIdx.y;
  p.begin = p.s * a.seg;
  p.end = min(a.T, p.begin + a.seg);
  p.len = a.lengths ? min(max(a.lengths[p.b], 0), a.T) : a.T;
  p.row = (long)p.b * a.NS + p.s;
  p.on = p.first + p.ch < a.Dg;
  p.d = p.g * a.Dg + p.first + p.ch;
  p.count = min(4, max(0, a.Dg - p.first - p.piece));
  p.d4 = p.g * a.Dg + p.first + p.piece;
  return p;
}

// A tile's rows as they are in memory.
template <typename In, int NG, bool GATE, bool DOUT>
struct TileRows {
  Four<In> x, delta, gate, dout, b[NG], c[NG];

  __device__ __forceinline__ void fetch(const Scan& a, const Place& p, int t0) {
    const int last = min(p.end, p.len);
    const int t = t0 + p.token;
    const int count = t < last ? p.count : 0;
    const auto row = [&](const Rows& r) {
      return load4(static_cast<const In*>(r.p) + p.b * r.batch + t * r.token + p.d4, count,
                   a.whole);
    };
    x = row(a.x);
    delta = row(a.delta);
    if (GATE) {
      if (a.gate.p) gate = row(a.gate);
      else gate.r = 0;
    }
    if (DOUT)
      dout = load4(static_cast<const In*>(a.dout) + ((long)p.b * a.T + t) * a.D + p.d4, count,
                   a.whole);
    const int k = t0 + p.ch;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int n = 16 * i + 4 * p.q;
      const int have = k < last ? min(4, max(0, a.N - n)) : 0;
      b[i] = load4(static_cast<const In*>(a.b.p) + p.b * a.b.batch + k * a.b.token +
                       p.g * a.bg + n, have, a.whole_bc);
      c[i] = load4(static_cast<const In*>(a.c.p) + p.b * a.c.batch + k * a.c.token +
                       p.g * a.cg + n, have, a.whole_bc);
    }
  }
};

template <int NG>
__device__ __forceinline__ void load_decays(const Scan& a, const Place& p, float (&rate)[NG][4]) {
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = 16 * i + 4 * p.q + r;
      float v = 0.f;
      if (p.on && n < a.N) {
        v = a.a[(long)p.d * a.N + n] * LOG2E;
        // (An infinite rate times the zero step of an absent token is no number.)
        v = v < -3.4e38f ? -3.4e38f : v > 3.4e38f ? 3.4e38f : v;
      }
      rate[i][r] = v;
    }
}

// States of one channel at `from` (or zeros).
template <int NG>
__device__ __forceinline__ void load_states(const Scan& a, const Place& p, const float* from,
                                            float (&h)[NG][4]) {
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int n = 16 * i + 4 * p.q;
    Four<float> v;
    v.r = 0;
    if (from && p.on) v = load4(from + n, min(4, max(0, a.N - n)), a.whole_n);
#pragma unroll
    for (int r = 0; r < 4; ++r) h[i][r] = v.get(r);
  }
}

template <int NG>
__device__ __forceinline__ void store_states(const Scan& a, const Place& p, float* to,
                                             const float (&h)[NG][4]) {
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int n = 16 * i + 4 * p.q;
    if (p.on) store4(to + n, h[i], min(4, max(0, a.N - n)), a.whole_n);
  }
}

// The steps of a lane's piece.
template <typename In>
__device__ __forceinline__ void steps(const Scan& a, const Four<In>& delta, const float (&bias)[4],
                                      bool here, float (&s)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float v = delta.get(e) + bias[e];
    s[e] = here ? (a.softplus ? softplus(v) : v) : 0.f;
  }
}

__device__ __forceinline__ void load_bias(const float* from, const Place& p, float (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from && e < p.count ? from[p.d4 + e] : 0.f;
}

// The sums over the tokens (lanes 4 apart) of a piece's four values, to [D].
__device__ __forceinline__ void store_token_sums(const Place& p, float (&v)[4], float* to) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = v[e];
    for (int m = 4; m < 64; m *= 2) x += __shfl_xor(x, m);
    if (p.token == 0 && e < p.count) to[p.d4 + e] = x;
  }
}

// ------------------------------------------------------------ forward

// OUT: a segment's outputs from its start state (and the last one's end state); else
// what the segment adds to the state, and the sum of its steps.
template <typename In, int NG, bool OUT>
__global__ __launch_bounds__(64 * WAVES) void scan_kernel(Scan a) {
  __shared__ f4 shared[WAVES][OUT ? 192 : 128];
  const Place p = place(a);
  if (p.first >= a.Dg) return;
  f2* su = reinterpret_cast<f2*>(shared[p.wave]);               // [16 tokens][16 channels]
  float* yl = reinterpret_cast<float*>(shared[p.wave] + 128);   // the same
  float rate[NG][4], h[NG][4], bias[4], skip[4], total[4] = {0.f, 0.f, 0.f, 0.f};
  load_decays(a, p, rate);
  load_bias(a.bias, p, bias);
  load_bias(a.skip, p, skip);
  const float* from = nullptr;
  if (OUT)
    from = a.NS > 1 ? a.ends + (p.row * a.D + p.d) * a.N
           : a.initial ? a.initial + ((long)p.b * a.D + p.d) * a.N : nullptr;
  load_states(a, p, from, h);
  const int tiles = (a.T + TILE - 1) / TILE;
  TileRows<In, NG, OUT, false> next;
  next.fetch(a, p, p.begin);
  for (int t0 = p.begin; t0 < p.end; t0 += TILE) {
    const bool here = t0 + p.token < min(p.end, p.len);
    const long at = ((long)p.b * a.T + t0 + p.token) * a.D + p.d4;
    if (t0 >= p.len) {
      if (!OUT) break;
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      if (t0 + p.token < p.end) store4(static_cast<In*>(a.out) + at, zero, p.count, a.whole);
      continue;
    }
    const TileRows<In, NG, OUT, false> now = next;
    next.fetch(a, p, t0 + TILE);
    if (OUT && a.kept)
      store_states(a, p, a.kept + (((long)p.b * tiles + t0 / TILE) * a.D + p.d) * a.N, h);
    float s[4];
    steps(a, now.delta, bias, here, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      su[p.token * 16 + p.piece + e] = f2{s[e], s[e] * now.x.get(e)};
      if (!OUT) total[e] += s[e];
    }
    wave_sync();
    float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      float bv[4], cv[4], part[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bv[r] = now.b[i].get(r);
        cv[r] = now.c[i].get(r);
      }
      unroll<0, TILE>([&](auto k) {
        constexpr int t = k.value;
        const f2 v = su[t * 16 + p.ch];
        if (OUT) part[t & 3] = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float keep = __builtin_amdgcn_exp2f(v.x * rate[i][r]);
          h[i][r] = fmaf(keep, h[i][r], v.y * lane_of_row<t>(bv[r]));
          if (OUT) part[t & 3] = fmaf(lane_of_row<t>(cv[r]), h[i][r], part[t & 3]);
        }
        if (OUT && (t & 3) == 3) y[t / 4] += join_rows(part);
      });
    }
    if (OUT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) yl[(4 * j + p.q) * 16 + p.ch] = y[j];
      wave_sync();
      const f4 v = *reinterpret_cast<const f4*>(yl + p.token * 16 + p.piece);
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(skip[e], now.x.get(e), v[e]);
        if (a.gate.p) {
          const float z = now.gate.get(e);
          o[e] *= z * sigmoid(z);
        }
        o[e] = here ? o[e] : 0.f;
      }
      if (t0 + p.token < p.end) store4(static_cast<In*>(a.out) + at, o, p.count, a.whole);
      wave_sync();
    }
  }
  if (!OUT) {
    store_states(a, p, a.ends + (p.row * a.D + p.d) * a.N, h);
    store_token_sums(p, total, a.sums + p.row * a.D);
  } else if (p.s == a.NS - 1) {
    store_states(a, p, a.state + ((long)p.b * a.D + p.d) * a.N, h);
  }
}

// What each segment starts from, in the place of what it adds: h <- exp(a sum s) h + end.
// Backward: from the last to the first, from the state's cotangent, to d_initial.
template <bool BWD>
__global__ __launch_bounds__(256) void carry_kernel(Scan a) {
  const long each = (long)a.D * a.N, count = a.B * each;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    const long b = i / each, rest = i - b * each;
    const long d = rest / a.N;
    float v = a.a[rest] * LOG2E;
    v = v < -3.4e38f ? -3.4e38f : v > 3.4e38f ? 3.4e38f : v;
    const float* from = BWD ? a.dstate : a.initial;
    float h = from ? from[i] : 0.f;
    for (int j = 0; j < a.NS; ++j) {
      const long row = b * a.NS + (BWD ? a.NS - 1 - j : j);
      const float end = a.ends[row * each + rest];
      a.ends[row * each + rest] = h;
      h = fmaf(__builtin_amdgcn_exp2f(a.sums[row * a.D + d] * v), h, end);
    }
    if (BWD && a.dinitial) a.dinitial[i] = h;
  }
}

// ------------------------------------------------------------ backward

// ALL: a segment's gradients from the cotangent of the state after it; else what the
// segment adds to the cotangent of the state before it, and the sum of its steps.
template <typename In, int NG, bool ALL>
__global__ __launch_bounds__(64 * WAVES) void scan_backward_kernel(Scan a) {
  // A wave's steps, inflows and cotangents [16 tokens][16 channels], then sums over the
  // states of the same shape; and every wave's sums over channels [16 tokens][16 states].
  __shared__ f4 shared[WAVES][ALL ? 256 : 128];
  __shared__ f4 sums[ALL ? 2 : 1][WAVES][ALL ? 128 : 1];
  const Place p = place(a);
  const bool idle = p.first >= a.Dg;
  if (!ALL && idle) return;
  const int active = min(WAVES, (a.Dg - p.block * BLOCK_CHANNELS + 15) / 16);
  f4* sud = shared[p.wave];
  float* joined = reinterpret_cast<float*>(shared[p.wave]);
  float rate[NG][4], g[NG][4], da[NG][4], bias[4], skip[4];
  float dskip[4] = {0.f, 0.f, 0.f, 0.f}, dbias[4] = {0.f, 0.f, 0.f, 0.f};
  load_decays(a, p, rate);
  load_bias(a.bias, p, bias);
  load_bias(a.skip, p, skip);
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) da[i][r] = 0.f;
  const float* from = nullptr;
  if (ALL)
    from = a.NS > 1 ? a.ends + (p.row * a.D + p.d) * a.N
           : a.dstate ? a.dstate + ((long)p.b * a.D + p.d) * a.N : nullptr;
  load_states(a, p, from, g);
  const int tiles = (a.T + TILE - 1) / TILE;
  const int first = p.begin / TILE, last = (p.end + TILE - 1) / TILE;
  // The tile to begin with: the last one with a token that is present.
  int tile = last - 1;
  for (; tile >= first && tile * TILE >= p.len; --tile) {
    const int t = tile * TILE + p.token;
    if (ALL && !idle && t < p.end) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      const long at = ((long)p.b * a.T + t) * a.D + p.d4;
      store4(static_cast<In*>(a.dx) + at, zero, p.count, a.whole);
      store4(static_cast<In*>(a.ddelta) + at, zero, p.count, a.whole);
      if (a.dgate) store4(static_cast<In*>(a.dgate) + at, zero, p.count, a.whole);
    }
  }
  TileRows<In, NG, true, true> next;
  if (tile >= first) next.fetch(a, p, tile * TILE);
  int turn = 0;
  for (; tile >= first; --tile) {
    const int t0 = tile * TILE;
    const bool here = t0 + p.token < min(p.end, p.len);
    const TileRows<In, NG, true, true> now = next;
    if (tile > first) next.fetch(a, p, t0 - TILE);
    float s[4], dy[4];
    steps(a, now.delta, bias, here, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float z = now.gate.get(e);
      dy[e] = now.dout.get(e) * (a.gate.p ? z * sigmoid(z) : 1.f);
      const f4 v = {s[e], s[e] * now.x.get(e), dy[e], 0.f};
      if (ALL) {
        sud[p.token * 16 + p.piece + e] = v;
      } else {
        reinterpret_cast<f2*>(sud)[p.token * 16 + p.piece + e] = f2{s[e], dy[e]};
        dbias[e] += s[e];
      }
    }
    wave_sync();
    if constexpr (!ALL) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float cv[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) cv[r] = now.c[i].get(r);
        unroll<0, TILE>([&](auto k) {
          constexpr int t = TILE - 1 - k.value;
          const f2 v = reinterpret_cast<f2*>(sud)[t * 16 + p.ch];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            g[i][r] = __builtin_amdgcn_exp2f(v.x * rate[i][r]) *
                      fmaf(lane_of_row<t>(cv[r]), v.y, g[i][r]);
        });
      }
      wave_sync();
    } else {
      float y[4] = {0.f, 0.f, 0.f, 0.f}, flow[4] = {0.f, 0.f, 0.f, 0.f},
            slope[4] = {0.f, 0.f, 0.f, 0.f};
      float start[NG][4];
      load_states(a, p, a.kept + (((long)p.b * tiles + tile) * a.D + p.d) * a.N, start);
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float* mine = reinterpret_cast<float*>(sums[turn][p.wave]);
        if (!idle) {
          float bv[4], cv[4], h[TILE][4], keep[TILE][4], part[4], part2[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            bv[r] = now.b[i].get(r);
            cv[r] = now.c[i].get(r);
          }
          unroll<0, TILE>([&](auto k) {
            constexpr int t = k.value;
            const f4 v = sud[t * 16 + p.ch];
            part[t & 3] = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float before = t ? h[t ? t - 1 : 0][r] : start[i][r];
              keep[t][r] = __builtin_amdgcn_exp2f(v.x * rate[i][r]);
              h[t][r] = fmaf(keep[t][r], before, v.y * lane_of_row<t>(bv[r]));
              part[t & 3] = fmaf(lane_of_row<t>(cv[r]), h[t][r], part[t & 3]);
            }
            if ((t & 3) == 3) y[t / 4] += join_rows(part);
          });
          unroll<0, TILE>([&](auto k) {
            constexpr int t = TILE - 1 - k.value;
            const f4 v = sud[t * 16 + p.ch];
            float pb[4], pc[4];
            part[t & 3] = 0.f;
            part2[t & 3] = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float before = t ? h[t ? t - 1 : 0][r] : start[i][r];
              g[i][r] = fmaf(lane_of_row<t>(cv[r]), v.z, g[i][r]);
              pc[r] = h[t][r] * v.z;
              pb[r] = g[i][r] * v.y;
              part[t & 3] = fmaf(lane_of_row<t>(bv[r]), g[i][r], part[t & 3]);
              g[i][r] *= keep[t][r];
              const float m = g[i][r] * before;
              part2[t & 3] = fmaf(m, rate[i][r], part2[t & 3]);
              da[i][r] = fmaf(m, v.x, da[i][r]);
            }
            // Bank j of row q: state 4 q + (j with its bits swapped).
            const int n = 4 * p.q + ((p.ch >> 3) | (p.ch >> 1 & 2));
            mine[t * 16 + n] = join_lanes(pb);
            mine[256 + t * 16 + n] = join_lanes(pc);
            if ((t & 3) == 0) {
              flow[t / 4] += join_rows(part);
              slope[t / 4] += join_rows(part2);
            }
          });
        }
        __syncthreads();
        // The block's channels, in their order.
        const float* all = reinterpret_cast<const float*>(sums[turn]);
        const int t = threadIdx.x >> 4, n = 16 * i + (threadIdx.x & 15);
        float db = 0.f, dc = 0.f;
        for (int w = 0; w < active; ++w) {
          db += all[w * 512 + threadIdx.x];
          dc += all[w * 512 + 256 + threadIdx.x];
        }
        if (n < a.N && t0 + t < min(p.end, p.len)) {
          const long tokens = (long)a.B * a.T;
          float* to = a.part_bc +
                      ((p.block * tokens + (long)p.b * a.T + t0 + t) * a.G + p.g) * 2 * a.N + n;
          to[0] = db;
          to[a.N] = dc;
        }
        turn ^= 1;
      }
      if (!idle) {
        wave_sync();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = (4 * j + p.q) * 16 + p.ch;
          joined[at] = y[j];
          joined[256 + at] = flow[j];
          joined[512 + at] = slope[j];
        }
        wave_sync();
        const int from4 = p.token * 16 + p.piece;
        const f4 yv = *reinterpret_cast<const f4*>(joined + from4);
        const f4 fv = *reinterpret_cast<const f4*>(joined + 256 + from4);
        const f4 sv = *reinterpret_cast<const f4*>(joined + 512 + from4);
        wave_sync();
        float dx[4], dd[4], dz[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = now.x.get(e), z = now.gate.get(e), sg = sigmoid(z);
          const float whole = fmaf(skip[e], x, yv[e]);
          dz[e] = here ? now.dout.get(e) * whole * (sg * fmaf(z, 1.f - sg, 1.f)) : 0.f;
          dx[e] = here ? fmaf(s[e], fv[e], skip[e] * dy[e]) : 0.f;
          float v = fmaf(x, fv[e], sv[e] * LN2);
          if (a.softplus) v *= sigmoid(now.delta.get(e) + bias[e]);
          dd[e] = here ? v : 0.f;
          dskip[e] += here ? dy[e] * x : 0.f;
          dbias[e] += dd[e];
        }
        if (t0 + p.token < p.end) {
          const long at = ((long)p.b * a.T + t0 + p.token) * a.D + p.d4;
          store4(static_cast<In*>(a.dx) + at, dx, p.count, a.whole);
          store4(static_cast<In*>(a.ddelta) + at, dd, p.count, a.whole);
          if (a.dgate) store4(static_cast<In*>(a.dgate) + at, dz, p.count, a.whole);
        }
      }
    }
  }
  if (idle) return;
  if (!ALL) {
    store_states(a, p, a.ends + (p.row * a.D + p.d) * a.N, g);
    store_token_sums(p, dbias, a.sums + p.row * a.D);
    return;
  }
  if (a.part_a) store_states(a, p, a.part_a + (p.row * a.D + p.d) * a.N, da);
  store_token_sums(p, dskip, a.part_d + p.row * 2 * a.D);
  store_token_sums(p, dbias, a.part_d + (p.row * 2 + 1) * a.D);
  if (a.NS == 1 && a.dinitial)
    store_states(a, p, a.dinitial + ((long)p.b * a.D + p.d) * a.N, g);
}

// The gradients of b and c: the sums over the channel blocks.
template <typename In>
__global__ __launch_bounds__(256) void join_bc_kernel(Join a) {
  const long each = (long)a.G * a.N, tokens = (long)a.B * a.T, count = tokens * each;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    const long token = i / each, rest = i - token * each;
    const long g = rest / a.N, n = rest - g * a.N;
    const long b = token / a.T;
    const bool here = !a.lengths || token - b * a.T < a.lengths[b];
    const float* from = a.part_bc + (token * a.G + g) * 2 * a.N + n;
    float db = 0.f, dc = 0.f;
    if (here)
      for (int j = 0; j < a.blocks; ++j) {
        db += from[j * tokens * each * 2];
        dc += from[j * tokens * each * 2 + a.N];
      }
    if constexpr (sizeof(In) == 4) {
      static_cast<float*>(a.db)[i] = db;
      static_cast<float*>(a.dc)[i] = dc;
    } else {
      static_cast<bf16_t*>(a.db)[i] = (bf16_t)pack(db, 0.f);
      static_cast<bf16_t*>(a.dc)[i] = (bf16_t)pack(dc, 0.f);
    }
  }
}

// Sums over rows ([rows][stride], `count` of each from `part` on): of the batch rows and
// segments.
__global__ __launch_bounds__(256) void join_rows_kernel(const float* part, long rows, long stride,
                                                        long count, float scale, float* out) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    float s = 0.f;
    for (long j = 0; j < rows; ++j) s += part[j * stride + i];
    out[i] = s * scale;
  }
}

// ------------------------------------------------------------ one token

// Bound by memory: the states are read and written once.  2^span lanes hold a
// channel, four states each at a time.
template <typename In>
__global__ __launch_bounds__(STEP_THREADS) void step_kernel(Step a) {
  const long i = (long)blockIdx.x * STEP_THREADS + threadIdx.x;
  const long row = i >> a.span;
  const int part = (int)(i & ((1 << a.span) - 1));
  if (row >= a.B * a.D) return;
  const long b = row / a.D;
  const int d = (int)(row - b * a.D), g = d / a.Dg;
  const bool on = !a.active || a.active[b];
  const auto one = [](const void* p, long at) {
    const In v = static_cast<const In*>(p)[at];
    if constexpr (sizeof(In) == 4) return (float)v;
    else return __uint_as_float((unsigned)v << 16);
  };
  const float* from = a.state + row * a.N;
  float* to = a.new_state + row * a.N;
  float x = 0.f, s = 0.f, y = 0.f;
  if (on) {
    x = one(a.x.p, b * a.x.batch + d);
    s = one(a.delta.p, b * a.delta.batch + d) + (a.bias ? a.bias[d] : 0.f);
    if (a.softplus) s = softplus(s);
  }
  const float u = s * x;
  const bool whole = a.whole_n;
  for (int n = 4 * part; n < a.N; n += 4 << a.span) {
    const int have = min(4, a.N - n);
    const Four<float> h = load4(from + n, have, whole);
    const Four<float> rate = load4(a.a + (long)d * a.N + n, have, whole);
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] = h.get(r);
      if (on && r < have) {
        v[r] = fmaf(__builtin_amdgcn_exp2f(s * (rate.get(r) * LOG2E)), v[r],
                    u * one(a.b.p, b * a.b.batch + g * a.bg + n + r));
        y = fmaf(one(a.c.p, b * a.c.batch + g * a.cg + n + r), v[r], y);
      }
    }
    if (on || to != from) store4(to + n, v, have, whole);
  }
  for (int m = 1; m < 1 << a.span; m *= 2) y += __shfl_xor(y, m);
  if (part) return;
  if (on) {
    if (a.skip) y = fmaf(a.skip[d], x, y);
    if (a.gate.p) {
      const float z = one(a.gate.p, b * a.gate.batch + d);
      y *= z * sigmoid(z);
    }
  }
  if constexpr (sizeof(In) == 4) static_cast<float*>(a.out)[row] = y;
  else static_cast<bf16_t*>(a.out)[row] = (bf16_t)pack(y, 0.f);
}

#define M4SL_SCAN(In)                                               \
  template __global__ void scan_kernel<In, 1, true>(Scan);          \
  template __global__ void scan_kernel<In, 2, true>(Scan);          \
  template __global__ void scan_kernel<In, 4, true>(Scan);          \
  template __global__ void scan_kernel<In, 1, false>(Scan);         \
  template __global__ void scan_kernel<In, 2, false>(Scan);         \
  template __global__ void scan_kernel<In, 4, false>(Scan);         \
  template __global__ void scan_backward_kernel<In, 1, true>(Scan); \
  template __global__ void scan_backward_kernel<In, 2, true>(Scan); \
  template __global__ void scan_backward_kernel<In, 4, true>(Scan); \
  template __global__ void scan_backward_kernel<In, 1, false>(Scan);\
  template __global__ void scan_backward_kernel<In, 2, false>(Scan);\
  template __global__ void scan_backward_kernel<In, 4, false>(Scan);\
  template __global__ void join_bc_kernel<In>(Join);                \
  template __global__ void step_kernel<In>(Step);
M4SL_SCAN(float)
M4SL_SCAN(bf16_t)
template __global__ void carry_kernel<false>(Scan);
template __global__ void carry_kernel<true>(Scan);

}  // namespace ss

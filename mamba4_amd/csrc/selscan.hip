// The selective scan for gfx950: every channel d has N states with a decay each,
//   s = softplus(delta + bias) (or without),  h[n] <- exp(s a[d,n]) h[n] + s b[n] x,
//   y = sum over n of c[n] h[n] + skip x,     out = y silu(gate).
// Gradient, with dy = dout silu(gate) and g the cotangent of h after a token:
//   g <- g + c dy,  dc[n] = sum over d of dy h,  db[n] = sum over d of g s x,
//   flow = sum over n of g b,  rate[n] = g exp(s a) h_before,  g <- g exp(s a),
//   dx = s flow + skip dy,  ds = x flow + sum over n of rate a,  da = sum of rate s.
// The decays differ by channel and state, so that no product of matrices takes the
// place of the recurrence: it is walked, and vector instructions bound it: five a state
// and token forwards (one of them the exponential, which takes a SIMD 8 cycles for 4 of the
// others), fourteen in the gradient, which walks forwards first.
//
// A wave holds 16 channels: lane 16 q + ch has the states 4 q .. 4 q + 3 of channel ch
// (and of each further 16 states).  Tokens come in tiles of 16: lane k of row q holds
// b and c of token k for the row's states, and a multiply-add reads them by the row
// broadcast of its operand; what belongs to a channel (the step, s x, dy) goes through
// the wave's own LDS, and so do the sums over the states: each row of lanes writes its own,
// four numbers a token and channel, and the lane that forms the result adds them (joined in
// registers by exchanges of rows they took 322 us in place of 301: T32768 D2048 N16,
// outputs).  Measured and left: b and c by token from LDS (335 us for 335), their
// products with x and h as outer products on the matrix units (427 for 355; of b x alone,
// no change).
#include <hip/hip_runtime.h>

#include "selscan.hpp"

namespace ss {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
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

// v where `mask` is all ones, zero where it is zero.  (A select costs 4.6 cycles a wave,
// and 23 where its condition is in VCC and was not just formed; this costs 3.)
__device__ __forceinline__ float masked(float v, unsigned mask) {
  return __uint_as_float(__float_as_uint(v) & mask);
}

// Rows through a buffer's descriptor: reads past its bytes are zero and writes dropped, so
// that absent tokens, and lanes without a channel (whose offset is ABSENT or more), need
// no branch and no clearing.
typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr unsigned ABSENT = 0x80000000u;

__device__ __forceinline__ Rsrc rsrc(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}
__device__ __forceinline__ void read4(Rsrc r, unsigned at, Four<float>& v) {
  v.r = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}
__device__ __forceinline__ void read4(Rsrc r, unsigned at, Four<bf16_t>& v) {
  v.r = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
}
__device__ __forceinline__ void write4(Rsrc r, unsigned at, const Four<float>& v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v.r), r, at, 0, 0);
}
__device__ __forceinline__ void write4(Rsrc r, unsigned at, const Four<bf16_t>& v) {
  __builtin_amdgcn_raw_buffer_store_b64(v.r, r, at, 0, 0);
}

// log(1 + exp(v)): of u = 1 + e, rounded, and of what the rounding lost, l = e - (u - 1).
// (That is l / u to first order; l itself is off by at most l e / u <= 2^-24 e / u, less than
// 2^-24 of log(1 + e) >= e / u, and spares a reciprocal of 8 cycles.)
__device__ __forceinline__ float softplus(float v) {
  const float e = __builtin_amdgcn_exp2f(-LOG2E * fabsf(v)), u = 1.f + e;
  return fmaxf(v, 0.f) + fmaf(__builtin_amdgcn_logf(u), LN2, e - (u - 1.f));
}

// 1 / (1 + exp(-v)), to 2^-24 of itself and of v.
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * v));
}

// acc + K's lane of src in each row of 16 lanes, times mul, as one instruction (the
// compiler takes two).  `settled` has to come between what writes src and this.
template <int K>
__device__ __forceinline__ void fmac_row(float& acc, float src, float mul) {
  asm("v_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf"
      : "+v"(acc)
      : "v"(src), "v"(mul), "n"(K));
}
template <int K>
__device__ __forceinline__ float mul_row(float src, float mul) {
  float r;
  asm("v_mul_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf"
      : "=v"(r)
      : "v"(src), "v"(mul), "n"(K));
  return r;
}

// The same as the first of a sum.
template <int K>
__device__ __forceinline__ void add_row(float& acc, float src, float mul, bool first) {
  if (first) acc = mul_row<K>(src, mul);
  else fmac_row<K>(acc, src, mul);
}

// The two wait states between an instruction that writes a register and one that reads it
// from other lanes, which the compiler does not see to inside inline assembly.  (The
// build checks the compiled code for them.)
__device__ __forceinline__ void settled(float (&v)[4], float (&w)[4]) {
  asm volatile("s_nop 1"
               : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(w[0]), "+v"(w[1]),
                 "+v"(w[2]), "+v"(w[3]));
}

// Sums of v and of w over the 16 lanes of a row: bank b (of four lanes) has that of v[b
// with its two bits swapped].  Each level adds the lanes 8, then 4 apart of one value in
// half of the banks and of another in the rest, so that four values take eight
// instructions; those of v and w alternate to keep two wait states between an
// instruction and the next that reads its result from other lanes.
__device__ __forceinline__ void join_lanes(const float (&v)[4], const float (&w)[4], float& sv,
                                           float& sw) {
  float a, b, c, d;
  asm("s_nop 1\n"
      "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0x3\n"
      "v_add_f32_dpp %2, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %3, %8, %8 row_ror:8 row_mask:0xf bank_mask:0x3\n"
      "v_add_f32_dpp %3, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %4, %10, %10 row_ror:8 row_mask:0xf bank_mask:0x3\n"
      "v_add_f32_dpp %4, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %5, %12, %12 row_ror:8 row_mask:0xf bank_mask:0x3\n"
      "v_add_f32_dpp %5, %13, %13 row_ror:8 row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0x5\n"
      "v_add_f32_dpp %0, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xa\n"
      "v_add_f32_dpp %1, %4, %4 row_half_mirror row_mask:0xf bank_mask:0x5\n"
      "v_add_f32_dpp %1, %5, %5 row_half_mirror row_mask:0xf bank_mask:0xa\n"
      "v_add_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "s_nop 0\n"
      "v_add_f32_dpp %1, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
      "s_nop 0\n"
      "v_add_f32_dpp %1, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf"
      : "=&v"(sv), "=&v"(sw), "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
      : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(w[0]), "v"(w[1]), "v"(w[2]), "v"(w[3]));
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
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.q = p.lane >> 4;
  p.ch = p.lane & 15;
  p.token = p.lane >> 2;
  p.piece = (p.lane & 3) * 4;
  const int rest = blockIdx.x / a.blocks;
  p.block = blockIdx.x - rest * a.blocks;
  p.b = rest / a.G;
  p.g = rest - p.b * a.G;
  p.first = p.block * BLOCK_CHANNELS + p.wave * 16;
  p.s = blockIdx.y + a.skipped;
  p.begin = p.s * a.seg;
  p.end = p.begin + min(a.T - p.begin, a.seg);
  p.len = a.lengths ? min(max(a.lengths[p.b], 0), a.T) : a.T;
  p.row = (long)p.b * a.NS + p.s;
  p.on = p.first + p.ch < a.Dg;
  p.d = p.g * a.Dg + p.first + p.ch;
  p.count = min(4, max(0, a.Dg - p.first - p.piece));
  p.d4 = p.g * a.Dg + p.first + p.piece;
  return p;
}

// An array's rows of a wave's channels (or of its group's states), from the segment's first
// token up to some last one: their bytes, that of a token, and where in a tile the lane
// reads.  (WHOLE: a segment and two tiles more are below 2^31 bytes.)
struct Lines {
  const char* base;
  int bytes, stride;
  unsigned at;
  __device__ __forceinline__ Rsrc rows() const { return rsrc(base, bytes); }
  __device__ __forceinline__ unsigned tile(int t) const { return at + (unsigned)(t * stride); }
};

// `last` - p.begin rows (or fewer than one: none) of a.D channels.
template <typename In>
__device__ __forceinline__ Lines channel_lines(const Scan& a, const Place& p, const void* data,
                                               long batch, long token, int last) {
  const In* base = static_cast<const In*>(data) + batch + p.begin * token + (p.d - p.ch);
  const int stride = (int)token * (int)sizeof(In), rows = last - p.begin,
            width = min(16, max(0, a.Dg - p.first)) * (int)sizeof(In);
  return Lines{reinterpret_cast<const char*>(base), rows > 0 ? (rows - 1) * stride + width : 0,
               stride,
               p.count > 0 ? (unsigned)(p.token * stride + p.piece * (int)sizeof(In)) : ABSENT};
}

// The arrays that a kernel reads by tiles.
template <typename In, int NG>
struct Sources {
  Lines x, delta, gate, dout, b, c;

  __device__ __forceinline__ Sources(const Scan& a, const Place& p, int last) {
    const auto lines = [&](const Rows& r) {
      return channel_lines<In>(a, p, r.p, p.b * r.batch, r.token, last);
    };
    x = lines(a.x);
    delta = lines(a.delta);
    gate = lines(a.gate);
    dout = channel_lines<In>(a, p, a.dout, (long)p.b * a.T * a.D, a.D, last);
    const auto states = [&](const Rows& r, long group) {
      const In* base =
          static_cast<const In*>(r.p) + p.b * r.batch + p.begin * r.token + p.g * group;
      const int stride = (int)r.token * (int)sizeof(In), rows = last - p.begin;
      return Lines{reinterpret_cast<const char*>(base),
                   rows > 0 ? (rows - 1) * stride + a.N * (int)sizeof(In) : 0, stride,
                   (unsigned)(p.ch * stride + 4 * p.q * (int)sizeof(In))};
    };
    b = states(a.b, a.bg);
    c = states(a.c, a.cg);
  }
};

// A tile's rows as they are in memory; absent tokens and channels are zero.  WHOLE: all
// rows consist of aligned pieces of four.
template <typename In, int NG, bool GATE, bool DOUT, bool WHOLE>
struct TileRows {
  Four<In> x, delta, gate, dout, b[NG], c[NG];

  // Tokens t0 .. t0 + 15 of those before `last`.
  __device__ __forceinline__ void fetch(const Scan& a, const Place& p, const Sources<In, NG>& from,
                                        int t0, int last) {
    if constexpr (WHOLE) {
      const int rel = t0 - p.begin;
      const auto read = [&](const Lines& l, Four<In>& v) { read4(l.rows(), l.tile(rel), v); };
      read(from.x, x);
      read(from.delta, delta);
      if (GATE) read(from.gate, gate);
      if (DOUT) read(from.dout, dout);
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const unsigned n = 16 * i + 4 * p.q, more = 16 * i * sizeof(In);
        const bool on = n < (unsigned)a.N;
        read4(from.b.rows(), on ? from.b.tile(rel) + more : ABSENT, b[i]);
        read4(from.c.rows(), on ? from.c.tile(rel) + more : ABSENT, c[i]);
      }
    } else {
      const int t = t0 + p.token, count = t < last ? p.count : 0;
      const auto row = [&](const Rows& r) {
        return load4(static_cast<const In*>(r.p) + p.b * r.batch + t * r.token + p.d4, count,
                     false);
      };
      x = row(a.x);
      delta = row(a.delta);
      if (GATE) gate = row(a.gate);
      if (DOUT)
        dout = load4(static_cast<const In*>(a.dout) + ((long)p.b * a.T + t) * a.D + p.d4, count,
                     false);
      const int k = t0 + p.ch;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int n = 16 * i + 4 * p.q, have = k < last ? min(4, max(0, a.N - n)) : 0;
        b[i] = load4(static_cast<const In*>(a.b.p) + p.b * a.b.batch + k * a.b.token + p.g * a.bg +
                         n, have, false);
        c[i] = load4(static_cast<const In*>(a.c.p) + p.b * a.c.batch + k * a.c.token + p.g * a.cg +
                         n, have, false);
      }
    }
  }
};

// Rows [B,T,D] that a kernel writes by tiles, of the wave's channels, up to the segment's
// end.
template <typename In, bool WHOLE>
struct Result {
  Lines l;
  In* to;
  __device__ __forceinline__ Result(const Scan& a, const Place& p, void* data) {
    l = channel_lines<In>(a, p, data, (long)p.b * a.T * a.D, a.D, p.end);
    to = static_cast<In*>(data) + (long)p.b * a.T * a.D + p.d4;
  }
  __device__ __forceinline__ void put(const Scan& a, const Place& p, int t0,
                                      const float (&v)[4]) const {
    if constexpr (WHOLE) {
      Four<In> f;
      f.set(v);
      write4(l.rows(), l.tile(t0 - p.begin), f);
    } else if (t0 + p.token < p.end) {
      store4(to + (long)(t0 + p.token) * a.D, v, p.count, false);
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

// The state that a segment of the forward starts from: the carry's steps over those before
// it, in its order, where there are few.
template <int NG>
__device__ __forceinline__ void segment_start(const Scan& a, const Place& p,
                                              const float (&rate)[NG][4], float (&h)[NG][4]) {
  const float* outer = a.initial;
  if (a.NS > 1 && !a.folded) outer = a.ends + p.row * a.D * a.N;
  else if (outer) outer += (long)p.b * a.D * a.N;
  load_states(a, p, outer ? outer + (long)p.d * a.N : nullptr, h);
  if (!a.folded) return;
  constexpr int U = NG == 1 ? 4 : 2;
  for (int j = 0; j < p.s; j += U) {
    float end[U][NG][4], sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long row = (long)p.b * a.NS + min(j + u, p.s - 1);
      load_states(a, p, a.ends + (row * a.D + p.d) * a.N, end[u]);
      sum[u] = p.on ? a.sums[row * a.D + p.d] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= p.s) continue;
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          h[i][r] = fmaf(__builtin_amdgcn_exp2f(sum[u] * rate[i][r]), h[i][r], end[u][i][r]);
    }
  }
}

__device__ __forceinline__ void store_some(const Scan& a, const Place& p, int i, float* to,
                                           const float (&h)[4]) {
  const int n = 16 * i + 4 * p.q;
  if (p.on) store4(to + n, h, min(4, max(0, a.N - n)), a.whole_n);
}
template <int NG>
__device__ __forceinline__ void store_states(const Scan& a, const Place& p, float* to,
                                             const float (&h)[NG][4]) {
#pragma unroll
  for (int i = 0; i < NG; ++i) store_some(a, p, i, to, h[i]);
}

// The states of a channel that are kept of a tile, before its tokens 0, KEPT, ...
template <int KEPT>
__device__ __forceinline__ float* kept_at(const Scan& a, const Place& p, int tiles, int tile) {
  return a.kept + (((long)p.b * tiles + tile) * (TILE / KEPT) * a.D + p.d) * a.N;
}

// All ones where token t is before `last`, else zero.  (Were its origin known, the compiler
// would make selects of what it masks.)
__device__ __forceinline__ unsigned present(int t, int last) {
  unsigned mask = (unsigned)((t - last) >> 31);
  asm("" : "+v"(mask));
  return mask;
}

// The steps of a lane's piece.
template <typename In>
__device__ __forceinline__ void steps(const Scan& a, const Four<In>& delta, const float (&bias)[4],
                                      unsigned here, float (&s)[4]) {
  if (a.softplus) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = softplus(delta.get(e) + bias[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = delta.get(e) + bias[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = masked(s[e], here);
}

template <typename In>
__device__ __forceinline__ void widen(const Four<In>& f, float (&v)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = f.get(r);
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
// what the segment adds to the state, and the sum of its steps.  A tile's steps are
// formed while the one before is computed, and its outputs written while the next is.
// T32768 D2048 N16 bfloat16, 64 segments: 315 us and 231, both issuing a vector instruction
// in every cycle: 478 and 348 a tile and wave, 320 and 256 of them the recurrence's own; the
// rest are softplus, gate, conversions and joins.  B16 T1024 D1536, walked from end to end:
// 176 us, 1.5 waves a SIMD, which leave a third of the cycles empty; in two to four
// segments 140 and the states' 65 to 75 more.
template <typename In, int NG, bool OUT, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, OUT || !WHOLE ? 2 : 4) void scan_kernel(Scan a) {
  __shared__ f2 shared_su[WAVES][2][256];              // [16 tokens][16 channels]
  __shared__ f4 shared_y[OUT ? WAVES : 1][256];        // the same, of the four rows' states
  const Place p = place(a);
  if (p.first >= a.Dg) return;
  constexpr int KEPT = kept_tokens(NG);
  auto& su = shared_su[p.wave];
  f4* yl = shared_y[OUT ? p.wave : 0];
  float* yr = reinterpret_cast<float*>(yl);
  float rate[NG][4], h[NG][4], bias[4], skip[4], total[4] = {0.f, 0.f, 0.f, 0.f};
  load_decays(a, p, rate);
  load_bias(a.bias, p, bias);
  load_bias(a.skip, p, skip);
  if (OUT) segment_start(a, p, rate, h);
  else load_states(a, p, nullptr, h);
  const int tiles = (a.T + TILE - 1) / TILE;
  const int last = min(p.end, p.len);
  const Sources<In, NG> from(a, p, last);
  const Result<In, WHOLE> out(a, p, a.out);
  using RowsOf = TileRows<In, NG, OUT, false, WHOLE>;

  const auto stage = [&](const RowsOf& rows, int t0, f2* to) {
    float s[4];
    steps(a, rows.delta, bias, present(t0 + p.token, last), s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      to[p.token * 16 + p.piece + e] = f2{s[e], s[e] * rows.x.get(e)};
      if (!OUT) total[e] += s[e];
    }
  };
  const auto finish = [&](const Four<In>& x, const Four<In>& gate, int t0) {
    const unsigned here = present(t0 + p.token, last);
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f4 v = yl[p.token * 16 + p.piece + e];
      o[e] = (v[0] + v[2]) + (v[1] + v[3]);
    }
    if (a.skip)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(skip[e], x.get(e), o[e]);
    if (a.gated)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = gate.get(e);
        o[e] *= z * sigmoid(z);
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = masked(o[e], here);
    out.put(a, p, t0, o);
  };

  if (p.begin < last) {
    RowsOf now, next;
    Four<In> x, gate;  // of the tile before
    now.fetch(a, p, from, p.begin, last);
    stage(now, p.begin, su[0]);
    next.fetch(a, p, from, p.begin + TILE, last);
    wave_sync();
    int turn = 0;
    for (int t0 = p.begin; t0 < last; t0 += TILE) {
      float* kept = nullptr;
      if (OUT && a.kept) kept = kept_at<KEPT>(a, p, tiles, t0 / TILE);
      stage(next, t0 + TILE, su[turn ^ 1]);
      if (OUT && t0 > p.begin) finish(x, gate, t0 - TILE);
      wave_sync();
      float y[TILE];
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float bv[4], cv[4];
        widen(now.b[i], bv);
        widen(now.c[i], cv);
        settled(bv, cv);
        unroll<0, TILE>([&](auto k) {
          constexpr int t = k.value;
          if (OUT && t % KEPT == 0 && kept)
            store_some(a, p, i, kept + t / KEPT * (long)a.D * a.N, h[i]);
          const f2 v = su[turn][t * 16 + p.ch];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float keep = __builtin_amdgcn_exp2f(v.x * rate[i][r]);
            h[i][r] = fmaf(keep, h[i][r], mul_row<t>(bv[r], v.y));
            if (OUT) add_row<t>(y[t], cv[r], h[i][r], i == 0 && r == 0);
          }
          if (OUT && i == NG - 1) yr[(t * 16 + p.ch) * 4 + p.q] = y[t];
        });
      }
      if (OUT) {
        x = now.x;
        gate = now.gate;
      }
      now = next;
      next.fetch(a, p, from, t0 + 2 * TILE, last);
      wave_sync();
      turn ^= 1;
    }
    if (OUT) {
      const int t0 = p.begin + (last - 1 - p.begin) / TILE * TILE;
      finish(x, gate, t0);
    }
  }
  if (!OUT) {
    store_states(a, p, a.ends + (p.row * a.D + p.d) * a.N, h);
    store_token_sums(p, total, a.sums + p.row * a.D);
    return;
  }
  if (p.s == a.NS - 1) store_states(a, p, a.state + ((long)p.b * a.D + p.d) * a.N, h);
  // Tiles without a token that is present.
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = p.begin + (max(0, last - p.begin) + TILE - 1) / TILE * TILE; t < p.end; t += TILE)
    out.put(a, p, t, zero);
}

// What each segment starts from, in the place of what it adds: h <- exp(a sum s) h + end.
// Bound by latency: a chain over the segments, 6 us for 16 (B8 T1000 D768 N16), 12 for 64
// (T32768 D2048).  The forward of few segments does without.
// Backward: from the last to the first, from the state's cotangent.  (What the last one of
// these adds is not needed, nor formed.)
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
    // A batch of segments is loaded at a time: one after the other, each would wait for
    // memory (B1 T2000 D1536 N16, 42 segments: 12 us).
    constexpr int U = 8;
    for (int j = 0; j < a.NS; j += U) {
      float end[U], keep[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long row = b * a.NS + (BWD ? max(0, a.NS - 1 - j - u) : min(a.NS - 1, j + u));
        end[u] = a.ends[row * each + rest];
        keep[u] = __builtin_amdgcn_exp2f(a.sums[row * a.D + d] * v);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j + u >= a.NS) continue;
        const long row = b * a.NS + (BWD ? a.NS - 1 - j - u : j + u);
        a.ends[row * each + rest] = h;
        h = fmaf(keep[u], h, end[u]);
      }
    }
  }
}

// ------------------------------------------------------------ backward

// ALL: a segment's gradients from the cotangent of the state after it; else what the
// segment adds to the cotangent of the state before it, and the sum of its steps.  A
// tile (or half of one) is walked forwards from the state that the forward call kept, its
// states and decays staying in registers, then backwards.  B16 T1024 D1536 N16 bfloat16, 4
// segments: 379 us and 88.  Two waves a SIMD issue in 77% of the cycles; three with half
// tiles came to the same (406 us for 387), and half tiles' twice as many kept states buy
// registers only for more than 16 states, where whole ones spill 54 to 165 a lane (N64
// training 2370 us, so 2116).  Of 1,510 vector instructions a tile and wave 900 are the
// recurrences', 290 the sums over a row's channels (through LDS: 439 us).
template <typename In, int NG, bool ALL, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, ALL || !WHOLE ? 2 : 4) void scan_backward_kernel(Scan a) {
  // A wave's steps, inflows, cotangents and x [16 tokens][16 channels], two sums over the
  // states of each row of lanes of the same shape, and every wave's sums over channels [16
  // tokens][16 states].
  __shared__ f4 shared_in[WAVES][2][256];
  __shared__ f4 shared_rows[ALL ? WAVES : 1][2][256];
  __shared__ float sums[ALL ? 2 : 1][WAVES][2][ALL ? 256 : 1];
  const Place p = place(a);
  const bool idle = p.first >= a.Dg;
  if (!ALL && idle) return;
  const int active = min(WAVES, (a.Dg - p.block * BLOCK_CHANNELS + 15) / 16);
  constexpr int KEPT = kept_tokens(NG);
  auto& in = shared_in[p.wave];
  auto& row_sums = shared_rows[ALL ? p.wave : 0];
  float* const rows0 = reinterpret_cast<float*>(row_sums[0]);
  float* const rows1 = reinterpret_cast<float*>(row_sums[1]);
  float rate[NG][4], g[NG][4], da[NG][4], bias[4], skip[4];
  float dskip[4] = {0.f, 0.f, 0.f, 0.f}, dbias[4] = {0.f, 0.f, 0.f, 0.f};
  load_decays(a, p, rate);
  load_bias(a.bias, p, bias);
  load_bias(a.skip, p, skip);
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) da[i][r] = 0.f;
  const float* begin = nullptr;
  if (ALL)
    begin = a.NS > 1 ? a.ends + (p.row * a.D + p.d) * a.N
           : a.dstate ? a.dstate + ((long)p.b * a.D + p.d) * a.N : nullptr;
  load_states(a, p, begin, g);
  const int tiles = (a.T + TILE - 1) / TILE;
  const int first = p.begin / TILE, last = min(p.end, p.len);
  const Sources<In, NG> from(a, p, last);
  const Result<In, WHOLE> dxs(a, p, a.dx), dds(a, p, a.ddelta), dzs(a, p, a.dgate);
  using RowsOf = TileRows<In, NG, true, true, WHOLE>;

  // Whether there are registers for the steps and cotangents of a lane's piece until its
  // results are formed (B16 T1024 D1536 N16 bfloat16 training 626 us from LDS, 607 so);
  // float32 and more states would spill others (648 us from LDS, 711 so).
  constexpr bool HELD = NG == 1 && sizeof(In) == 2;
  float s[4], dy[4];  // of the tile that is staged
  const auto stage = [&](const RowsOf& rows, int t0, f4* to) {
    steps(a, rows.delta, bias, present(t0 + p.token, last), s);
#pragma unroll
    for (int e = 0; e < 4; ++e) dy[e] = rows.dout.get(e);
    if (a.gated)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = rows.gate.get(e);
        dy[e] *= z * sigmoid(z);
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = rows.x.get(e);
      to[p.token * 16 + p.piece + e] = f4{s[e], s[e] * x, dy[e], x};
      if (!ALL) dbias[e] += s[e];
    }
  };

  // From the last tile with a token that is present.
  int tile = (last + TILE - 1) / TILE - 1;
  if (tile >= first) {
    RowsOf now, next;
    now.fetch(a, p, from, tile * TILE, last);
    stage(now, tile * TILE, in[0]);
    if (tile > first) next.fetch(a, p, from, (tile - 1) * TILE, last);
    constexpr int PARTS = TILE / KEPT;
    const long part_stride = (long)a.D * a.N;
    float start[PARTS][NG][4];
    const auto load_starts = [&](int of) {
#pragma unroll
      for (int j = 0; j < PARTS; ++j)
        load_states(a, p, kept_at<KEPT>(a, p, tiles, of) + j * part_stride, start[j]);
    };
    if (ALL) load_starts(tile);
    wave_sync();
    int turn = 0;
    for (; tile >= first; --tile) {
      const int t0 = tile * TILE;
      const f4* sud = in[turn];
      if constexpr (!ALL) {
        if (tile > first) stage(next, t0 - TILE, in[turn ^ 1]);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          float cv[4], none[4] = {0.f, 0.f, 0.f, 0.f};
          widen(now.c[i], cv);
          settled(cv, none);
          unroll<0, TILE>([&](auto k) {
            constexpr int t = TILE - 1 - k.value;
            const f4 v = sud[t * 16 + p.ch];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              fmac_row<t>(g[i][r], cv[r], v.z);
              g[i][r] *= __builtin_amdgcn_exp2f(v.x * rate[i][r]);
            }
          });
        }
        now = next;
        if (tile > first + 1) next.fetch(a, p, from, t0 - 2 * TILE, last);
        wave_sync();
      } else {
        float yv[4] = {0.f, 0.f, 0.f, 0.f}, fv[4] = {0.f, 0.f, 0.f, 0.f},
              sv[4] = {0.f, 0.f, 0.f, 0.f};
        const auto join = [&](const f4* from, unsigned mask, float (&sum)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f4 v = from[p.token * 16 + p.piece + e];
            sum[e] += masked((v[0] + v[2]) + (v[1] + v[3]), mask);
          }
        };
        int side = NG == 1 ? turn : 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          auto& mine = sums[side][p.wave];
          if (!idle) {
            float bv[4], cv[4];
            widen(now.b[i], bv);
            widen(now.c[i], cv);
            settled(bv, cv);
            // Bank j of row q: state 4 q + (j with its bits swapped).
            const int n = 4 * p.q + ((p.ch >> 3) | (p.ch >> 1 & 2));
            unroll<0, PARTS>([&](auto of) {
              constexpr int o = PARTS - 1 - of.value, t0 = o * KEPT;
              float h[KEPT][4], keep[KEPT][4];
              unroll<0, KEPT>([&](auto k) {
                constexpr int t = t0 + k.value;
                const f4 v = sud[t * 16 + p.ch];
                float y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float before = k.value ? h[k.value ? k.value - 1 : 0][r] : start[o][i][r];
                  keep[k.value][r] = __builtin_amdgcn_exp2f(v.x * rate[i][r]);
                  h[k.value][r] = fmaf(keep[k.value][r], before, mul_row<t>(bv[r], v.y));
                  add_row<t>(y, cv[r], h[k.value][r], r == 0);
                }
                rows0[(t * 16 + p.ch) * 4 + p.q] = y;
              });
              wave_sync();
              join(row_sums[0], PARTS == 1 || p.token / KEPT == o ? ~0u : 0u, yv);
              wave_sync();
              unroll<0, KEPT>([&](auto back) {
                constexpr int k = KEPT - 1 - back.value, t = t0 + k;
                const f4 v = sud[t * 16 + p.ch];
                float pb[4], pc[4], sb, sc, flow, slope;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float before = k ? h[k ? k - 1 : 0][r] : start[o][i][r];
                  fmac_row<t>(g[i][r], cv[r], v.z);
                  pc[r] = h[k][r] * v.z;
                  pb[r] = g[i][r] * v.y;
                  add_row<t>(flow, bv[r], g[i][r], r == 0);
                  g[i][r] *= keep[k][r];
                  const float m = g[i][r] * before;
                  slope = r ? fmaf(m, rate[i][r], slope) : m * rate[i][r];
                  da[i][r] = fmaf(m, v.x, da[i][r]);
                }
                join_lanes(pb, pc, sb, sc);
                mine[0][t * 16 + n] = sb;
                mine[1][t * 16 + n] = sc;
                rows0[(t * 16 + p.ch) * 4 + p.q] = slope;
                rows1[(t * 16 + p.ch) * 4 + p.q] = flow;
              });
            });
            wave_sync();
            join(row_sums[0], ~0u, sv);
            join(row_sums[1], ~0u, fv);
            wave_sync();
          }
          __syncthreads();
          // The block's channels, in their order.
          const int t = threadIdx.x >> 4, n = 16 * i + (threadIdx.x & 15);
          float db = 0.f, dc = 0.f;
          for (int w = 0; w < active; ++w) {
            db += sums[side][w][0][threadIdx.x];
            dc += sums[side][w][1][threadIdx.x];
          }
          if (n < a.N && t0 + t < last) {
            const long tokens = (long)a.B * a.T;
            float* to = a.part_bc +
                        ((p.block * tokens + (long)p.b * a.T + t0 + t) * a.G + p.g) * 2 * a.N + n;
            to[0] = db;
            to[a.N] = dc;
          }
          side ^= 1;
        }
        const RowsOf was = now;
        f4 piece[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          piece[e] = HELD ? f4{s[e], 0.f, dy[e], was.x.get(e)} : sud[p.token * 16 + p.piece + e];
        now = next;
        if (tile > first) {
          stage(now, t0 - TILE, in[turn ^ 1]);
          load_starts(tile - 1);
        }
        if (tile > first + 1) next.fetch(a, p, from, t0 - 2 * TILE, last);
        if (!idle) {
          const unsigned here = present(t0 + p.token, last);
          float dx[4], dd[4], whole[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            whole[e] = yv[e];
            dx[e] = piece[e].x * fv[e];
            dd[e] = fmaf(piece[e].w, fv[e], sv[e] * LN2);
            dskip[e] = fmaf(piece[e].z, piece[e].w, dskip[e]);
          }
          if (a.skip)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              whole[e] = fmaf(skip[e], piece[e].w, whole[e]);
              dx[e] = fmaf(skip[e], piece[e].z, dx[e]);
            }
          if (a.softplus)
#pragma unroll
            for (int e = 0; e < 4; ++e) dd[e] *= sigmoid(was.delta.get(e) + bias[e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dx[e] = masked(dx[e], here);
            dd[e] = masked(dd[e], here);
            dbias[e] += dd[e];
          }
          dxs.put(a, p, t0, dx);
          dds.put(a, p, t0, dd);
          if (a.dgate) {
            float dz[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float z = was.gate.get(e), sg = sigmoid(z);
              dz[e] = masked(was.dout.get(e) * whole[e] * (sg * fmaf(z, 1.f - sg, 1.f)), here);
            }
            dzs.put(a, p, t0, dz);
          }
        }
        wave_sync();
      }
      turn ^= 1;
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
  if (p.s == 0 && a.dinitial)
    store_states(a, p, a.dinitial + ((long)p.b * a.D + p.d) * a.N, g);
  // Tiles without a token that is present.
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = p.begin + (max(0, last - p.begin) + TILE - 1) / TILE * TILE; t < p.end; t += TILE) {
    dxs.put(a, p, t, zero);
    dds.put(a, p, t, zero);
    if (a.dgate) dzs.put(a, p, t, zero);
  }
}

// Bound by latency and memory (B16 T1024 D1536: 11 us for 50 MB of parts).
// The gradients of b and c: the sums over the channel blocks, in their order; by the
// first `bc_blocks` blocks.  By the rest those of a, skip and the bias: the sums over the
// batch rows and segments, in four parts, joined in their order.
template <typename In>
__global__ __launch_bounds__(256) void join_kernel(Join a) {
  constexpr int U = 8;
  if (blockIdx.x < a.bc_blocks) {
    const long each = (long)a.G * a.N, tokens = (long)a.B * a.T, count = tokens * each;
    const long stride = 2 * tokens * each;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += a.bc_blocks * 256L) {
      const long token = i / each, rest = i - token * each;
      const long g = rest / a.N, n = rest - g * a.N;
      const long b = token / a.T;
      const bool here = !a.lengths || token - b * a.T < a.lengths[b];
      const float* from = a.part_bc + (token * a.G + g) * 2 * a.N + n;
      float db = 0.f, dc = 0.f;
      if (here)
        for (int j = 0; j < a.blocks; j += U) {
          float vb[U], vc[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const long at = min(j + u, a.blocks - 1) * stride;
            vb[u] = from[at];
            vc[u] = from[at + a.N];
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (j + u < a.blocks) {
              db += vb[u];
              dc += vc[u];
            }
        }
      if constexpr (sizeof(In) == 4) {
        static_cast<float*>(a.db)[i] = db;
        static_cast<float*>(a.dc)[i] = dc;
      } else {
        static_cast<bf16_t*>(a.db)[i] = (bf16_t)pack(db, 0.f);
        static_cast<bf16_t*>(a.dc)[i] = (bf16_t)pack(dc, 0.f);
      }
    }
    return;
  }
  __shared__ float fold[256];
  const int slice = threadIdx.x >> 6;
  const long states = (long)a.D * a.N;
  const long i = (long)(blockIdx.x - a.bc_blocks) * 64 + (threadIdx.x & 63);
  const bool on = i < states + 2L * a.D, of_a = i < states;
  const float* from = of_a ? a.part_a + i : a.part_d + (i - states);
  const long stride = of_a ? states : 2L * a.D;
  const long quarter = (a.rows + 3) / 4, end = min(a.rows, (slice + 1) * quarter);
  float s = 0.f;
  for (long j = slice * quarter; on && j < end; j += U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = from[min(j + u, end - 1) * stride];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u < end) s += v[u];
  }
  fold[threadIdx.x] = s;
  __syncthreads();
  if (slice || !on) return;
  for (int k = 1; k < 4; ++k) s += fold[threadIdx.x + 64 * k];
  const long d = i - states;
  float* to = of_a ? a.da : d < a.D ? a.dskip : a.dbias;
  if (to) to[of_a ? i : d < a.D ? d : d - a.D] = s;
}

// ------------------------------------------------------------ one token

// Bound by memory: the states are read and written once.  2^span lanes hold a channel,
// four states each, and take ROWS batch rows, whose loads are in flight together; what
// belongs to the channel stays in registers.  2,048 rows of D1536 N16 bfloat16 in place, an
// tenth of them idle: 95 us for 0.39 GB, 4.1 TB/s (one row a thread 149, two 105, eight 125;
// states past the caches, as here where there are several rows: 104 without); 4 rows 3.6 us.
template <typename In, int ROWS>
__global__ __launch_bounds__(STEP_THREADS) void step_kernel(Step a) {
  const int rows = blockIdx.x / a.blocks;
  const long i = (long)(blockIdx.x - rows * a.blocks) * STEP_THREADS + threadIdx.x;
  const int d = (int)(i >> a.span), n = 4 * ((int)i & ((1 << a.span) - 1));
  if (d >= a.D) return;
  const int g = d / a.Dg, have = min(4, max(0, a.N - n));
  const auto one = [](const void* p, long at) {
    const In v = static_cast<const In*>(p)[at];
    if constexpr (sizeof(In) == 4) return (float)v;
    else return __uint_as_float((unsigned)v << 16);
  };
  Four<float> rate = load4(a.a + (long)d * a.N + n, have, a.whole_n);
  const float bias = a.bias ? a.bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
  const long first = (long)rows * ROWS;
  constexpr bool ONCE = ROWS > 1;
  const auto load_state = [](const Step& a, long at, int have) {
    Four<float> v;
    v.r = 0;
    if (!ONCE || !a.whole_n) v = load4(a.state + at, have, a.whole_n);
    else if (have > 0) v.r = __builtin_nontemporal_load(reinterpret_cast<const f4*>(a.state + at));
    return v;
  };
  const auto store_state = [](const Step& a, long at, const float (&v)[4], int have) {
    if (!ONCE || !a.whole_n)
      store4(a.new_state + at, v, have, a.whole_n);
    else if (have > 0)
      __builtin_nontemporal_store(f4{v[0], v[1], v[2], v[3]},
                                  reinterpret_cast<f4*>(a.new_state + at));
  };
  Four<float> h[ROWS];
  Four<In> b[ROWS], c[ROWS];
  float x[ROWS], delta[ROWS], z[ROWS];
  bool on[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const long row = first + j;
    on[j] = row < a.B && (!a.active || a.active[row]);
    if (on[j] || (row < a.B && a.new_state != a.state))
      h[j] = load_state(a, (row * a.D + d) * a.N + n, have);
    if (!on[j]) continue;
    b[j] = load4(static_cast<const In*>(a.b.p) + row * a.b.batch + g * a.bg + n, have, a.whole_bc);
    c[j] = load4(static_cast<const In*>(a.c.p) + row * a.c.batch + g * a.cg + n, have, a.whole_bc);
    x[j] = one(a.x.p, row * a.x.batch + d);
    delta[j] = one(a.delta.p, row * a.delta.batch + d);
    if (a.gate.p) z[j] = one(a.gate.p, row * a.gate.batch + d);
  }
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const long row = first + j;
    if (row >= a.B) return;
    float v[4], y = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = h[j].get(r);
    if (on[j]) {
      float s = delta[j] + bias;
      if (a.softplus) s = softplus(s);
      const float u = s * x[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = fmaf(__builtin_amdgcn_exp2f(s * (rate.get(r) * LOG2E)), v[r], u * b[j].get(r));
        y = fmaf(c[j].get(r), v[r], y);
      }
    }
    if (on[j] || a.new_state != a.state)
      store_state(a, (row * a.D + d) * a.N + n, v, have);
    for (int m = 1; m < 1 << a.span; m *= 2) y += __shfl_xor(y, m);
    if (n) continue;
    if (on[j]) {
      if (a.skip) y = fmaf(skip, x[j], y);
      if (a.gate.p) y *= z[j] * sigmoid(z[j]);
    }
    if constexpr (sizeof(In) == 4) static_cast<float*>(a.out)[row * a.D + d] = y;
    else static_cast<bf16_t*>(a.out)[row * a.D + d] = (bf16_t)pack(y, 0.f);
  }
}

#define M4SL_SCAN_GROUPS(In, NG)                                            \
  template __global__ void scan_kernel<In, NG, true, true>(Scan);           \
  template __global__ void scan_kernel<In, NG, true, false>(Scan);          \
  template __global__ void scan_kernel<In, NG, false, true>(Scan);          \
  template __global__ void scan_kernel<In, NG, false, false>(Scan);         \
  template __global__ void scan_backward_kernel<In, NG, true, true>(Scan);  \
  template __global__ void scan_backward_kernel<In, NG, true, false>(Scan); \
  template __global__ void scan_backward_kernel<In, NG, false, true>(Scan); \
  template __global__ void scan_backward_kernel<In, NG, false, false>(Scan);
#define M4SL_SCAN(In)                                \
  M4SL_SCAN_GROUPS(In, 1)                            \
  M4SL_SCAN_GROUPS(In, 2)                            \
  M4SL_SCAN_GROUPS(In, 4)                            \
  template __global__ void join_kernel<In>(Join);    \
  template __global__ void step_kernel<In, 1>(Step); \
  template __global__ void step_kernel<In, 4>(Step);
M4SL_SCAN(float)
M4SL_SCAN(bf16_t)
template __global__ void carry_kernel<false>(Scan);
template __global__ void carry_kernel<true>(Scan);

}  // namespace ss

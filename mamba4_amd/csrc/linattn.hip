// Decayed linear attention for gfx950.
//
// Per batch row and head, with keys and queries of width n and values of p:
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t.
// In chunks of 64 tokens, P the chunk's running sum of g:
//   O  = scale (A V + e^{P_i} Q S),   A_ij = (q_i . k_j) e^{P_i - P_j}, j <= i,
//   S <- e^{P_L} S + (K e^{P_L - P_j})^T V.
// The gradients are three more of the same:
//   dQ = scale attention(dO, V, K) on the state S^T,
//   dV = attention(K, Q, dO) and dK = attention(V, dO, Q) with time reversed,
//        on the cotangent R of the state and R^T
//        (R <- e^{P_L} R + scale (Q e^{P_i})^T dO, weights e^{P_i - P_j}, i >= j),
//   dg_t = <S_T, R_T> + sum over i >= t of (q_i . dq_i - k_i . dk_i),
// which sums (q_i . k_j)(do_i . v_j) scale e^{P_i - P_j} over pairs i >= t > j
// (the pairs i = j are in both products and left out of both).  The sums start
// anew at each segment's end with <S, R> there, so that they do not cancel over
// the whole sequence.
// So one body serves all of them ("roles"); a block walks the chunks of one
// (b, h) for 64 columns of the values, keeping the state in registers.
//
// Products run on bfloat16 MFMA with float32 accumulation.  An operand is a sum of
// bfloat16 planes: a bfloat16 input is one plane; what is computed in float32 is
// three planes (all 24 bits) where the result is float32 (the weighted K of the
// states, A and S where dg follows from the output), and two beside bfloat16
// inputs where it is rounded to bfloat16 (2^-17 of A and S left out; one plane saved
// a tenth of the time and left an error like that rounding's own).  Float32 inputs
// are three planes, with the six largest plane products: a sixth of the bfloat16
// rate, 2.7 times that of float32 MFMA.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "linattn.hpp"

namespace la {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr unsigned kNoLoad = 0x80000000u;  // an offset past every resource

__device__ __forceinline__ Rsrc rsrc(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}

template <typename In>
struct Type;
template <>
struct Type<bf16_t> {
  static constexpr int IN = 1, ROUGH = 2;  // planes of an input, of an operand of rounded results
};
template <>
struct Type<float> {
  static constexpr int IN = 3, ROUGH = 3;
};
constexpr int FINE = 3;  // planes of a computed operand of a float32 result

// Eight consecutive elements as loaded.
template <typename In>
struct Piece {
  u4 w[sizeof(In) / 2];
};

// MFMA operand fragments of 16x16x32: lane (g, r) = (lane >> 4, lane & 15)
// holds row (or column) r at eight of the 32 k, as PLANES bfloat16 planes.
template <int PLANES>
struct Frag {
  b8 p[PLANES];
};

__device__ __forceinline__ unsigned pack(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}
__device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// Two float32 values as bfloat16 planes: each plane is what is left of them,
// rounded to the nearest.
template <int PLANES>
__device__ __forceinline__ void split2(float a, float b, unsigned (&out)[PLANES]) {
#pragma unroll
  for (int i = 0; i < PLANES; ++i) {
    out[i] = pack(a, b);
    a -= low(out[i]);
    b -= high(out[i]);
  }
}

template <int PLANES>
__device__ __forceinline__ Frag<PLANES> split8(const float (&x)[8]) {
  u4 w[PLANES];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    unsigned part[PLANES];
    split2<PLANES>(x[2 * e], x[2 * e + 1], part);
#pragma unroll
    for (int i = 0; i < PLANES; ++i) w[i][e] = part[i];
  }
  Frag<PLANES> f;
#pragma unroll
  for (int i = 0; i < PLANES; ++i) f.p[i] = __builtin_bit_cast(b8, w[i]);
  return f;
}

__device__ __forceinline__ Frag<1> planes(const Piece<bf16_t>& x) {
  return Frag<1>{{__builtin_bit_cast(b8, x.w[0])}};
}
__device__ __forceinline__ Frag<3> planes(const Piece<float>& x) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(x.w[e >> 2][e & 3]);
  return split8<3>(v);
}

// acc[i] += a[i] b over the plane products that count: the sum of the planes'
// indexes below the larger number of planes.  Products of different accumulators
// follow each other, so that none waits for the one before.
template <int N, int PA, int PB>
__device__ __forceinline__ void mma(const Frag<PA> (&a)[N], const Frag<PB>& b, f4* acc) {
  constexpr int most = PA > PB ? PA : PB;
#pragma unroll
  for (int s = most - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (s - i >= 0 && s - i < PB)
#pragma unroll
        for (int n = 0; n < N; ++n)
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[n].p[i], b.p[s - i], acc[n], 0, 0, 0);
}
// acc[i] += a b[i].
template <int N, int PA, int PB>
__device__ __forceinline__ void mma(const Frag<PA>& a, const Frag<PB> (&b)[N], f4* acc) {
  constexpr int most = PA > PB ? PA : PB;
#pragma unroll
  for (int s = most - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (s - i >= 0 && s - i < PB)
#pragma unroll
        for (int n = 0; n < N; ++n)
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b[n].p[s - i], acc[n], 0, 0, 0);
}

// Elements col..col+7 of a row of `width` at byte offset `row`, zeros past the
// width (and past the resource): rows are whole 16-byte pieces.
__device__ __forceinline__ Piece<bf16_t> load_piece(Rsrc r, unsigned row, int col, int width,
                                                    const bf16_t*) {
  Piece<bf16_t> x;
  const unsigned off = row + 2 * col;
  x.w[0] = __builtin_bit_cast(
      u4, __builtin_amdgcn_raw_buffer_load_b128(r, col < width ? off : kNoLoad, 0, 0));
  return x;
}
__device__ __forceinline__ Piece<float> load_piece(Rsrc r, unsigned row, int col, int width,
                                                   const float*) {
  Piece<float> x;
  const unsigned off = row + 4 * col;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    x.w[i] = __builtin_bit_cast(
        u4, __builtin_amdgcn_raw_buffer_load_b128(
                r, col + 4 * i < width ? off + 16 * i : kNoLoad, 0, 0));
  return x;
}

// Elements col..col+3 as loaded, and as float32.
template <typename In>
struct Quad;
template <>
struct Quad<bf16_t> {
  u2 u;
  __device__ __forceinline__ f4 get() const {
    return f4{low(u[0]), high(u[0]), low(u[1]), high(u[1])};
  }
};
template <>
struct Quad<float> {
  f4 u;
  __device__ __forceinline__ f4 get() const { return u; }
};
__device__ __forceinline__ Quad<bf16_t> load_quad(Rsrc r, unsigned row, int col, int width,
                                                  const bf16_t*) {
  const unsigned off = row + 2 * col;
  return {__builtin_bit_cast(
      u2, __builtin_amdgcn_raw_buffer_load_b64(r, col < width ? off : kNoLoad, 0, 0))};
}
__device__ __forceinline__ Quad<float> load_quad(Rsrc r, unsigned row, int col, int width,
                                                 const float*) {
  const unsigned off = row + 4 * col;
  return {__builtin_bit_cast(
      f4, __builtin_amdgcn_raw_buffer_load_b128(r, col < width ? off : kNoLoad, 0, 0))};
}

// LDS tiles of bfloat16, 64 columns wide (wider ones are side by side): the
// 16-byte units of a row change places by the row's low bits, with which the
// transposing reads and the row reads below are free of bank conflicts (with
// rows padded by 16 bytes instead, both took twice the cycles).
__device__ __forceinline__ int unit(int row, int u) { return 64 * row + 8 * (u ^ (row & 7)); }

// SP planes of the state (0: only states are formed).
template <typename In, int NT, int SP>
struct Shared {
  alignas(16) bf16_t k[Type<In>::IN][NT][C * 64];                 // K [token][n]
  alignas(16) bf16_t v[Type<In>::IN][1][C * TILE];                // V [token][column]
  alignas(16) bf16_t s[SP ? SP : 1][NT][SP ? TILE * 64 : 8];      // S^T [column][n]
  // Each wave's own, of the chunk's tokens: the running log2 decay in two
  // parts and the decays between a token and the wave's strip (outputs), and the
  // weights of the tokens in the next state (states).
  alignas(16) float ph[SP ? WAVES : 1][C], pl[SP ? WAVES : 1][C], far[SP ? WAVES : 1][C];
  alignas(16) float update[WAVES][C];
};

__device__ __forceinline__ Frag<1> cat(s4 a, s4 b) {
  typedef short s8 __attribute__((ext_vector_type(8)));
  return Frag<1>{{__builtin_bit_cast(b8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]})}};
}

// Column fragments of a row-major tile by transposing reads: lane (g, r)
// receives column 16 cb + r of its 64 at the tokens 16 ja + 4 g + (0..3) and 16 jb
// + 4 g + (0..3).  That is the order in which the scores' accumulators hold the
// tokens of two blocks, so those are operands as they are.
template <int PLANES, int NT>
__device__ __forceinline__ Frag<PLANES> columns(const bf16_t (&tile)[PLANES][NT][C * 64], int nt,
                                                int ja, int jb, int cb, int g, int r) {
  typedef __attribute__((address_space(3))) s4* lds4;
  Frag<PLANES> f;
  const int at = unit(4 * g + (r >> 2), 2 * cb + ((r >> 1) & 1)) + 4 * (r & 1);
#pragma unroll
  for (int i = 0; i < PLANES; ++i) {
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(&tile[i][nt][at + 16 * 64 * ja]));
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(&tile[i][nt][at + 16 * 64 * jb]));
    f.p[i] = cat(a, b).p[0];
  }
  return f;
}

// Row fragments: lane (g, r) receives row r0 + r at n = 32 kk + 8 g + (0..7).
template <int PLANES, int NT>
__device__ __forceinline__ Frag<PLANES> rows(const bf16_t (&tile)[PLANES][NT][C * 64], int r0,
                                             int kk, int g, int r) {
  Frag<PLANES> f;
#pragma unroll
  for (int i = 0; i < PLANES; ++i)
    f.p[i] = __builtin_bit_cast(
        b8, *reinterpret_cast<const u4*>(
                &tile[i][kk >> 1][64 * r0 + unit(r, 4 * (kk & 1) + g)]));
  return f;
}

// A fragment with zeros in place of what is not finite.
template <int PLANES>
__device__ __forceinline__ Frag<PLANES> finite(Frag<PLANES> f) {
#pragma unroll
  for (int i = 0; i < PLANES; ++i) {
    u4 u = __builtin_bit_cast(u4, f.p[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((u[e] & 0x7f80u) == 0x7f80u) u[e] &= 0xffff0000u;
      if ((u[e] & 0x7f800000u) == 0x7f800000u) u[e] &= 0xffffu;
    }
    f.p[i] = __builtin_bit_cast(b8, u);
  }
  return f;
}

// The eight values of a fragment, times eight weights, as computed planes.
template <int MADE>
__device__ __forceinline__ Frag<MADE> weighted(const Frag<1>& f, const float (&w)[8]) {
  const u4 u = __builtin_bit_cast(u4, f.p[0]);
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = low(u[e]) * w[2 * e];
    x[2 * e + 1] = high(u[e]) * w[2 * e + 1];
  }
  return split8<MADE>(x);
}
template <int MADE>
__device__ __forceinline__ Frag<MADE> weighted(const Frag<3>& f, const float (&w)[8]) {
  const u4 a = __builtin_bit_cast(u4, f.p[0]), b = __builtin_bit_cast(u4, f.p[1]),
           c = __builtin_bit_cast(u4, f.p[2]);
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = (low(a[e]) + (low(b[e]) + low(c[e]))) * w[2 * e];
    x[2 * e + 1] = (high(a[e]) + (high(b[e]) + high(c[e]))) * w[2 * e + 1];
  }
  return split8<MADE>(x);
}

// x of the lanes below, DPP row shifts and broadcasts on both halves of a
// double; zero where there is none.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_double(double x) {
  const u2 u = __builtin_bit_cast(u2, x);
  const unsigned a = __builtin_amdgcn_update_dpp(0, u[0], CTRL, ROW_MASK, 0xf, true);
  const unsigned b = __builtin_amdgcn_update_dpp(0, u[1], CTRL, ROW_MASK, 0xf, true);
  return __builtin_bit_cast(double, u2{a, b});
}
__device__ __forceinline__ double wave_prefix(double x) {
  x += dpp_double<0x111, 0xf>(x);
  x += dpp_double<0x112, 0xf>(x);
  x += dpp_double<0x114, 0xf>(x);
  x += dpp_double<0x118, 0xf>(x);
  x += dpp_double<0x142, 0xa>(x);
  x += dpp_double<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double lane_double(double x, int lane) {
  const u2 u = __builtin_bit_cast(u2, x);
  const unsigned a = __builtin_amdgcn_readlane(u[0], lane);
  const unsigned b = __builtin_amdgcn_readlane(u[1], lane);
  return __builtin_bit_cast(double, u2{a, b});
}

// Sum over the four lanes that share r.
__device__ __forceinline__ float sum_groups(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A chunk's decays, by each wave for itself (lane = token): P, the running sum
// of log decays, in base 2.  The sum is in float64 and kept as two float32, so
// that e^{P_i - P_j} of near tokens is exact to float32 after any decay before them.
// A log decay below -2000 (-infinity, a type's lowest value) counts as -2000: its
// exponential is zero either way and the differences behind it stay finite.
__device__ __forceinline__ double running(float g) {
  return wave_prefix((double)(g < -2000.f ? -2000.f : g) * 1.4426950408889634);
}

// For the outputs of strip w.  Between strips of 16 tokens the decay is taken in
// two factors, from the key to the near end of the query's strip (`far`, a table)
// and on to the query (`near`): for decays below one neither can overflow, and the
// product costs two multiplications a score instead of an exponential.
struct Reach {
  float inter;  // of this lane's token: the state's part in its output
  float near;   // from the near end of the wave's strip (tokens of the strip)
};
template <bool REV>
__device__ __forceinline__ Reach reach(float (&ph)[C], float (&pl)[C], float (&far)[C], float g,
                                       int lane, int w) {
  const double p = running(g), edge = lane_double(p, REV ? 16 * w + 15 : 16 * w);
  const float high = (float)p, to_edge = (float)(REV ? p - edge : edge - p);
  ph[lane] = high;
  pl[lane] = (float)(p - high);
  far[lane] = __builtin_amdgcn_exp2f(to_edge);
  return Reach{__builtin_amdgcn_exp2f(REV ? (float)(lane_double(p, 63) - p) : high),
               __builtin_amdgcn_exp2f(-to_edge)};
}

// For the state: the tokens' weights; returns the chunk's decay.
template <bool REV>
__device__ __forceinline__ float weigh(float (&weights)[C], float g, int lane, float update) {
  const double p = running(g), last = lane_double(p, 63);
  weights[lane] = update * __builtin_amdgcn_exp2f((float)(REV ? p : last - p));
  return __builtin_amdgcn_exp2f((float)last);
}

// Four consecutive columns of a token's output, `left` of them within the width.
__device__ __forceinline__ void store_some(void* base, long at, f4 v, int left, bool f32) {
  if (f32) {
    float* p = static_cast<float*>(base) + at;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < left) p[q] = v[q];
  } else {
    bf16_t* p = static_cast<bf16_t*>(base) + at;
    const u2 u{pack(v[0], v[1]), pack(v[2], v[3])};
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < left) p[q] = (bf16_t)(u[q >> 1] >> (16 * (q & 1)));
  }
}

// The thread's index, opaque to the compiler: what is computed from it inside a
// loop is computed there, instead of keeping registers over the whole loop.
__device__ __forceinline__ int thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Where an operand's rows of (b, h) begin, and their token stride in bytes.
struct Source {
  const char* base;
  unsigned stride;
  int bytes;  // of one row
};
template <typename In>
__device__ __forceinline__ Source source(const Rows& x, int b, int h) {
  return Source{static_cast<const char*>(x.base) +
                    (b * x.sb + (x.share > 1 ? h / x.share : h) * x.sh) * (long)sizeof(In),
                (unsigned)(x.st * sizeof(In)), (int)(x.width * sizeof(In))};
}
// Chunk c's rows: a resource that ends with row `rows` - 1.
__device__ __forceinline__ Rsrc chunk_rows(const Source& x, int c, int rows) {
  return rsrc(x.base + (long)c * (C * (long)x.stride),
              rows > 0 ? (rows - 1) * (int)x.stride + x.bytes : 0);
}

// What a block does: 64 value columns of one (b, h), the chunks c0..c1-1 (in
// reverse if REV).
//
// A segment of a.seg chunks keeps its own state (from zero) apart from the
// state at its start; the state in use is decay * start + own.  So a split run, whose
// blocks take one segment each, has the bits of a walk over all of them.
template <typename In, int NT, bool REV>
struct Block {
  static constexpr int IN = Type<In>::IN;
  static constexpr int KP = 2 * NT;               // pieces of K a thread loads
  static constexpr int GROUP = IN > 1 ? 2 : 4;    // products between which no wait is needed
  const Args& a;
  const Role& R;
  int tile, b, h, w;
  int col0, bh, length;
  const float* gs;

  __device__ __forceinline__ Block(const Args& args, const Role& role, int tile_, int b_, int h_)
      : a(args), R(role), tile(tile_), b(b_), h(h_) {
    w = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & (WAVES - 1));
    col0 = TILE * tile;
    bh = b * a.H + h;
    length = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    gs = a.g + b * a.gb + h;
  }
  __device__ __forceinline__ int have(int c) const { return min(length - c * C, C); }
  // Whether the decays' tables have to be formed for chunk c: a constant decay's are
  // those of any chunk with as many tokens.
  __device__ __forceinline__ bool unknown(int c, int* known) const {
    const bool fresh = a.gt != 0 || have(c) != *known;
    *known = have(c);
    return fresh;
  }
  __device__ __forceinline__ float decay(int c, int lane) const {
    return lane < have(c) ? gs[((long)c * C + lane) * a.gt] : 0.f;
  }
  __device__ __forceinline__ void fetch_k(Piece<In> (&raw)[KP], const Source& src, int c, int t) {
    const int col = 8 * (t & (8 * NT - 1)), row = t / (8 * NT);
    const Rsrc r = chunk_rows(src, c, have(c));
#pragma unroll
    for (int i = 0; i < KP; ++i)
      raw[i] = load_piece(r, (row + 32 / NT * i) * src.stride, col, R.n, (const In*)nullptr);
  }
  __device__ __forceinline__ void fetch_v(Piece<In> (&raw)[2], const Source& src, int c, int t) {
    const int col = 8 * (t & 7), row = t >> 3;
    const Rsrc r = chunk_rows(src, c, have(c));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      raw[i] = load_piece(r, (row + 32 * i) * src.stride, col0 + col, R.p,
                                 (const In*)nullptr);
  }
  template <typename Sh>
  __device__ __forceinline__ void stage_k(Sh& sh, const Piece<In> (&raw)[KP], int t) {
    const int col = 8 * (t & (8 * NT - 1)), row = t / (8 * NT);
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const Frag<IN> f = planes(raw[i]);
#pragma unroll
      for (int j = 0; j < IN; ++j)
        *reinterpret_cast<u4*>(&sh.k[j][col >> 6][unit(row + 32 / NT * i, (col >> 3) & 7)]) =
            __builtin_bit_cast(u4, f.p[j]);
    }
  }
  template <typename Sh>
  __device__ __forceinline__ void stage_v(Sh& sh, const Piece<In> (&raw)[2], int t) {
    const int col = 8 * (t & 7), row = t >> 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Frag<IN> f = planes(raw[i]);
#pragma unroll
      for (int j = 0; j < IN; ++j)
        *reinterpret_cast<u4*>(&sh.v[j][0][unit(row + 32 * i, col >> 3)]) =
            __builtin_bit_cast(u4, f.p[j]);
    }
  }

  // The blocks of 16 keys in turn from a wave's own strip, into the past (REV:
  // the future) and round: the first `seen` of them reach the strip's queries.
  __device__ __forceinline__ static int seen(int strip) { return REV ? WAVES - strip : strip + 1; }
  __device__ __forceinline__ static int block(int strip, int i) {
    return (REV ? strip + i : strip - i) & (WAVES - 1);
  }
  // The strip, opaque, so that the addresses that follow from it are not kept in
  // registers over the loop.
  __device__ __forceinline__ int opaque_strip() const {
    int strip = w;
    asm volatile("" : "+s"(strip));
    return strip;
  }

  // State rows n = 64 nt + 16 w + 4 g + q, columns 16 pb + r: own <- decay own +
  // weighted K^T V.
  template <typename Sh>
  __device__ __forceinline__ void advance(Sh& sh, f4 (&own)[NT][4], float decay, int g, int r) {
    const int strip = opaque_strip();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int pb = 0; pb < 4; ++pb) own[nt][pb] *= decay;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int ja = block(strip, 2 * s), jb = block(strip, 2 * s + 1);
      const f4 ua = *reinterpret_cast<const f4*>(&sh.update[w][16 * ja + 4 * g]);
      const f4 ub = *reinterpret_cast<const f4*>(&sh.update[w][16 * jb + 4 * g]);
      const float wt[8] = {ua[0], ua[1], ua[2], ua[3], ub[0], ub[1], ub[2], ub[3]};
      Frag<FINE> kw[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        kw[nt] = weighted<FINE>(columns<IN, NT>(sh.k, nt, ja, jb, w, g, r), wt);
#pragma unroll
      for (int p0 = 0; p0 < 4; p0 += GROUP) {
        Frag<IN> vf[GROUP];
#pragma unroll
        for (int pb = 0; pb < GROUP; ++pb)
          vf[pb] = columns<IN, 1>(sh.v, 0, ja, jb, p0 + pb, g, r);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma(kw[nt], vf, &own[nt][p0]);
      }
    }
  }

  __device__ __forceinline__ float* slot(int seg) const {
    return R.starts + ((long)(tile * a.B * a.H + bh) * a.NS + seg) * (NT * 4096);
  }

  // Split runs: the segment's own state, from zero, and its decay.  Four waves.
  __device__ __forceinline__ void states(int seg, int c0, int c1, Shared<In, NT, 0>& sh) {
    f4 own[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int pb = 0; pb < 4; ++pb) own[nt][pb] = f4{0.f, 0.f, 0.f, 0.f};
    float since = 1.f;
    const Source ks = source<In>(R.k, b, h), vs = source<In>(R.v, b, h);
    Piece<In> kraw[KP], vraw[2];
    float graw;
    auto fetch = [&](int c) {
      const int t = thread();
      fetch_k(kraw, ks, c, t);
      fetch_v(vraw, vs, c, t);
      graw = decay(c, t & 63);
    };
    fetch(REV ? c1 - 1 : c0);
    float whole = 1.f;
    int known = -1;
    for (int it = 0; it < c1 - c0; ++it) {
      const int c = REV ? c1 - 1 - it : c0 + it;
      const int t = thread(), lane = t & 63;
      if (have(c) > 0) {
        stage_k(sh, kraw, t);
        stage_v(sh, vraw, t);
        if (unknown(c, &known)) whole = weigh<REV>(sh.update[w], graw, lane, R.update);
      }
      __syncthreads();
      if (it + 1 < c1 - c0) fetch(REV ? c - 1 : c + 1);
      if (have(c) > 0) {
        since *= whole;
        advance(sh, own, whole, lane >> 4, lane & 15);
      }
      __syncthreads();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int pb = 0; pb < 4; ++pb)
        *reinterpret_cast<f4*>(slot(seg) + ((nt * 4 + pb) * 64 * WAVES + threadIdx.x) * 4) =
            own[nt][pb];
    if (threadIdx.x == 0) R.decays[(long)(tile * a.B * a.H + bh) * a.NS + seg] = since;
  }

  // Outputs from the state at the first chunk.  Eight waves: four form the
  // outputs of a strip of 16 tokens each, four keep the state (16 rows of its n
  // and of every 64 each), so that a chunk's two halves run beside each other.
  template <int SP, bool DOTS>
  __device__ __forceinline__ void outputs(int seg, int c0, int c1, Shared<In, NT, SP>& sh) {
    if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) < WAVES)
      write_outputs<SP, DOTS>(c0, c1, sh);
    else
      keep_state<SP, DOTS>(seg, c0, c1, sh);
  }

  template <int SP, bool DOTS>
  __device__ __forceinline__ void keep_state(int seg, int c0, int c1, Shared<In, NT, SP>& sh) {
    f4 start[NT][4], own[NT][4];
    float since = 1.f;  // decay since the segment's start
    {
      const int t = thread() & (64 * WAVES - 1), g = (t >> 4) & 3, r = t & 15;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pb = 0; pb < 4; ++pb) {
          own[nt][pb] = start[nt][pb] = f4{0.f, 0.f, 0.f, 0.f};
          if (seg >= 0) {
            start[nt][pb] = *reinterpret_cast<const f4*>(
                slot(seg) + ((nt * 4 + pb) * 64 * WAVES + t) * 4);
          } else if (R.initial.base) {
            const float* s = R.initial.base + (long)bh * R.n * R.p;
            const int p = col0 + 16 * pb + r;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int n = 64 * nt + 16 * w + 4 * g + q;
              if (n < R.n && p < R.p)
                start[nt][pb][q] = s[(long)n * R.initial.sn + (long)p * R.initial.sp];
            }
          }
        }
    }
    const Source ks = source<In>(R.k, b, h);
    Piece<In> kraw[KP];
    float graw;
    auto fetch = [&](int c) {
      const int t = thread() & (64 * WAVES - 1);
      fetch_k(kraw, ks, c, t);
      graw = decay(c, t & 63);
    };
    fetch(REV ? c1 - 1 : c0);
    float whole = 1.f;
    int known = -1;
    for (int it = 0; it < c1 - c0; ++it) {
      const int c = REV ? c1 - 1 - it : c0 + it;
      const int t = thread() & (64 * WAVES - 1), lane = t & 63, g = lane >> 4, r = lane & 15;
      if (have(c) > 0) {
        stage_k(sh, kraw, t);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int pb = 0; pb < 4; ++pb) {
            float s[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) s[q] = fmaf(since, start[nt][pb][q], own[nt][pb][q]);
            unsigned lo[SP], hi[SP];
            split2<SP>(s[0], s[1], lo);
            split2<SP>(s[2], s[3], hi);
#pragma unroll
            for (int j = 0; j < SP; ++j)
              *reinterpret_cast<u2*>(
                  &sh.s[j][nt][64 * 16 * pb + unit(r, 2 * w + (g >> 1)) + 4 * (g & 1)]) =
                  u2{lo[j], hi[j]};
          }
        if (unknown(c, &known)) whole = weigh<REV>(sh.update[w], graw, lane, R.update);
      }
      __syncthreads();
      if (it + 1 < c1 - c0) fetch(REV ? c - 1 : c + 1);
      if (have(c) > 0) {
        since *= whole;
        advance(sh, own, whole, g, r);
      }
      __syncthreads();
      // A segment ends: its state joins the start.
      if (REV ? c % a.seg == 0 : c % a.seg == a.seg - 1 || c == a.NC - 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int pb = 0; pb < 4; ++pb) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              start[nt][pb][q] = fmaf(since, start[nt][pb][q], own[nt][pb][q]);
            own[nt][pb] = f4{0.f, 0.f, 0.f, 0.f};
          }
        since = 1.f;
        // What the carries of a split run leave: the next segment's start state.
        const int next = c / a.seg + (REV ? -1 : 1);
        if (DOTS && seg < 0 && next >= 0 && next < a.NS) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pb = 0; pb < 4; ++pb)
              *reinterpret_cast<f4*>(slot(next) + ((nt * 4 + pb) * 64 * WAVES + t) * 4) =
                  start[nt][pb];
        }
      }
    }
    if (R.final.base && (REV ? c0 == 0 : c1 == a.NC)) {
      const int t = thread() & (64 * WAVES - 1), g = (t >> 4) & 3, r = t & 15;
      float* s = R.final.base + (long)bh * R.n * R.p;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pb = 0; pb < 4; ++pb)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = 64 * nt + 16 * w + 4 * g + q, p = col0 + 16 * pb + r;
            if (n < R.n && p < R.p)
              s[(long)n * R.final.sn + (long)p * R.final.sp] = start[nt][pb][q];
          }
    }
  }

  // The scores of the blocks ja and jb (the s-th pair from the strip) with their decays,
  // zeros where the queries do not look.  With dots, a token's score with itself is kept
  // out of them.
  template <bool DOTS, typename Sh>
  __device__ __forceinline__ void decayed(const Sh& sh, int s, int ja, int jb, int reached,
                                          float near, int g, int r, f4 (&acc)[2],
                                          float* diagonal) const {
    if (s == 0) {
      const float ph = sh.ph[w][16 * w + r], pl = sh.pl[w][16 * w + r];
      const f4 kh = *reinterpret_cast<const f4*>(&sh.ph[w][16 * w + 4 * g]);
      const f4 kl = *reinterpret_cast<const f4*>(&sh.pl[w][16 * w + 4 * g]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float gap = (ph - kh[q]) + (pl - kl[q]);
        const int ahead = REV ? 4 * g + q - r : r - 4 * g - q;  // query - key
        const float x = acc[0][q] * (__builtin_amdgcn_exp2f(REV ? -gap : gap) * R.intra);
        acc[0][q] = ahead > (DOTS ? 0 : -1) ? x : 0.f;
        if (DOTS && ahead == 0) *diagonal = x;
      }
    } else {
      acc[0] *= near * *reinterpret_cast<const f4*>(&sh.far[w][16 * ja + 4 * g]);
    }
    // A block past the last one seen gives no scores.
    const f4 far = near * *reinterpret_cast<const f4*>(&sh.far[w][16 * jb + 4 * g]);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[1][q] = 2 * s + 1 < reached ? acc[1][q] * far[q] : 0.f;
  }

  // Whether any output of the wave is not finite.
  __device__ __forceinline__ static bool unsound(const f4 (&out)[4]) {
    f4 x = out[0] * 0.f;
#pragma unroll
    for (int pb = 1; pb < 4; ++pb)
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = fmaf(out[pb][q], 0.f, x[q]);
    const float y = (x[0] + x[1]) + (x[2] + x[3]);
    return __any(y != y);
  }
  // Whether any of the chunk's values is (each lane looks at a token's).
  template <typename Sh>
  __device__ __forceinline__ static bool spoiled(const Sh& sh, int lane) {
    bool bad = false;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const u4 u = *reinterpret_cast<const u4*>(&sh.v[0][0][64 * lane + 8 * i]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        bad |= (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
    }
    return __any(bad);
  }

  // The outputs of the wave's strip once more, the same products in the same order, where
  // one of the chunk's values is not finite: it counts as zero, which keeps it from the
  // tokens that do not look back on it (a score of zero times NaN is NaN), and then
  // makes its column of the others' outputs NaN.  Few registers rather than fast: it
  // costs other calls up to 2% (T32768 H16 N128 P128 271 -> 278 us, B16 T1024 H12
  // forward and backward 233 -> 234).
  template <int SP, bool DOTS>
  __device__ __forceinline__ float attend_finite(const Shared<In, NT, SP>& sh, const Source& qs,
                                                 int c, const Reach& d, int g, int r,
                                                 f4 (&out)[4]) const {
    const int strip = opaque_strip(), reached = seen(strip), t = 16 * w + r;
    const Rsrc qr = chunk_rows(qs, c, have(c));
    auto query = [&](int kk) {
      return planes(load_piece(qr, t * qs.stride, 32 * kk + 8 * g, R.n, (const In*)nullptr));
    };
    auto apart = [] { asm volatile("" ::: "memory"); };
#pragma unroll
    for (int pb = 0; pb < 4; ++pb) out[pb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int kk = 0; kk < 2 * NT; ++kk) {
      const Frag<IN> qf = query(kk);
#pragma unroll
      for (int pb = 0; pb < 4; ++pb) {
        const Frag<SP> sf[1] = {rows<SP, NT>(sh.s, 16 * pb, kk, g, r)};
        mma(sf, qf, &out[pb]);
        apart();
      }
    }
    const float inter = R.inter * __shfl(d.inter, t);
    const float near = R.intra * __shfl(d.near, t);
#pragma unroll
    for (int pb = 0; pb < 4; ++pb) out[pb] *= inter;
    float diagonal = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (2 * s >= reached) continue;
      const int ja = block(strip, 2 * s), jb = block(strip, 2 * s + 1);
      f4 acc[2] = {f4{0.f, 0.f, 0.f, 0.f}, f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
      for (int kk = 0; kk < 2 * NT; ++kk) {
        const Frag<IN> qf = query(kk);
        const Frag<IN> kf[2] = {rows<IN, NT>(sh.k, 16 * ja, kk, g, r),
                                rows<IN, NT>(sh.k, 16 * jb, kk, g, r)};
        mma(kf, qf, acc);
      }
      decayed<DOTS>(sh, s, ja, jb, reached, near, g, r, acc, &diagonal);
      const float x[8] = {acc[0][0], acc[0][1], acc[0][2], acc[0][3],
                          acc[1][0], acc[1][1], acc[1][2], acc[1][3]};
      const Frag<SP> score = split8<SP>(x);
#pragma unroll
      for (int pb = 0; pb < 4; ++pb) {
        const Frag<IN> vf[1] = {finite(columns<IN, 1>(sh.v, 0, ja, jb, pb, g, r))};
        mma(vf, score, &out[pb]);
        apart();
      }
    }
#pragma unroll 1
    for (int j = 0; j < C; ++j) {
      const int ahead = REV ? j - t : t - j;
#pragma unroll
      for (int pb = 0; pb < 4; ++pb) {
        const u2 u = *reinterpret_cast<const u2*>(
            &sh.v[0][0][unit(j, 2 * pb + (g >> 1)) + 4 * (g & 1)]);
        const f4 v{low(u[0]), high(u[0]), low(u[1]), high(u[1])};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float x = v[q] * 0.f;
          if (ahead > (DOTS ? 0 : -1) && x != x) out[pb][q] = x;
        }
      }
    }
    return diagonal;
  }

  template <int SP, bool DOTS>
  __device__ __forceinline__ void write_outputs(int c0, int c1, Shared<In, NT, SP>& sh) {
    const Source vs = source<In>(R.v, b, h), qs = source<In>(R.q, b, h);
    Piece<In> vraw[2], qraw[2 * NT];
    float graw;
    auto fetch = [&](int c) {
      const int t = thread(), lane = t & 63;
      fetch_v(vraw, vs, c, t);
      const Rsrc qr = chunk_rows(qs, c, have(c));
#pragma unroll
      for (int kk = 0; kk < 2 * NT; ++kk)
        qraw[kk] = load_piece(qr, (16 * w + (lane & 15)) * qs.stride,
                                     32 * kk + 8 * (lane >> 4), R.n, (const In*)nullptr);
      graw = decay(c, lane);
    };
    auto fetch_e = [&](Quad<In> (&e)[4], int c, int g, int r) {
      const Source es = source<In>(R.e, b, h);
      const Rsrc er = chunk_rows(es, c, have(c));
#pragma unroll
      for (int pb = 0; pb < 4; ++pb)
        e[pb] = load_quad(er, (16 * w + r) * es.stride, col0 + 16 * pb + 4 * g, R.p,
                          (const In*)nullptr);
    };
    fetch(REV ? c1 - 1 : c0);
    Reach d{};
    int known = -1;
    for (int it = 0; it < c1 - c0; ++it) {
      const int c = REV ? c1 - 1 - it : c0 + it, t0 = c * C;
      const int tid = thread(), lane = tid & 63, g = lane >> 4, r = lane & 15;
      Frag<IN> qf[2 * NT];
      Quad<In> e[4];
      if (have(c) > 0) {
        stage_v(sh, vraw, tid);
#pragma unroll
        for (int kk = 0; kk < 2 * NT; ++kk) qf[kk] = planes(qraw[kk]);
        if (unknown(c, &known)) d = reach<REV>(sh.ph[w], sh.pl[w], sh.far[w], graw, lane, w);
        // Before the next chunk's loads, so that their wait does not include those.
        if constexpr (DOTS) fetch_e(e, c, g, r);
      }
      __syncthreads();
      if (it + 1 < c1 - c0) fetch(REV ? c - 1 : c + 1);
      if (have(c) > 0) {
        const int strip = opaque_strip(), reached = seen(strip);
        // The state's part, transposed: columns 16 pb + 4 g + q of token 16 w + r.
        f4 out[4];
#pragma unroll
        for (int pb = 0; pb < 4; ++pb) out[pb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 2 * NT; ++kk)
#pragma unroll
          for (int p0 = 0; p0 < 4; p0 += GROUP) {
            Frag<SP> sf[GROUP];
#pragma unroll
            for (int pb = 0; pb < GROUP; ++pb)
              sf[pb] = rows<SP, NT>(sh.s, 16 * (p0 + pb), kk, g, r);
            mma(sf, qf[kk], &out[p0]);
          }
        const float inter = R.inter * __shfl(d.inter, 16 * w + r);
        const float near = R.intra * __shfl(d.near, 16 * w + r);
#pragma unroll
        for (int pb = 0; pb < 4; ++pb) out[pb] *= inter;
        float diagonal = 0.f;  // with dots: a token's score with itself, kept out of score
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (2 * s >= reached) continue;
          const int ja = block(strip, 2 * s), jb = block(strip, 2 * s + 1);
          // Scores, transposed: keys 16 ja (jb) + 4 g + q of query 16 w + r.
          f4 acc[2] = {f4{0.f, 0.f, 0.f, 0.f}, f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int kk = 0; kk < 2 * NT; ++kk) {
            const Frag<IN> kf[2] = {rows<IN, NT>(sh.k, 16 * ja, kk, g, r),
                                    rows<IN, NT>(sh.k, 16 * jb, kk, g, r)};
            mma(kf, qf[kk], acc);
          }
          decayed<DOTS>(sh, s, ja, jb, reached, near, g, r, acc, &diagonal);
          const float x[8] = {acc[0][0], acc[0][1], acc[0][2], acc[0][3],
                              acc[1][0], acc[1][1], acc[1][2], acc[1][3]};
          const Frag<SP> score = split8<SP>(x);
#pragma unroll
          for (int p0 = 0; p0 < 4; p0 += GROUP) {
            Frag<IN> vf[GROUP];
#pragma unroll
            for (int pb = 0; pb < GROUP; ++pb)
              vf[pb] = columns<IN, 1>(sh.v, 0, ja, jb, p0 + pb, g, r);
            mma(vf, score, &out[p0]);
          }
        }
        if (__builtin_expect(unsound(out), 0) && spoiled(sh, lane)) {
          // (What is on its way is fetched again afterwards, so that it takes no registers.)
          diagonal = attend_finite<SP, DOTS>(sh, qs, c, d, g, r, out);
          if constexpr (DOTS) fetch_e(e, c, g, r);
          if (it + 1 < c1 - c0) fetch(REV ? c - 1 : c + 1);
        }
        const int t = 16 * w + r;
        if constexpr (DOTS) {
          float dot = 0.f;
#pragma unroll
          for (int pb = 0; pb < 4; ++pb)
#pragma unroll
            for (int q = 0; q < 4; ++q) dot = fmaf(out[pb][q], e[pb].get()[q], dot);
          dot = sum_groups(dot);
          if (g == 0 && t < have(c))
            R.dots[((long)(tile * a.B + b) * a.H + h) * a.T + t0 + t] = dot;
          // The token's own term, which the dots leave out.
          const float own_score = sum_groups(diagonal);
#pragma unroll
          for (int pb = 0; pb < 4; ++pb)
#pragma unroll
            for (int i = IN - 1; i >= 0; --i) {
              const u2 u = *reinterpret_cast<const u2*>(
                  &sh.v[i][0][unit(t, 2 * pb + (g >> 1)) + 4 * (g & 1)]);
              out[pb] += own_score * f4{low(u[0]), high(u[0]), low(u[1]), high(u[1])};
            }
        }
        if (t0 + t < a.T) store(out, t0 + t, t < have(c), g);
      } else {
        // Past the row's length: zeros.
        const f4 zero[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t0 + 16 * i + r < a.T && (i & 3) == w) store(zero, t0 + 16 * i + r, false, g);
      }
      __syncthreads();
    }
  }

  // A token's output, columns 16 pb + 4 g + q; zeros past the row's length.
  __device__ __forceinline__ void store(const f4 (&out)[4], int t, bool here, int g) {
    const long at = (((long)b * a.T + t) * a.H + h) * R.p + col0 + 4 * g;
    const int left = R.p - col0 - 4 * g;
    const f4 zero{0.f, 0.f, 0.f, 0.f};
    if (R.p & 3) {
#pragma unroll
      for (int pb = 0; pb < 4; ++pb)
        store_some(R.out, at + 16 * pb, here ? out[pb] : zero, left - 16 * pb, R.out_f32);
    } else if (R.out_f32) {
      float* p = static_cast<float*>(R.out) + at;
#pragma unroll
      for (int pb = 0; pb < 4; ++pb)
        if (16 * pb < left) *reinterpret_cast<f4*>(p + 16 * pb) = here ? out[pb] : zero;
    } else {
      bf16_t* p = static_cast<bf16_t*>(R.out) + at;
#pragma unroll
      for (int pb = 0; pb < 4; ++pb)
        if (16 * pb < left)
          *reinterpret_cast<u2*>(p + 16 * pb) =
              here ? u2{pack(out[pb][0], out[pb][1]), pack(out[pb][2], out[pb][3])} : u2{0u, 0u};
    }
  }
};

// Blocks of one (b, h) (its roles' tiles) differ by 8 in the grid: with
// consecutive blocks on the 8 XCDs in turn they share an L2, and so the rows.
__device__ __forceinline__ bool block_of(const Args& a, int x, int* which, int* b, int* h) {
  const int group = x / (8 * a.blocks), rest = x - group * 8 * a.blocks;
  const int bh = group * 8 + (rest & 7);
  *which = rest >> 3;
  *b = bh / a.H;
  *h = bh - *b * a.H;
  return bh < a.B * a.H;
}

// A block's chunks: of one segment (blockIdx.y) in split runs, else all.
__device__ __forceinline__ int chunks_of(const Args& a, int* c0, int* c1) {
  const bool split = a.split;
  *c0 = split ? (int)blockIdx.y * a.seg : 0;
  *c1 = split ? min(a.NC, *c0 + a.seg) : a.NC;
  return split ? (int)blockIdx.y : -1;
}

// Eight waves a block: two blocks a compute unit need no more than 128 registers
// (float32 with wide keys: one block, by its LDS).  That costs spills: 8 registers a lane
// of bfloat16 with wide keys, 14 of float32 with narrow ones.  Bound by the issue of
// vector and matrix instructions, 64 and 20% of a busy unit's cycles: B16 T1024 H12 N64
// P128 bfloat16 62 us, its 151 MB 30 us.
constexpr int waves_per_simd(int bytes, int nt) { return bytes == 4 && nt == 2 ? 2 : 4; }

template <typename In, int NT>
__global__ __launch_bounds__(128 * WAVES, waves_per_simd(sizeof(In), NT)) void attention_kernel(
    Args a) {
  constexpr int SP = Type<In>::ROUGH;
  __shared__ Shared<In, NT, SP> sh;
  int which, b, h, c0, c1;
  if (!block_of(a, blockIdx.x, &which, &b, &h)) return;
  const int seg = chunks_of(a, &c0, &c1);
  Block<In, NT, false>(a, a.role[0], which, b, h).template outputs<SP, false>(seg, c0, c1,
                                                                                     sh);
}

// The gradients: dQ forward in time, dK and dV in reverse; NP and NN 64s of the
// value and key widths, DOTS with what the decays' gradient needs.  Bound as the
// forward (69 and 25%): B16 T1024 H12 N64 P128 bfloat16 175 us.  Float32 with narrow
// widths spills most, 113 registers a lane and 135 with DOTS, and its waves wait 61% of
// their cycles: B8 T1000 H8 N64 P64 53 us.
template <typename In, int NP, int NN, bool DOTS>
__global__ __launch_bounds__(128 * WAVES, waves_per_simd(sizeof(In), NP > NN ? NP : NN)) void
attention_backward_kernel(Args a) {
  constexpr int SP = DOTS ? FINE : Type<In>::ROUGH, SV = Type<In>::ROUGH;
  __shared__ union {
    Shared<In, NP, SP> p;
    Shared<In, NN, SV> n;
  } sh;
  int which, b, h, c0, c1;
  if (!block_of(a, blockIdx.x, &which, &b, &h)) return;
  const int seg = chunks_of(a, &c0, &c1);
  if (which < a.role[0].tiles)
    return Block<In, NP, false>(a, a.role[0], which, b, h)
        .template outputs<SP, DOTS>(seg, c0, c1, sh.p);
  which -= a.role[0].tiles;
  if (which < a.role[1].tiles)
    return Block<In, NP, true>(a, a.role[1], which, b, h)
        .template outputs<SP, DOTS>(seg, c0, c1, sh.p);
  Block<In, NN, true>(a, a.role[2], which - a.role[1].tiles, b, h)
      .template outputs<SV, false>(seg, c0, c1, sh.n);
}

// Split runs: the segments' own states, of all roles.  Bound by issue (VALU 74, MFMA 34%
// of the busy cycles): T32768 H16 N128 P128 bfloat16 with keys shared by four heads 76
// us, 402 MB of loads of 168 MB of rows.
template <typename In, int NT>
__global__ __launch_bounds__(64 * WAVES) void attention_states_kernel(Args a) {
  __shared__ Shared<In, NT, 0> sh;
  int which, b, h, i = 0, c0, c1;
  if (!block_of(a, blockIdx.x, &which, &b, &h)) return;
  while (which >= a.role[i].tiles) which -= a.role[i++].tiles;
  const Role& R = a.role[i];
  const int seg = chunks_of(a, &c0, &c1);
  if (seg == (R.rev ? 0 : a.NS - 1)) return;  // no segment starts from its end
  if constexpr (NT == 2) {
    if (R.n <= 64) {
      Shared<In, 1, 0>& narrow = reinterpret_cast<Shared<In, 1, 0>&>(sh);
      if (R.rev) return Block<In, 1, true>(a, R, which, b, h).states(seg, c0, c1, narrow);
      return Block<In, 1, false>(a, R, which, b, h).states(seg, c0, c1, narrow);
    }
  }
  if (R.rev) return Block<In, NT, true>(a, R, which, b, h).states(seg, c0, c1, sh);
  Block<In, NT, false>(a, R, which, b, h).states(seg, c0, c1, sh);
}

// Split runs: each segment's start state from the segments' own states and
// decays, in place (the last one's own was not formed, and is read for nothing).  Four
// state elements a thread.
__global__ void carry_kernel(Args a) {
  int which, b, h, i = 0;
  if (!block_of(a, blockIdx.x, &which, &b, &h)) return;
  while (which >= a.role[i].tiles) which -= a.role[i++].tiles;
  const Role& R = a.role[i];
  const int nts = R.n > 64 ? 2 : 1, part = blockIdx.y;  // part = (nt * 4 + pb)
  if (part >= 4 * nts) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, r = lane & 15;
  const int bh = b * a.H + h, nt = part >> 2, p = TILE * which + 16 * (part & 3) + r;
  f4 x{0.f, 0.f, 0.f, 0.f};
  if (R.initial.base) {
    const float* s = R.initial.base + (long)bh * R.n * R.p;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = 64 * nt + 16 * w + 4 * g + q;
      if (n < R.n && p < R.p) x[q] = s[(long)n * R.initial.sn + (long)p * R.initial.sp];
    }
  }
  const long first = (long)(which * a.B * a.H + bh) * a.NS;
  float* own = R.starts + first * (nts * 4096) + (part * 64 * WAVES + tid) * 4;
  const float* decays = R.decays + first;
  constexpr int AHEAD = 8;  // segments loaded together
  for (int s0 = 0; s0 < a.NS; s0 += AHEAD) {
    f4 l[AHEAD];
    float d[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int s = min(s0 + k, a.NS - 1), at = R.rev ? a.NS - 1 - s : s;
      l[k] = *reinterpret_cast<const f4*>(own + (long)at * (nts * 4096));
      d[k] = decays[at];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (s0 + k >= a.NS) break;
      const int at = R.rev ? a.NS - 1 - s0 - k : s0 + k;
      *reinterpret_cast<f4*>(own + (long)at * (nts * 4096)) = x;
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = fmaf(d[k], x[q], l[k][q]);
    }
  }
}

// d log_decay: one block per (b, h) and segment, from its last token to its
// first, sums in float64.  At the segment's end they start with <S, R>, from the states
// that the roles of dQ and dK have there (both [value][key]), at the sequence's end
// with that of the final state and its cotangent.
__global__ __launch_bounds__(GRAD_THREADS) void decay_grad_kernel(DecayGrad a) {
  constexpr int W = GRAD_THREADS / 64;
  __shared__ double part[W];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, seg = blockIdx.y;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const long bh = blockIdx.x, rows = (long)a.B * a.H, slab = rows * a.T;
  auto block_sum = [&](double x) {
    x = lane_double(wave_prefix(x), 63);
    __syncthreads();
    if (lane == 0) part[w] = x;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < W; ++i) s += part[i];
    return s;
  };
  double x = 0.0;
  if (seg + 1 < a.NS) {
    for (int tile = 0; tile < a.tiles; ++tile) {
      const long row = (tile * rows + bh) * a.NS;
      const f4* s = reinterpret_cast<const f4*>(a.starts_q + (row + seg + 1) * a.slot);
      const f4* r = reinterpret_cast<const f4*>(a.starts_k + (row + seg) * a.slot);
      for (int i = tid; i < a.slot / 4; i += GRAD_THREADS)
#pragma unroll
        for (int q = 0; q < 4; ++q) x += (double)s[i][q] * (double)r[i][q];
    }
  } else if (a.state) {
    const long count = (long)a.n * a.p;
    for (long i = tid; i < count; i += GRAD_THREADS)
      x += (double)a.state[bh * count + i] * (double)a.d_state[bh * count + i];
  }
  double carry = block_sum(x), sum = 0.0;
  const int first = seg * a.seg * C;
  for (int end = min(a.T, first + a.seg * C); end > first; end -= GRAD_THREADS) {
    // Thread i takes token end - 1 - i: a suffix sum is a prefix sum here.
    const int t = end - 1 - tid;
    x = 0.0;
    if (t >= first && t < length) {
      for (int i = 0; i < a.tiles; ++i)
        x += (double)a.dots_q[i * slab + bh * a.T + t] - (double)a.dots_k[i * slab + bh * a.T + t];
    }
    x = wave_prefix(x);
    const double all = lane_double(x, 63);
    __syncthreads();
    if (lane == 0) part[w] = all;
    __syncthreads();
    x += carry;
    for (int i = 0; i < W; ++i) {
      if (i < w) x += part[i];
      carry += part[i];
    }
    if (t >= first) {
      // No gradient past the length, nor where the decay is exactly zero.
      const float g = t < length ? a.g[b * a.gb + t * a.gt + h] : 0.f;
      if (t >= length || g < -2000.f) x = 0.0;
      if (a.d_g) a.d_g[((long)b * a.T + t) * a.H + h] = (float)x;
      sum += x;
    }
  }
  if (a.head) {
    sum = block_sum(sum);
    if (tid == 0) a.head[bh * a.NS + seg] = sum;
  }
}

// One block per head: the sums of its segments over the rows.
__global__ __launch_bounds__(64) void decay_heads_kernel(const double* head, int B, int H, int NS,
                                                         float* d_g) {
  const int h = blockIdx.x;
  double s = 0.0;
  for (long i = threadIdx.x; i < (long)B * NS; i += 64)
    s += head[(i / NS * H + h) * NS + i % NS];
  s = lane_double(wave_prefix(s), 63);
  if (threadIdx.x == 0) d_g[h] = (float)s;
}

// Gradients of shared heads: out[b,t,j,:] = sum over the heads h of group j
// of part[b,t,h,:], float32 rounded once.
template <typename Out>
__global__ void share_sum_kernel(const float* part, long tokens, int heads, int share, int width,
                                 Out* out) {
  const int own = heads / share;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < tokens * own * width;
       i += (long)gridDim.x * blockDim.x) {
    const int x = (int)(i % width);
    const long row = i / width;
    const long t = row / own;
    const int j = (int)(row - t * own);
    const float* p = part + ((t * heads) + (long)j * share) * width + x;
    float s = 0.f;
    for (int k = 0; k < share; ++k) s += p[(long)k * width];
    if constexpr (sizeof(Out) == 2)
      out[i] = (bf16_t)pack(s, 0.f);
    else
      out[i] = s;
  }
}

// Rows that are no whole 16-byte pieces (by width, stride or address), copied to
// padded ones; a thread writes one piece.  Bound by memory: 500 MB in 132 us at B16
// T1024 H12 N63 P127, forward and backward, whose attention then takes 310 us.  (Read
// an element at a time where they are used, such rows took 587 us.)
template <typename In>
__global__ __launch_bounds__(256) void pack_kernel(Pack a) {
  constexpr int V = 16 / sizeof(In);
  const int which = blockIdx.y, pieces = a.padded[which] / V, heads = a.heads[which];
  const Rows& x = a.from[which];
  const long count = (long)a.B * a.T * heads * pieces;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    const int piece = (int)(i % pieces);
    const long row = i / pieces, token = row / heads;
    const int h = (int)(row - token * heads), b = (int)(token / a.T), t = (int)(token % a.T);
    const In* from = static_cast<const In*>(x.base) + b * x.sb + t * x.st + h * x.sh + piece * V;
    typedef In piece_t __attribute__((ext_vector_type(V)));
    piece_t v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = piece * V + e < x.width ? from[e] : (In)0;
    *reinterpret_cast<piece_t*>(static_cast<In*>(a.to[which]) + i * V) = v;
  }
}

// One token: S' = e^g S + k v^T, o = scale S'^T q.  The state is read and
// written once, which is all the time there is: a block takes one (b, h), its
// threads a piece of V columns of every R-th row each, and all of a thread's loads are
// issued (after those of q, k and v) before the first is used.  Bound by memory: B2048
// H8 N64 P64 86 us, 6.4 TB/s.
template <typename In>
__device__ __forceinline__ float load_one(const void* p, long i) {
  if constexpr (sizeof(In) == 2)
    return __uint_as_float((unsigned)static_cast<const bf16_t*>(p)[i] << 16);
  else
    return static_cast<const float*>(p)[i];
}

template <typename In, int V, int PASSES>
__global__ __launch_bounds__(STEP_THREADS) void step_kernel(Step a) {
  typedef float piece __attribute__((ext_vector_type(V)));
  __shared__ float q[MAX_WIDTH], k[MAX_WIDTH], v[MAX_WIDTH], part[STEP_THREADS * V];
  const int tid = threadIdx.x, b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
  const bool on = !a.active || a.active[b];
  const long bh = blockIdx.x, at = bh * a.N * a.P;
  const float g = a.g[b * a.gb + h];
  float qx = 0.f, kx = 0.f, vx = 0.f;
  if (tid < a.N) {
    qx = load_one<In>(a.q, b * a.qb + (h / a.q_share) * a.qh + tid);
    kx = load_one<In>(a.k, b * a.kb + (h / a.k_share) * a.kh + tid);
  }
  if (tid < a.P) vx = load_one<In>(a.v, b * a.vb + (h / a.v_share) * a.vh + tid);
  // Thread (row, column) of the 2^span threads along a row.
  const int p = (tid & ((1 << a.span) - 1)) * V, row = tid >> a.span;
  const int step = STEP_THREADS >> a.span;
  piece s[PASSES];
  piece o(0.f);
  for (int n0 = 0; n0 < a.N; n0 += PASSES * step) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int n = n0 + i * step + row;
      s[i] = piece(0.f);
      if (n < a.N && p < a.P)
        s[i] = __builtin_nontemporal_load(
            reinterpret_cast<const piece*>(a.state + at + (long)n * a.P + p));
    }
    if (n0 == 0) {
      if (tid < a.N) q[tid] = qx, k[tid] = kx;
      if (tid < a.P) v[tid] = vx;
      __syncthreads();
    }
    const float lam = expf(g);
    if (p < a.P) {
      piece vp;
#pragma unroll
      for (int c = 0; c < V; ++c) vp[c] = v[p + c];
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int n = n0 + i * step + row;
        if (n >= a.N) continue;
        const float kn = k[n], qn = q[n];
        piece x = s[i];
        if (on) {
#pragma unroll
          for (int c = 0; c < V; ++c) x[c] = fmaf(lam, s[i][c], kn * vp[c]);
        }
        if (on || a.new_state != a.state)
          __builtin_nontemporal_store(
              x, reinterpret_cast<piece*>(a.new_state + at + (long)n * a.P + p));
#pragma unroll
        for (int c = 0; c < V; ++c) o[c] = fmaf(qn, x[c], o[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < V; ++c) part[tid * V + c] = o[c];
  __syncthreads();
  if (tid < a.P) {
    float x = 0.f;
    for (int r = 0; r < step; ++r) x += part[(r << a.span) * V + tid];
    x = on ? a.scale * x : 0.f;
    if constexpr (sizeof(In) == 2)
      static_cast<bf16_t*>(a.out)[bh * a.P + tid] = (bf16_t)pack(x, 0.f);
    else
      static_cast<float*>(a.out)[bh * a.P + tid] = x;
  }
}

#define LA_INSTANCES(In)                                                       \
  template __global__ void attention_kernel<In, 1>(Args);                      \
  template __global__ void attention_kernel<In, 2>(Args);                      \
  template __global__ void attention_states_kernel<In, 1>(Args);               \
  template __global__ void attention_states_kernel<In, 2>(Args);               \
  template __global__ void attention_backward_kernel<In, 1, 1, false>(Args);   \
  template __global__ void attention_backward_kernel<In, 1, 1, true>(Args);    \
  template __global__ void attention_backward_kernel<In, 1, 2, false>(Args);   \
  template __global__ void attention_backward_kernel<In, 1, 2, true>(Args);    \
  template __global__ void attention_backward_kernel<In, 2, 1, false>(Args);   \
  template __global__ void attention_backward_kernel<In, 2, 1, true>(Args);    \
  template __global__ void attention_backward_kernel<In, 2, 2, false>(Args);   \
  template __global__ void attention_backward_kernel<In, 2, 2, true>(Args);    \
  template __global__ void step_kernel<In, 4, 4>(Step);                        \
  template __global__ void step_kernel<In, 4, 8>(Step);                        \
  template __global__ void step_kernel<In, 4, 16>(Step);                       \
  template __global__ void step_kernel<In, 1, 16>(Step);                       \
  template __global__ void pack_kernel<In>(Pack);                              \
  template __global__ void share_sum_kernel<In>(const float*, long, int, int, int, In*);
LA_INSTANCES(float)
LA_INSTANCES(bf16_t)
#undef LA_INSTANCES

}  // namespace la

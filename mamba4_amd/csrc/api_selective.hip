// C ABI of the selective layer's operators (include/mamba4_selective.h): the checks
// of the arguments and the launches.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <initializer_list>

#include "../../include/mamba4_selective.h"
#include "api_common.hpp"
#include "conv.hpp"
#include "rms.hpp"
#include "selscan.hpp"

namespace ss {
template <typename In, int NG, bool OUT, bool WHOLE>
__global__ void scan_kernel(Scan);
template <typename In, int NG, bool ALL, bool WHOLE>
__global__ void scan_backward_kernel(Scan);
template <bool BWD>
__global__ void carry_kernel(Scan);
template <typename In>
__global__ void join_kernel(Join);
template <typename In, int ROWS>
__global__ void step_kernel(Step);
}  // namespace ss

namespace cv {
template <typename In, int V, int W>
__global__ void conv_kernel(Conv);
template <typename In, int V, int W>
__global__ void conv_backward_kernel(Conv);
template <typename In, int V, int W, int ROWS>
__global__ void conv_step_kernel(Step);
__global__ void conv_join_kernel(const float*, int, int, int, float*, float*);
}  // namespace cv

namespace rn {
template <typename X, typename R, int V, int IT, bool E4M3>
__global__ void rms_kernel(Rms);
template <typename X, typename R, int V, int IT>
__global__ void rms_backward_kernel(Rms);
__global__ void rms_join_kernel(const float*, int, int, float*);
}  // namespace rn

namespace {

using m4::align256;
using m4::api_fail;
using m4::api_launch;
using m4::bad_workspace;
using m4::Carver;

// Whether a launch of `blocks` of `threads` is more than it takes: 2^32 threads.
bool too_many(double blocks, int threads) { return blocks * threads >= 4294967296.0; }

// Blocks of 256 threads that take an element each in turn.
unsigned element_blocks(long count) {
  return (unsigned)std::min<long>((count + 255) / 256, 1 << 16);
}

bool misaligned(int bf16, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % (bf16 ? 2 : 4)) return true;
  return false;
}

// Whether pieces of four elements at these addresses are aligned to their size.
bool whole_at(int bf16, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % (bf16 ? 8 : 16)) return false;
  return true;
}

// Threads that keep the card busy.
long busy_threads() { return 768L * m4::api_compute_units(); }

// ---------------------------------------------------------- selective scan --

int tiles_of(int T) { return (T + ss::TILE - 1) / ss::TILE; }

// Groups of 16 states that a lane holds four of.
int groups_of(int N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }

int blocks_of(const m4sl_scan& s) {
  return (s.D / s.G + ss::BLOCK_CHANNELS - 1) / ss::BLOCK_CHANNELS;
}

// `tokens`: whether the call has a time axis.
bool bad_scan(const m4sl_scan* s, bool tokens, std::string* why) {
  if (!s) {
    *why = "a required pointer is NULL";
    return true;
  }
  if (s->B <= 0 || (tokens && s->T <= 0) || s->D <= 0) {
    *why = "B, T and D must be positive";
    return true;
  }
  if (s->G <= 0 || s->D % s->G) {
    *why = "G must divide D";
    return true;
  }
  if (s->N <= 0 || s->N > M4SL_MAX_STATES) {
    *why = "the states must be in 1.." + std::to_string(M4SL_MAX_STATES);
    return true;
  }
  if (too_many((double)s->B * s->G * blocks_of(*s), 64 * ss::WAVES) ||
      (tokens && s->T > INT_MAX - (1 << 16)) || (double)s->D * (s->N + 2) > 1e9) {
    *why = "problem too large";
    return true;
  }
  if (!s->x.data || !s->delta.data || !s->b.data || !s->c.data || !s->a) {
    *why = "a required pointer is NULL";
    return true;
  }
  if (misaligned(s->bf16, {s->x.data, s->delta.data, s->gate.data, s->b.data, s->c.data})) {
    *why = "rows must be aligned to their elements";
    return true;
  }
  return false;
}

// Microseconds a tile of a SIMD with `waves` waves: of the results, or of what a segment
// adds.  A wave alone takes the latency of its instructions, several the throughput
// (bfloat16, N16: T32768 D2048, 3 waves a SIMD 3.9 and 2.8, 8 waves 9.6 and 7.1; B16 T1024
// D1536, 2 waves, 2.7).  The backward keeps two waves a SIMD and takes more in turn (two
// 7.4; what a segment adds, 5 waves, 5.4).
double tile_pace(double waves, bool backward, bool results) {
  if (!results) return (backward ? 1.0 : 0.86) * (std::max(2.0, waves) + 0.3);
  if (!backward) return 1.16 * (std::max(2.0, waves) + 0.35);
  const double pairs = std::floor(waves / 2), rest = waves - 2 * pairs;
  return 7.4 * pairs + (rest <= 0 ? 0.0 : rest <= 1 ? 5.5 : 7.4);
}

// Most tiles of a segment whose rows stay, with two tiles more, below 2^31 bytes (as they
// have to where they are read through descriptors).
int most_tiles(const m4sl_scan& s) {
  long widest = s.D;
  for (const m4sl_rows* r : {&s.x, &s.delta, &s.gate, &s.b, &s.c})
    if (r->data) widest = std::max(widest, r->token_stride);
  return (int)(INT_MAX / 4 / ss::TILE / widest) - 2;
}

// Tiles of the segments that a sequence is cut into.  A walk from end to end leaves SIMDs
// idle where there are few sequences; segments cost their states first, a carry and two
// launches.  Of the cuts that fill every SIMD with 1, 2, ... waves the best by the paces
// above (B16 T1024 D1536: the forward walks, the backward takes four segments, 636 -> 606 us
// together; B1 T2000: 21 segments, 41 us for 46 with 63; T32768 D2048: 64, 446 us for 490
// with 24).  M4SL_SEGMENTS = a number overrides the choice; results differ by rounding.
int segment_tiles(const m4sl_scan& s, bool backward) {
  const int tiles = tiles_of(s.T);
  const long waves = (long)s.B * s.G * ((s.D / s.G + 15) / 16);
  const int least = (tiles + 59999) / 60000;  // (segments are a launch's y blocks)
  const int most = std::max(least, std::min(tiles, most_tiles(s)));
  if (const char* e = std::getenv("M4SL_SEGMENTS"))
    if (const int cut = std::atoi(e); cut > 0)
      return std::max(least, std::min(most, (int)((tiles + cut - 1L) / cut)));
  const long units = 4L * m4::api_compute_units();
  int best = most, each = 0;
  double time = 0;
  for (int fill = 0; fill <= 16; ++fill) {
    const long want = std::max(1L, fill * units / waves);
    const int size = (int)std::max<long>(least, std::min<long>(most, (tiles + want - 1) / want));
    if (size == each) continue;
    each = size;
    const int cut = (tiles + each - 1) / each;
    const double all = std::ceil(waves * (double)cut / units),
                 some = std::ceil(waves * (cut - 1.0) / units);
    double t = each * tile_pace(all, backward, true);
    if (cut > 1) t += 14.0 + 0.15 * cut + each * tile_pace(some, backward, false);
    if (fill == 0 || t < 0.99 * time) {
      best = each;
      time = t;
    }
  }
  return best;
}

ss::Rows rows_of(const m4sl_rows& r) { return ss::Rows{r.data, r.batch_stride, r.token_stride}; }

// Whether rows of `width` can be read through a segment's descriptor: aligned pieces of
// four, tokens at least a row apart, and a segment and two tiles more below 2^31 bytes.
bool tile_rows(const ss::Rows& r, int width, int seg, int bf16) {
  return width % 4 == 0 && r.batch % 4 == 0 && r.token % 4 == 0 && whole_at(bf16, {r.p}) &&
         r.token >= width && r.token <= INT_MAX / 4 / (seg + 2L * ss::TILE);
}

// Whether all rows are such (the kernels read others an element at a time).
bool whole_scan(const ss::Scan& a, int bf16, std::initializer_list<const void*> results) {
  const ss::Rows dense{nullptr, 0, a.D};
  return a.Dg % 4 == 0 && a.bg % 4 == 0 && a.cg % 4 == 0 && whole_at(bf16, results) &&
         tile_rows(dense, a.D, a.seg, bf16) && tile_rows(a.x, a.D, a.seg, bf16) &&
         tile_rows(a.delta, a.D, a.seg, bf16) && tile_rows(a.gate, a.D, a.seg, bf16) &&
         tile_rows(a.b, a.N, a.seg, bf16) && tile_rows(a.c, a.N, a.seg, bf16);
}

// Bytes that a forward's segments may read of those before them to start by themselves,
// instead of from a launch that carries the states (B1 T2000 D1536, 21 segments, 20 MB: 37
// us for 40; B1 T8000, 43 MB, the same; the backward of B16 T1024 607 us for 602).
constexpr double FOLDED_BYTES = 32e6;

ss::Scan scan_of(const m4sl_scan& s, const int* lengths, bool backward) {
  ss::Scan a{};
  a.x = rows_of(s.x);
  a.delta = rows_of(s.delta);
  a.gate = rows_of(s.gate.data ? s.gate : s.x);
  a.gated = s.gate.data != nullptr;
  a.b = rows_of(s.b);
  a.c = rows_of(s.c);
  a.bg = s.b_group_stride;
  a.cg = s.c_group_stride;
  if (s.T == 1) {  // (Strides of one token are no strides.)
    a.x.token = a.delta.token = a.gate.token = s.D;
    a.b.token = a.c.token = s.N;
  }
  a.a = s.a;
  a.skip = s.skip;
  a.bias = s.delta_bias;
  a.lengths = lengths;
  a.B = s.B;
  a.T = s.T;
  a.D = s.D;
  a.G = s.G;
  a.Dg = s.D / s.G;
  a.N = s.N;
  a.softplus = s.softplus;
  a.blocks = blocks_of(s);
  a.seg = segment_tiles(s, backward) * ss::TILE;
  a.NS = (s.T + a.seg - 1) / a.seg;
  const double read = 0.5 * a.NS * (a.NS - 1.0) * s.B * s.D * s.N * sizeof(float);
  a.folded = !backward && a.NS > 1 && read <= FOLDED_BYTES;
  return a;
}

size_t take_segments(Carver& c, ss::Scan* a) {
  const size_t rows = a->NS > 1 ? (size_t)a->B * a->NS : 0;
  a->ends = c.take<float>(rows * a->D * a->N);
  a->sums = c.take<float>(rows * a->D);
  return c.used;
}

size_t take_backward(Carver& c, ss::Scan* a) {
  take_segments(c, a);
  const size_t rows = (size_t)a->B * a->NS;
  a->part_bc = c.take<float>((size_t)a->blocks * a->B * a->T * a->G * 2 * a->N);
  a->part_a = c.take<float>(rows * a->D * a->N);
  a->part_d = c.take<float>(rows * 2 * a->D);
  return c.used;
}

template <typename In, int NG, bool WHOLE>
void start_groups(const ss::Scan& a, bool backward, bool all, hipStream_t st) {
  // (What a sequence's last segment adds, backward the first one's, nobody starts from.)
  const dim3 grid(a.B * a.G * a.blocks, all ? a.NS : a.NS - 1), block(64 * ss::WAVES);
  if (backward) {
    if (all)
      hipLaunchKernelGGL((ss::scan_backward_kernel<In, NG, true, WHOLE>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((ss::scan_backward_kernel<In, NG, false, WHOLE>), grid, block, 0, st, a);
  } else {
    if (all)
      hipLaunchKernelGGL((ss::scan_kernel<In, NG, true, WHOLE>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((ss::scan_kernel<In, NG, false, WHOLE>), grid, block, 0, st, a);
  }
}

template <typename In, bool WHOLE>
void start_states(const ss::Scan& a, bool backward, bool all, hipStream_t st) {
  if (groups_of(a.N) == 1) return start_groups<In, 1, WHOLE>(a, backward, all, st);
  if (groups_of(a.N) == 2) return start_groups<In, 2, WHOLE>(a, backward, all, st);
  return start_groups<In, 4, WHOLE>(a, backward, all, st);
}

// `all`: the results; else what the segments add.
int run_scan(const char* name, const ss::Scan& a, int bf16, bool whole, bool backward, bool all,
             hipStream_t st) {
  return api_launch(name, st, [&] {
    if (bf16)
      whole ? start_states<ss::bf16_t, true>(a, backward, all, st)
            : start_states<ss::bf16_t, false>(a, backward, all, st);
    else
      whole ? start_states<float, true>(a, backward, all, st)
            : start_states<float, false>(a, backward, all, st);
  });
}

template <bool BWD>
int run_carry(const ss::Scan& a, hipStream_t st) {
  const unsigned blocks = element_blocks((long)a.B * a.D * a.N);
  return api_launch(BWD ? "scan_backward_carry" : "scan_carry", st, [&] {
    hipLaunchKernelGGL(ss::carry_kernel<BWD>, dim3(blocks), dim3(256), 0, st, a);
  });
}

template <typename In>
void start_step(const ss::Step& a, int rows, unsigned blocks, hipStream_t st) {
  const dim3 grid(blocks), block(ss::STEP_THREADS);
  if (rows == 4)
    hipLaunchKernelGGL((ss::step_kernel<In, 4>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ss::step_kernel<In, 1>), grid, block, 0, st, a);
}

}  // namespace

extern "C" {

long m4sl_scan_kept_floats(const m4sl_scan* s) {
  std::string why;
  if (bad_scan(s, true, &why)) return 0;
  return (long)s->B * tiles_of(s->T) * (ss::TILE / ss::kept_tokens(groups_of(s->N))) * s->D * s->N;
}

size_t m4sl_scan_workspace_bytes(const m4sl_scan* s) {
  std::string why;
  if (bad_scan(s, true, &why)) return 0;
  ss::Scan a = scan_of(*s, nullptr, false);
  Carver c{nullptr};
  return take_segments(c, &a);
}

int m4sl_scan_forward(const m4sl_scan* s, const float* initial, const int* lengths, void* output,
                      float* state, float* kept, void* workspace, size_t workspace_bytes,
                      void* stream) {
  const char* name = "m4sl_scan_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_scan(s, true, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!output || !state) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(s->bf16, {output}))
      return api_fail(M4MR_EINVAL, at + "rows must be aligned to their elements");
    ss::Scan a = scan_of(*s, lengths, false);
    Carver c{static_cast<char*>(workspace)};
    if (bad_workspace(workspace, workspace_bytes, take_segments(c, &a), &why))
      return api_fail(M4MR_EINVAL, at + why);
    const bool whole = whole_scan(a, s->bf16, {output});
    a.initial = initial;
    a.out = output;
    a.state = state;
    a.kept = kept;
    a.whole_n = a.N % 4 == 0 && whole_at(0, {a.a, initial, state, kept});
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.NS > 1) {
      int rc = run_scan("scan_states", a, s->bf16, whole, false, false, st);
      if (!rc && !a.folded) rc = run_carry<false>(a, st);
      if (rc) return rc;
    }
    return run_scan("scan", a, s->bf16, whole, false, true, st);
  });
}

size_t m4sl_scan_backward_workspace_bytes(const m4sl_scan* s) {
  std::string why;
  if (bad_scan(s, true, &why)) return 0;
  ss::Scan a = scan_of(*s, nullptr, true);
  Carver c{nullptr};
  return take_backward(c, &a);
}

int m4sl_scan_backward(const m4sl_scan* s, const int* lengths, const void* d_output,
                       const float* d_state, const float* kept, const m4sl_scan_grads* grads,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4sl_scan_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_scan(s, true, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!d_output || !kept || !grads || !grads->x || !grads->delta || !grads->b || !grads->c)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(s->bf16, {d_output, grads->x, grads->delta, grads->gate, grads->b, grads->c}))
      return api_fail(M4MR_EINVAL, at + "rows must be aligned to their elements");
    ss::Scan a = scan_of(*s, lengths, true);
    Carver c{static_cast<char*>(workspace)};
    if (bad_workspace(workspace, workspace_bytes, take_backward(c, &a), &why))
      return api_fail(M4MR_EINVAL, at + why);
    const bool whole =
        whole_scan(a, s->bf16, {d_output, grads->x, grads->delta, grads->gate});
    a.dout = d_output;
    a.dstate = d_state;
    a.kept = const_cast<float*>(kept);
    a.dx = grads->x;
    a.ddelta = grads->delta;
    a.dgate = s->gate.data ? grads->gate : nullptr;
    a.dinitial = grads->initial;
    a.whole_n = a.N % 4 == 0 && whole_at(0, {a.a, d_state, kept, a.dinitial});
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc;
    if (a.NS > 1) {
      a.skipped = 1;
      rc = run_scan("scan_backward_states", a, s->bf16, whole, true, false, st);
      a.skipped = 0;
      if (!rc) rc = run_carry<true>(a, st);
      if (rc) return rc;
    }
    rc = run_scan("scan_backward", a, s->bf16, whole, true, true, st);
    if (rc) return rc;
    ss::Join j{};
    j.part_bc = a.part_bc;
    j.part_a = a.part_a;
    j.part_d = a.part_d;
    j.bc_blocks = element_blocks((long)a.B * a.T * a.G * a.N);
    j.blocks = a.blocks;
    j.rows = (long)a.B * a.NS;
    j.B = a.B;
    j.T = a.T;
    j.D = a.D;
    j.G = a.G;
    j.N = a.N;
    j.lengths = lengths;
    j.db = grads->b;
    j.dc = grads->c;
    j.da = grads->a;
    j.dskip = s->skip ? grads->skip : nullptr;
    j.dbias = s->delta_bias ? grads->delta_bias : nullptr;
    const bool sums = j.da || j.dskip || j.dbias;
    const long columns = sums ? (long)a.D * (a.N + 2) : 0;
    return api_launch("scan_join", st, [&] {
      const dim3 grid(j.bc_blocks + (unsigned)((columns + 63) / 64)), block(256);
      if (s->bf16)
        hipLaunchKernelGGL(ss::join_kernel<ss::bf16_t>, grid, block, 0, st, j);
      else
        hipLaunchKernelGGL(ss::join_kernel<float>, grid, block, 0, st, j);
    });
  });
}

int m4sl_scan_step(const m4sl_scan* s, const uint8_t* active, const float* state,
                   float* new_state, void* output, void* stream) {
  const char* name = "m4sl_scan_step";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_scan(s, false, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!state || !new_state || !output)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(s->bf16, {output}))
      return api_fail(M4MR_EINVAL, at + "rows must be aligned to their elements");
    ss::Step a{};
    a.x = rows_of(s->x);
    a.delta = rows_of(s->delta);
    a.gate = rows_of(s->gate);
    a.b = rows_of(s->b);
    a.c = rows_of(s->c);
    a.bg = s->b_group_stride;
    a.cg = s->c_group_stride;
    a.a = s->a;
    a.skip = s->skip;
    a.bias = s->delta_bias;
    a.active = active;
    a.state = state;
    a.new_state = new_state;
    a.out = output;
    a.B = s->B;
    a.D = s->D;
    a.Dg = s->D / s->G;
    a.N = s->N;
    a.softplus = s->softplus;
    a.whole_n = a.N % 4 == 0 && whole_at(0, {a.a, state, new_state});
    a.whole_bc = s->N % 4 == 0 && a.b.batch % 4 == 0 && a.c.batch % 4 == 0 && a.bg % 4 == 0 &&
                 a.cg % 4 == 0 && whole_at(s->bf16, {a.b.p, a.c.p});
    while (4 << a.span < s->N) ++a.span;
    const long lanes = (long)s->D << a.span;
    // Four rows a thread, where that leaves the card busy.
    const int rows = lanes * s->B >= 4 * busy_threads() ? 4 : 1;
    a.blocks = (int)((lanes + ss::STEP_THREADS - 1) / ss::STEP_THREADS);
    const double blocks = (double)a.blocks * ((s->B + rows - 1) / rows);
    if (too_many(blocks, ss::STEP_THREADS))
      return api_fail(M4MR_EINVAL, at + "problem too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return api_launch("scan_step", st, [&] {
      if (s->bf16)
        start_step<ss::bf16_t>(a, rows, (unsigned)blocks, st);
      else
        start_step<float>(a, rows, (unsigned)blocks, st);
    });
  });
}

}  // extern "C"

// ------------------------------------------------------ causal convolution --

namespace {

bool bad_conv(const m4sl_rows* x, const float* weight, int B, int T, int D, int W, int activation,
              std::string* why) {
  if (B <= 0 || T <= 0 || D <= 0) {
    *why = "B, T and D must be positive";
    return true;
  }
  if (W <= 0 || W > M4SL_MAX_TAPS) {
    *why = "the taps must be in 1.." + std::to_string(M4SL_MAX_TAPS);
    return true;
  }
  if (activation != M4SL_NONE && activation != M4SL_SILU) {
    *why = "unknown activation";
    return true;
  }
  if (T > INT_MAX - (1 << 16) || D > INT_MAX - (1 << 16) || (double)B * T * D > 1e15) {
    *why = "problem too large";
    return true;
  }
  if (!x || !x->data || !weight) {
    *why = "a required pointer is NULL";
    return true;
  }
  return false;
}

// Whether all rows consist of aligned pieces of `vec` channels, and the parameters
// (float32) are aligned to pieces of four.
bool conv_pieces(int vec, const m4sl_rows& x, int T, int D, int bf16, const float* weight,
                 const float* bias, std::initializer_list<const void*> arrays) {
  const int bytes = vec * (bf16 ? 2 : 4);
  bool whole = D % vec == 0 && x.batch_stride % vec == 0 && (T == 1 || x.token_stride % vec == 0) &&
               reinterpret_cast<uintptr_t>(x.data) % bytes == 0 && whole_at(0, {weight, bias});
  for (const void* p : arrays) whole = whole && reinterpret_cast<uintptr_t>(p) % bytes == 0;
  return whole;
}

// Channels of a thread's piece: four if they can be.
int conv_vec(const m4sl_rows& x, int T, int D, int bf16, const float* weight, const float* bias,
             std::initializer_list<const void*> arrays) {
  return conv_pieces(4, x, T, D, bf16, weight, bias, arrays) ? 4 : 1;
}

// The backward's lines (runs of rows) and blocks.
struct ConvPlan {
  int run, runs, cols, wide, lines;
  unsigned rows, columns;  // blocks
};

// Runs are as short as a busy card needs: the W - 1 rows at an edge are read twice.
ConvPlan conv_plan(int B, int T, int D, int W, int vec) {
  ConvPlan p{};
  p.cols = D / vec;
  p.wide = 1;
  while (p.wide < 64 && p.wide < p.cols) p.wide *= 2;
  p.lines = cv::THREADS / p.wide;
  p.columns = (unsigned)((p.cols + p.wide - 1) / p.wide);
  const long each = (long)B * T * p.cols / busy_threads();
  const int fours = (int)std::min(16L, std::max(W > 4 ? 3L : 2L, (each + W + 2) / 4));
  p.run = 4 * fours - (W - 1);
  p.runs = (T + p.run - 1) / p.run;
  const long blocks = ((long)B * p.runs + p.lines - 1) / p.lines;
  const long most = std::max(1L, 4L * m4::api_compute_units() / p.columns);
  p.rows = (unsigned)std::min(blocks, most);
  return p;
}

template <typename In, int V, int W>
void start_conv(const cv::Conv& a, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((cv::conv_kernel<In, V, W>), grid, dim3(cv::THREADS), 0, st, a);
}
template <typename In, int V, int W>
void start_conv_backward(const cv::Conv& a, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((cv::conv_backward_kernel<In, V, W>), grid, dim3(cv::THREADS), 0, st, a);
}
template <typename In, int V, int W, int ROWS>
void start_conv_step(const cv::Step& a, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((cv::conv_step_kernel<In, V, W, ROWS>), grid, dim3(cv::THREADS), 0, st, a);
}

enum class Conv { FORWARD, BACKWARD, STEP, STEP_ROWS };
constexpr int STEP_ROWS = 4;

template <Conv WHAT, typename In, int V, int W, typename Args>
void start_one(const Args& a, dim3 grid, hipStream_t st) {
  if constexpr (WHAT == Conv::FORWARD) start_conv<In, V, W>(a, grid, st);
  else if constexpr (WHAT == Conv::BACKWARD) start_conv_backward<In, V, W>(a, grid, st);
  else start_conv_step<In, V, W, WHAT == Conv::STEP ? 1 : STEP_ROWS>(a, grid, st);
}

template <Conv WHAT, typename In, int V, typename Args>
void start_taps(const Args& a, int W, dim3 grid, hipStream_t st) {
  switch (W) {
    case 1: return start_one<WHAT, In, V, 1>(a, grid, st);
    case 2: return start_one<WHAT, In, V, 2>(a, grid, st);
    case 3: return start_one<WHAT, In, V, 3>(a, grid, st);
    case 4: return start_one<WHAT, In, V, 4>(a, grid, st);
    case 5: return start_one<WHAT, In, V, 5>(a, grid, st);
    case 6: return start_one<WHAT, In, V, 6>(a, grid, st);
    case 7: return start_one<WHAT, In, V, 7>(a, grid, st);
    default: return start_one<WHAT, In, V, 8>(a, grid, st);
  }
}

template <Conv WHAT, typename Args>
void start_width(const Args& a, int bf16, int vec, int W, dim3 grid, hipStream_t st) {
  if (bf16) {
    if constexpr (WHAT == Conv::FORWARD)
      if (vec == 8) return start_taps<WHAT, cv::bf16_t, 8>(a, W, grid, st);
    if (vec == 4) return start_taps<WHAT, cv::bf16_t, 4>(a, W, grid, st);
    return start_taps<WHAT, cv::bf16_t, 1>(a, W, grid, st);
  }
  if (vec == 4) return start_taps<WHAT, float, 4>(a, W, grid, st);
  return start_taps<WHAT, float, 1>(a, W, grid, st);
}

cv::Conv conv_of(const m4sl_rows& x, const float* weight, const float* bias, const void* initial,
                 const int* lengths, int B, int T, int D, int activation) {
  cv::Conv a{};
  a.x = x.data;
  a.xb = x.batch_stride;
  a.xt = x.token_stride;
  a.weight = weight;
  a.bias = bias;
  a.initial = initial;
  a.lengths = lengths;
  a.B = B;
  a.T = T;
  a.D = D;
  a.act = activation;
  return a;
}

}  // namespace

extern "C" {

int m4sl_conv_forward(const m4sl_rows* x, const float* weight, const float* bias,
                      const void* initial, const int* lengths, int bf16, int B, int T, int D,
                      int W, int activation, void* output, void* state, void* stream) {
  const char* name = "m4sl_conv_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_conv(x, weight, B, T, D, W, activation, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!output) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(bf16, {x->data, initial, output, state}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    const bool wide =
        bf16 && conv_pieces(8, *x, T, D, bf16, weight, bias, {initial, output, state});
    const int vec = wide ? 8 : conv_vec(*x, T, D, bf16, weight, bias, {initial, output, state});
    cv::Conv a = conv_of(*x, weight, bias, initial, lengths, B, T, D, activation);
    a.y = output;
    a.state = state;
    a.cols = D / vec;
    // Runs of eight tokens, longer ones where those are more than a busy card needs.
    const long eights = (long)B * T * a.cols / busy_threads() / 8;
    a.run = 8 * (int)std::min(8L, std::max(1L, eights));
    a.runs = (T + a.run - 1) / a.run;
    const double blocks = ((double)B * a.runs * a.cols + cv::THREADS - 1) / cv::THREADS;
    if (too_many(blocks, cv::THREADS)) return api_fail(M4MR_EINVAL, at + "problem too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return api_launch("conv", st, [&] {
      start_width<Conv::FORWARD>(a, bf16, vec, W, dim3((unsigned)blocks), st);
    });
  });
}

size_t m4sl_conv_backward_workspace_bytes(int B, int T, int D, int W) {
  std::string why;
  const m4sl_rows any{&why, 0, 0};
  if (bad_conv(&any, reinterpret_cast<const float*>(&why), B, T, D, W, M4SL_NONE, &why)) return 0;
  // (The pieces depend on addresses.)
  size_t rows = conv_plan(B, T, D, W, 1).rows;
  if (D % 4 == 0) rows = std::max<size_t>(rows, conv_plan(B, T, D, W, 4).rows);
  return align256(rows * (W + 1) * D * sizeof(float));
}

int m4sl_conv_backward(const m4sl_rows* x, const float* weight, const float* bias,
                       const void* initial, const int* lengths, const void* d_output,
                       const void* d_state, int bf16, int B, int T, int D, int W,
                       int activation, void* d_x, void* d_initial, float* d_weight,
                       float* d_bias, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4sl_conv_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_conv(x, weight, B, T, D, W, activation, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!d_output) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(bf16, {x->data, initial, d_output, d_state, d_x, d_initial}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    const size_t need = m4sl_conv_backward_workspace_bytes(B, T, D, W);
    if (bad_workspace(workspace, workspace_bytes, need, &why))
      return api_fail(M4MR_EINVAL, at + why);
    const int vec = conv_vec(*x, T, D, bf16, weight, bias,
                             {initial, d_output, d_state, d_x, d_initial});
    const ConvPlan p = conv_plan(B, T, D, W, vec);
    cv::Conv a = conv_of(*x, weight, bias, initial, lengths, B, T, D, activation);
    const bool sums = d_weight || d_bias;
    a.run = p.run;
    a.runs = p.runs;
    a.cols = p.cols;
    a.lines = p.lines;
    a.dy = d_output;
    a.dstate = d_state;
    a.dx = d_x;
    a.dinitial = d_initial;
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    if (p.columns > 65535) return api_fail(M4MR_EINVAL, at + "problem too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = api_launch("conv_backward", st, [&] {
      start_width<Conv::BACKWARD>(a, bf16, vec, W, dim3(p.rows, p.columns), st);
    });
    if (rc || !sums) return rc;
    return api_launch("conv_join", st, [&] {
      hipLaunchKernelGGL(cv::conv_join_kernel, dim3((D + 63) / 64, W + 1), dim3(1024), 0, st,
                         a.part, (int)p.rows, W, D, d_weight, d_bias);
    });
  });
}

int m4sl_conv_step(const m4sl_rows* x, const float* weight, const float* bias,
                   const uint8_t* active, int bf16, int B, int D, int W, int activation,
                   const void* state, void* new_state, void* output, void* stream) {
  const char* name = "m4sl_conv_step";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_conv(x, weight, B, 1, D, W, activation, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!output || (W > 1 && (!state || !new_state)))
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(bf16, {x->data, state, new_state, output}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    const int vec = conv_vec(*x, 1, D, bf16, weight, bias, {state, new_state, output});
    cv::Step a{};
    a.x = x->data;
    a.xb = x->batch_stride;
    a.weight = weight;
    a.bias = bias;
    a.active = active;
    a.state = state;
    a.new_state = new_state;
    a.y = output;
    a.B = B;
    a.D = D;
    a.act = activation;
    a.cols = D / vec;
    a.blocks = (a.cols + cv::THREADS - 1) / cv::THREADS;
    const bool rows = (long)B * a.cols >= STEP_ROWS * busy_threads() / 2;
    const double blocks = (double)a.blocks * (rows ? (B + STEP_ROWS - 1) / STEP_ROWS : B);
    if (too_many(blocks, cv::THREADS)) return api_fail(M4MR_EINVAL, at + "problem too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)blocks);
    return api_launch("conv_step", st, [&] {
      if (rows)
        start_width<Conv::STEP_ROWS>(a, bf16, vec, W, grid, st);
      else
        start_width<Conv::STEP>(a, bf16, vec, W, grid, st);
    });
  });
}

}  // extern "C"

// ---------------------------------------------------- root-mean-square norm --

namespace {

bool bad_rms(long M, int C, std::string* why) {
  if (M <= 0 || C <= 0) {
    *why = "M and C must be positive";
    return true;
  }
  if (C > M4SL_MAX_NORM) {
    *why = "the channels must be at most " + std::to_string(M4SL_MAX_NORM);
    return true;
  }
  if ((double)M * C > 1e15) {
    *why = "problem too large";
    return true;
  }
  return false;
}

// Channels of a piece: eight, where all rows consist of such pieces.
int rms_vec(int C, std::initializer_list<const void*> arrays) {
  bool whole = C % 8 == 0;
  for (const void* p : arrays) whole = whole && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  return whole ? 8 : 1;
}

// How a row is spread: `pieces` of a lane, lanes of a wave up to 128 pieces of eight, more
// waves beyond.
struct RmsPlan {
  int pieces, threads;
  unsigned blocks;
};

RmsPlan rms_plan(long M, int C, int vec, bool backward, rn::Rms* a) {
  const int count = (C + vec - 1) / vec;
  RmsPlan p{};
  if (count <= 64) {
    p.pieces = 1;
    a->lanes = 1;
    while (a->lanes < count) a->lanes *= 2;
  } else {
    const int few = vec == 8 ? 2 : count <= 256 ? 4 : 8;
    p.pieces = count <= few * 1024 ? few : vec == 8 ? 4 : 32;
    a->lanes = ((count + p.pieces - 1) / p.pieces + 63) / 64 * 64;
  }
  a->rows = a->lanes <= 64 ? (backward ? 1024 : rn::THREADS) / a->lanes : 1;
  p.threads = a->lanes * a->rows;
  // (The backward's blocks leave partial sums: as few as keep the card busy.)
  const long most = (backward ? 1024L : 2048L) * m4::api_compute_units() / p.threads;
  p.blocks = (unsigned)std::min((M + a->rows - 1) / a->rows, std::max(1L, most));
  a->M = M;
  a->C = C;
  return p;
}

// What the launches do: the result in x's type, in 8 bits, or the gradient.
enum class Norm { FORWARD, E4M3, BACKWARD };

template <Norm WHAT, typename X, typename R, int V, int IT>
void start_rms_pieces(const rn::Rms& a, const RmsPlan& p, hipStream_t st) {
  const dim3 grid(p.blocks), block(p.threads);
  if constexpr (WHAT == Norm::BACKWARD)
    hipLaunchKernelGGL((rn::rms_backward_kernel<X, R, V, IT>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((rn::rms_kernel<X, R, V, IT, WHAT == Norm::E4M3>), grid, block, 0, st, a);
}

template <Norm WHAT, typename X, typename R>
void start_rms(const rn::Rms& a, const RmsPlan& p, int vec, hipStream_t st) {
  if (vec == 8) {
    if (p.pieces == 1) return start_rms_pieces<WHAT, X, R, 8, 1>(a, p, st);
    if (p.pieces == 2) return start_rms_pieces<WHAT, X, R, 8, 2>(a, p, st);
    return start_rms_pieces<WHAT, X, R, 8, 4>(a, p, st);
  }
  if (p.pieces == 1) return start_rms_pieces<WHAT, X, R, 1, 1>(a, p, st);
  if (p.pieces == 4) return start_rms_pieces<WHAT, X, R, 1, 4>(a, p, st);
  if (p.pieces == 8) return start_rms_pieces<WHAT, X, R, 1, 8>(a, p, st);
  return start_rms_pieces<WHAT, X, R, 1, 32>(a, p, st);
}

template <Norm WHAT>
int run_rms(const char* name, const rn::Rms& a, const RmsPlan& p, int vec, int x_bf16, int r_bf16,
            hipStream_t st) {
  return api_launch(name, st, [&] {
    if (x_bf16)
      r_bf16 ? start_rms<WHAT, rn::bf16_t, rn::bf16_t>(a, p, vec, st)
             : start_rms<WHAT, rn::bf16_t, float>(a, p, vec, st);
    else
      r_bf16 ? start_rms<WHAT, float, rn::bf16_t>(a, p, vec, st)
             : start_rms<WHAT, float, float>(a, p, vec, st);
  });
}

// The forward's checks, shared by both forms of the result.
bool bad_rms_forward(const void* x, int x_bf16, const void* residual, int residual_bf16, long M,
                     int C, const void* output, int output_bytes, const void* sum,
                     std::string* why) {
  if (bad_rms(M, C, why)) return true;
  if (!x || !output) {
    *why = "a required pointer is NULL";
    return true;
  }
  if (!residual && sum) {
    *why = "without a residual there is no sum";
    return true;
  }
  if (misaligned(x_bf16, {x}) || misaligned(residual_bf16, {residual, sum}) ||
      reinterpret_cast<uintptr_t>(output) % output_bytes) {
    *why = "arrays must be aligned to their elements";
    return true;
  }
  return false;
}

}  // namespace

extern "C" {

int m4sl_rms_forward(const void* x, int x_bf16, const void* residual, int residual_bf16,
                     const float* weight, long M, int C, float eps, void* output, void* sum,
                     float* inverse, void* stream) {
  const char* name = "m4sl_rms_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_rms_forward(x, x_bf16, residual, residual_bf16, M, C, output, x_bf16 ? 2 : 4, sum,
                        &why))
      return api_fail(M4MR_EINVAL, at + why);
    const int vec = rms_vec(C, {x, residual, weight, output, sum});
    rn::Rms a{};
    const RmsPlan p = rms_plan(M, C, vec, false, &a);
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.eps = eps;
    a.y = output;
    a.sum = sum;
    a.inverse = inverse;
    return run_rms<Norm::FORWARD>("rms", a, p, vec, x_bf16, residual ? residual_bf16 : x_bf16,
                                  static_cast<hipStream_t>(stream));
  });
}

int m4sl_rms_e4m3(const void* x, int x_bf16, const void* residual, int residual_bf16,
                  const float* weight, long M, int C, float eps, int block, void* output,
                  float* scale, void* sum, void* stream) {
  const char* name = "m4sl_rms_e4m3";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_rms_forward(x, x_bf16, residual, residual_bf16, M, C, output, 1, sum, &why))
      return api_fail(M4MR_EINVAL, at + why);
    if (!scale) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    const bool power = block >= 32 && block <= 512 && (block & (block - 1)) == 0;
    if (block <= 0 || (block < C && !power))
      return api_fail(M4MR_EINVAL,
                      at + "a scale's block must be a power of two in 32..512, or at least C");
    const int vec = rms_vec(C, {x, residual, weight, output, sum});
    rn::Rms a{};
    const RmsPlan p = rms_plan(M, C, vec, false, &a);
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.eps = eps;
    a.y = output;
    a.sum = sum;
    a.scale = scale;
    a.block = std::min(block, M4SL_MAX_NORM);
    a.blocks = (C + a.block - 1) / a.block;
    a.group = std::min(64, a.lanes);
    if (block < C) a.group = std::min(a.group, block / vec);
    return run_rms<Norm::E4M3>("rms_e4m3", a, p, vec, x_bf16, residual ? residual_bf16 : x_bf16,
                               static_cast<hipStream_t>(stream));
  });
}

size_t m4sl_rms_backward_workspace_bytes(long M, int C) {
  std::string why;
  if (bad_rms(M, C, &why)) return 0;
  // (The pieces depend on addresses.)
  rn::Rms a{};
  unsigned blocks = rms_plan(M, C, 1, true, &a).blocks;
  if (C % 8 == 0) blocks = std::max(blocks, rms_plan(M, C, 8, true, &a).blocks);
  return align256((size_t)blocks * C * sizeof(float));
}

int m4sl_rms_backward(const void* sum, int sum_bf16, const float* weight, const float* inverse,
                      const void* d_output, int x_bf16, const void* d_sum, long M, int C,
                      void* d_x, void* d_residual, float* d_weight, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const char* name = "m4sl_rms_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_rms(M, C, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!sum || !inverse || !d_output)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(x_bf16, {d_output, d_x}) || misaligned(sum_bf16, {sum, d_sum, d_residual}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    if (bad_workspace(workspace, workspace_bytes, m4sl_rms_backward_workspace_bytes(M, C), &why))
      return api_fail(M4MR_EINVAL, at + why);
    const int vec = rms_vec(C, {sum, weight, d_output, d_sum, d_x, d_residual});
    rn::Rms a{};
    const RmsPlan p = rms_plan(M, C, vec, true, &a);
    a.x = sum;
    a.weight = weight;
    a.inverse = const_cast<float*>(inverse);
    a.dy = d_output;
    a.dsum = d_sum;
    a.dx = d_x;
    a.dresidual = d_residual;
    a.part = d_weight ? static_cast<float*>(workspace) : nullptr;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = run_rms<Norm::BACKWARD>("rms_backward", a, p, vec, x_bf16, sum_bf16, st);
    if (rc || !d_weight) return rc;
    return api_launch("rms_join", st, [&] {
      hipLaunchKernelGGL(rn::rms_join_kernel, dim3((C + 63) / 64), dim3(1024), 0, st, a.part,
                         (int)p.blocks, C, d_weight);
    });
  });
}

}  // extern "C"

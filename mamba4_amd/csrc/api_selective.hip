// C ABI of the selective layer's operators (include/mamba4_selective.h): the checks
// of the arguments and the launches.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <cstring>
#include <initializer_list>

#include "../../include/mamba4_selective.h"
#include "api_common.hpp"
#include "selscan.hpp"

namespace ss {
template <typename In, int NG, bool OUT>
__global__ void scan_kernel(Scan);
template <typename In, int NG, bool ALL>
__global__ void scan_backward_kernel(Scan);
template <bool BWD>
__global__ void carry_kernel(Scan);
template <typename In>
__global__ void join_bc_kernel(Join);
__global__ void join_rows_kernel(const float*, long, long, long, float, float*);
template <typename In>
__global__ void step_kernel(Step);
}  // namespace ss

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

bool whole_rows(const m4sl_rows& r) {
  return r.batch_stride % 4 == 0 && r.token_stride % 4 == 0;
}

// ---------------------------------------------------------- selective scan --

int tiles_of(int T) { return (T + ss::TILE - 1) / ss::TILE; }

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
      (tokens && s->T > INT_MAX - (1 << 16)) || (double)s->D * s->N > 1e9) {
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

// Segments that a sequence is cut into.  A walk from end to end takes a tile's latency
// a tile; segments cost their states first (0.75 of the outputs' instructions, again),
// so that sequences are cut only where their waves leave the card idle, and into no
// more than fill it.
int segments(const m4sl_scan& s) {
  const long waves = (long)s.B * s.G * ((s.D / s.G + 15) / 16);
  const long full = 4L * m4::api_compute_units();
  if (waves >= full) return 1;
  const long want = (3 * full + waves - 1) / waves, most = tiles_of(s.T) / 2;
  const long cut = std::min(want, most);
  return cut < 3 ? 1 : (int)std::min(cut, 4096L);
}

ss::Rows rows_of(const m4sl_rows& r) { return ss::Rows{r.data, r.batch_stride, r.token_stride}; }

ss::Scan scan_of(const m4sl_scan& s, const int* lengths) {
  ss::Scan a{};
  a.x = rows_of(s.x);
  a.delta = rows_of(s.delta);
  a.gate = rows_of(s.gate);
  a.b = rows_of(s.b);
  a.c = rows_of(s.c);
  a.bg = s.b_group_stride;
  a.cg = s.c_group_stride;
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
  a.whole = a.Dg % 4 == 0 && whole_rows(s.x) && whole_rows(s.delta) && whole_rows(s.gate) &&
            whole_at(s.bf16, {s.x.data, s.delta.data, s.gate.data});
  a.whole_bc = s.N % 4 == 0 && whole_rows(s.b) && whole_rows(s.c) && a.bg % 4 == 0 &&
               a.cg % 4 == 0 && whole_at(s.bf16, {s.b.data, s.c.data});
  a.blocks = blocks_of(s);
  const int cut = segments(s), tiles = tiles_of(s.T);
  a.seg = (tiles + cut - 1) / cut * ss::TILE;
  a.NS = (s.T + a.seg - 1) / a.seg;
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

template <typename In, bool OUT>
void start_scan(const ss::Scan& a, hipStream_t st) {
  const dim3 grid(a.B * a.G * a.blocks, a.NS), block(64 * ss::WAVES);
  if (a.N <= 16)
    hipLaunchKernelGGL((ss::scan_kernel<In, 1, OUT>), grid, block, 0, st, a);
  else if (a.N <= 32)
    hipLaunchKernelGGL((ss::scan_kernel<In, 2, OUT>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ss::scan_kernel<In, 4, OUT>), grid, block, 0, st, a);
}

template <typename In, bool ALL>
void start_scan_backward(const ss::Scan& a, hipStream_t st) {
  const dim3 grid(a.B * a.G * a.blocks, a.NS), block(64 * ss::WAVES);
  if (a.N <= 16)
    hipLaunchKernelGGL((ss::scan_backward_kernel<In, 1, ALL>), grid, block, 0, st, a);
  else if (a.N <= 32)
    hipLaunchKernelGGL((ss::scan_backward_kernel<In, 2, ALL>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ss::scan_backward_kernel<In, 4, ALL>), grid, block, 0, st, a);
}

template <bool BWD>
int run_carry(const ss::Scan& a, hipStream_t st) {
  const unsigned blocks = element_blocks((long)a.B * a.D * a.N);
  return api_launch(BWD ? "scan_backward_carry" : "scan_carry", st, [&] {
    hipLaunchKernelGGL(ss::carry_kernel<BWD>, dim3(blocks), dim3(256), 0, st, a);
  });
}

int run_join(const char* name, const float* part, long rows, long stride, long count, float* out,
             hipStream_t st) {
  return api_launch(name, st, [&] {
    hipLaunchKernelGGL(ss::join_rows_kernel, dim3(element_blocks(count)), dim3(256), 0, st, part,
                       rows, stride, count, 1.f, out);
  });
}

}  // namespace

extern "C" {

long m4sl_scan_kept_floats(const m4sl_scan* s) {
  std::string why;
  if (bad_scan(s, true, &why)) return 0;
  return (long)s->B * tiles_of(s->T) * s->D * s->N;
}

size_t m4sl_scan_workspace_bytes(const m4sl_scan* s) {
  std::string why;
  if (bad_scan(s, true, &why)) return 0;
  ss::Scan a = scan_of(*s, nullptr);
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
    ss::Scan a = scan_of(*s, lengths);
    Carver c{static_cast<char*>(workspace)};
    if (bad_workspace(workspace, workspace_bytes, take_segments(c, &a), &why))
      return api_fail(M4MR_EINVAL, at + why);
    a.whole = a.whole && whole_at(s->bf16, {output});
    a.initial = initial;
    a.out = output;
    a.state = state;
    a.kept = kept;
    a.whole_n = a.N % 4 == 0 && whole_at(0, {a.a, initial, state, kept});
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.NS > 1) {
      int rc = api_launch("scan_states", st, [&] {
        s->bf16 ? start_scan<ss::bf16_t, false>(a, st) : start_scan<float, false>(a, st);
      });
      if (rc) return rc;
      rc = run_carry<false>(a, st);
      if (rc) return rc;
    }
    return api_launch("scan", st, [&] {
      s->bf16 ? start_scan<ss::bf16_t, true>(a, st) : start_scan<float, true>(a, st);
    });
  });
}

size_t m4sl_scan_backward_workspace_bytes(const m4sl_scan* s) {
  std::string why;
  if (bad_scan(s, true, &why)) return 0;
  ss::Scan a = scan_of(*s, nullptr);
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
    ss::Scan a = scan_of(*s, lengths);
    Carver c{static_cast<char*>(workspace)};
    if (bad_workspace(workspace, workspace_bytes, take_backward(c, &a), &why))
      return api_fail(M4MR_EINVAL, at + why);
    a.whole = a.whole && whole_at(s->bf16, {d_output, grads->x, grads->delta, grads->gate});
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
      rc = api_launch("scan_backward_states", st, [&] {
        s->bf16 ? start_scan_backward<ss::bf16_t, false>(a, st)
                : start_scan_backward<float, false>(a, st);
      });
      if (rc) return rc;
      rc = run_carry<true>(a, st);
      if (rc) return rc;
    }
    rc = api_launch("scan_backward", st, [&] {
      s->bf16 ? start_scan_backward<ss::bf16_t, true>(a, st)
              : start_scan_backward<float, true>(a, st);
    });
    if (rc) return rc;
    ss::Join j{a.part_bc, a.blocks, a.B, a.T, a.G, a.N, lengths, grads->b, grads->c};
    rc = api_launch("scan_join_bc", st, [&] {
      const dim3 grid(element_blocks((long)a.B * a.T * a.G * a.N)), block(256);
      if (s->bf16)
        hipLaunchKernelGGL(ss::join_bc_kernel<ss::bf16_t>, grid, block, 0, st, j);
      else
        hipLaunchKernelGGL(ss::join_bc_kernel<float>, grid, block, 0, st, j);
    });
    if (rc) return rc;
    const long rows = (long)a.B * a.NS, states = (long)a.D * a.N;
    if (grads->a) rc = run_join("scan_join_a", a.part_a, rows, states, states, grads->a, st);
    if (!rc && grads->skip && s->skip)
      rc = run_join("scan_join_skip", a.part_d, rows, 2L * a.D, a.D, grads->skip, st);
    if (!rc && grads->delta_bias && s->delta_bias)
      rc = run_join("scan_join_bias", a.part_d + a.D, rows, 2L * a.D, a.D, grads->delta_bias, st);
    return rc;
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
    while (a.span < 2 && 4 << a.span < s->N) ++a.span;
    const double blocks =
        ((double)s->B * s->D * (1 << a.span) + ss::STEP_THREADS - 1) / ss::STEP_THREADS;
    if (too_many(blocks, ss::STEP_THREADS))
      return api_fail(M4MR_EINVAL, at + "problem too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return api_launch("scan_step", st, [&] {
      const dim3 grid((unsigned)blocks), block(ss::STEP_THREADS);
      if (s->bf16)
        hipLaunchKernelGGL(ss::step_kernel<ss::bf16_t>, grid, block, 0, st, a);
      else
        hipLaunchKernelGGL(ss::step_kernel<float>, grid, block, 0, st, a);
    });
  });
}

}  // extern "C"

// C ABI of the retention layer's operators (include/mamba4_retention.h): the
// checks of the arguments and the launches.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <initializer_list>

#include "../../include/mamba4_retention.h"
#include "api_common.hpp"
#include "embed.hpp"
#include "linattn.hpp"
#include "norm.hpp"

namespace la {
template <typename In, int NT>
__global__ void attention_kernel(Args);
template <typename In, int NT>
__global__ void attention_states_kernel(Args);
template <typename In, int NP, int NN, bool DOTS>
__global__ void attention_backward_kernel(Args);
__global__ void carry_kernel(Args);
__global__ void decay_grad_kernel(DecayGrad);
__global__ void decay_heads_kernel(const double*, int, int, int, float*);
template <typename Out>
__global__ void share_sum_kernel(const float*, long, int, int, int, Out*);
template <typename In>
__global__ void pack_kernel(Pack);
template <typename In, int V, int PASSES>
__global__ void step_kernel(Step);
}  // namespace la

namespace gn {
template <typename In, int V, int IT, bool BWD>
__global__ void norm_rows_kernel(Norm);
template <typename In, int V, bool BWD, int PHASE>
__global__ void norm_positions_kernel(Norm);
__global__ void norm_columns_kernel(const float*, int, int, float*, float*);
}  // namespace gn

namespace em {
template <typename In, typename Out, int V>
__global__ void lookup_kernel(Lookup);
__global__ void count_kernel(Sort, unsigned*, Clear);
__global__ void scatter_kernel(Sort);
template <typename In, typename Out, int V>
__global__ void sum_kernel(Sum, unsigned);
template <typename Out, int V>
__global__ void join_kernel(Sum);
}  // namespace em

namespace {

using m4::align256;
using m4::api_fail;
using m4::api_launch;
using m4::bad_workspace;
using m4::Carver;

// ------------------------------------------------------ linear attention --

constexpr int MAX_GRID_Y = 65535;

struct Shape {
  int B, T, H, N, P, bf16;
  int chunks() const { return (T + la::C - 1) / la::C; }
};

int tiles_of(int width) { return (width + la::TILE - 1) / la::TILE; }

// Chunks of a segment, by the chunk-tiles of one row (`blocks` tiles a head):
// 4 while a segment is latency, up to 16 where the segments' states are traffic.
// It does not depend on the batch size (segments decide the bits).  Forward calls,
// bfloat16, 4 / 8 / 16: B1 T2000 H12 N64 P128 29 / 37 / 62 us, B1 T4200 H32 N128 P128
// 101 / 96 / 105, B1 T32768 H16 N128 P128 390 / 334 / 319; forward and backward, B1
// T2100 and T4200 H32 N128 P128 206 / 193 / 252 and 412 / 351 / 343.  Longer ones only
// keep the segments within a launch's y blocks (past 67M tokens).
int segment(const Shape& s, int blocks) {
  const long each = (long)s.chunks() * s.H * blocks / 768;
  int seg = each >= 16 ? 16 : each >= 8 ? 8 : 4;
  while ((s.chunks() - 1) / seg >= MAX_GRID_Y) seg *= 2;
  return seg;
}

int segments(const Shape& s, int blocks) {
  const int seg = segment(s, blocks);
  return (s.chunks() + seg - 1) / seg;
}

// `blocks`, `threads`: blocks of the widest launch for each (b, h), and of a block.
bool bad_shape(const Shape& s, int blocks, int threads, std::string* why) {
  if (s.B <= 0 || s.T <= 0 || s.H <= 0) {
    *why = "B, T and H must be positive";
    return true;
  }
  if (s.N <= 0 || s.P <= 0 || s.N > M4RT_MAX_WIDTH || s.P > M4RT_MAX_WIDTH) {
    *why = "key and value widths must be in 1.." + std::to_string(M4RT_MAX_WIDTH);
    return true;
  }
  // A launch takes fewer than 2^32 threads along x; (b, h) are rounded up to eights.
  if (((double)s.B * s.H + 8) * blocks * threads >= 4294967296.0 || s.T > INT_MAX / 16) {
    *why = "problem too large";
    return true;
  }
  return false;
}

// Whether the sequences are split into segments (their states formed first,
// then carried, then all walked at once) instead of walked from end to end.  A walk
// takes a chunk's latency a chunk while the card has a block a compute unit, and the
// chunks' throughput beyond; a split run three launches, a segment's latency twice,
// and 1.7 times the throughput.  Walk / split in us, calls: forward bfloat16 N64 P128
// H12 B4 T2000 73 / 49, B8 T1024 40 / 47, B16 T1024 57 / 79; float32 B4 T1024 78 / 56,
// B8 T1024 80 / 83; forward and backward float32 N64 P64 H8 B8 T1000 191 / 153.
// M4RT_ATTENTION = "walk" or "split" overrides the choice; the bits are the same.
bool attention_splits(const Shape& s, int blocks) {
  if (segments(s, blocks) < 2) return false;
  if (const char* mode = std::getenv("M4RT_ATTENTION")) {
    if (std::strcmp(mode, "walk") == 0) return false;
    if (std::strcmp(mode, "split") == 0) return true;
  }
  const bool backward = blocks > tiles_of(s.P), wide = s.N > 64 || (backward && s.P > 64);
  // us a chunk: alone, and of a busy compute unit.
  const double more = wide ? 1.5 : 1.0;
  const double latency = more * (s.bf16 ? 2.1 : 4.1) * (backward ? (s.bf16 ? 1.2 : 1.6) : 1.0);
  const double busy = more * (s.bf16 ? 1.9 : 3.9) * (backward ? (s.bf16 ? 1.25 : 1.1) : 1.0);
  const double units = m4::api_compute_units(), walks = (double)s.B * s.H * blocks;
  const double walk = s.chunks() * std::max(latency, busy * std::ceil(walks / units));
  const double split = 8.0 + std::max(1.6 * segment(s, blocks) * latency,
                                      1.7 * busy * s.chunks() * walks / units);
  return split < walk;
}

// How a call runs its sequences.  Settled once a call: the workspace is carved for it.
struct Route {
  int segments;
  bool split;
};

Route attention_route(const Shape& s, int blocks) {
  return Route{segments(s, blocks), attention_splits(s, blocks)};
}

// The segments' states of one role (n keys wide, `tiles` blocks of values); no
// segments: none are kept.
void take_states(Carver& c, const Shape& s, int n, int tiles, int segments, la::Role* role) {
  const size_t slots = (size_t)tiles * s.B * s.H * segments;
  role->starts = c.take<float>(slots * tiles_of(n) * la::TILE * la::TILE);
  role->decays = c.take<float>(slots);
}

// Rows as the kernels take them: whole, where every row consists of 16-byte
// pieces at multiples of 16 bytes.
la::Rows rows_of(const m4rt_rows& r, int H, int bf16) {
  const int piece = bf16 ? 8 : 4;
  const bool whole = reinterpret_cast<uintptr_t>(r.data) % 16 == 0 &&
                     r.batch_stride % piece == 0 && r.token_stride % piece == 0 &&
                     r.head_stride % piece == 0 && r.width % piece == 0;
  return la::Rows{r.data, r.batch_stride, r.token_stride, r.head_stride, H / r.heads, r.width,
                  whole};
}

// The rows in the order given, those that are no 16-byte pieces copied to padded
// rows: space for the copies, and their kernel.
struct Packing {
  la::Pack a{};
  int count = 0;
  long most = 0;  // pieces of the largest copy
};

// The token stride of dense rows; of one token, whose stride is no stride, the width.
long token_stride(int T, int heads, int width) { return T > 1 ? (long)heads * width : width; }

void pack_rows(Carver& c, const Shape& s, la::Rows* r, int heads, Packing* out) {
  if (r->whole) return;
  const int piece = s.bf16 ? 8 : 4, i = out->count++;
  const int width = (r->width + piece - 1) / piece * piece;
  const size_t rows = (size_t)s.B * s.T * heads;
  out->a.from[i] = *r;
  out->a.to[i] = c.take<char>(rows * width * (16 / piece));
  out->a.heads[i] = heads;
  out->a.padded[i] = width;
  out->most = std::max(out->most, (long)(rows * (width / piece)));
  *r = la::Rows{out->a.to[i], (long)s.T * heads * width, token_stride(s.T, heads, width), width,
                r->share, width, 1};
}

// Blocks of 256 threads that take an element each in turn: as many as the elements
// need, within a launch's 2^32 threads (the kernels walk on from there).
unsigned element_blocks(long count) {
  return (unsigned)std::min<long>((count + 255) / 256, 1 << 16);
}

int run_packing(Packing& p, const Shape& s, hipStream_t st) {
  if (p.count == 0) return M4MR_OK;
  p.a.B = s.B;
  p.a.T = s.T;
  const dim3 grid(element_blocks(p.most), p.count), block(256);
  return api_launch("attention_pack", st, [&] {
    if (s.bf16)
      hipLaunchKernelGGL(la::pack_kernel<la::bf16_t>, grid, block, 0, st, p.a);
    else
      hipLaunchKernelGGL(la::pack_kernel<float>, grid, block, 0, st, p.a);
  });
}

// A chunk's rows are addressed by 32-bit byte offsets.
bool bad_stride(long token_stride, std::string* why) {
  if (token_stride <= INT_MAX / (4 * la::C)) return false;
  *why = "a token stride must be at least the width, and 64 of it below 2^31 bytes";
  return true;
}

// The token stride of `r` as the kernels read it: of its copy, if it is copied.
long read_stride(const m4rt_rows& r, int T, int H, int bf16) {
  const int piece = bf16 ? 8 : 4;
  return rows_of(r, H, bf16).whole
             ? r.token_stride
             : token_stride(T, r.heads, (r.width + piece - 1) / piece * piece);
}

// T: tokens, or zero for rows without that axis.
bool bad_rows(const m4rt_rows* r, int H, int bf16, int T, std::string* why) {
  if (!r->data) {
    *why = "a required pointer is NULL";
    return true;
  }
  if (r->heads <= 0 || H % r->heads) {
    *why = "the heads of queries, keys and values must divide H";
    return true;
  }
  if (reinterpret_cast<uintptr_t>(r->data) % (bf16 ? 2 : 4)) {
    *why = "rows must be aligned to their elements";
    return true;
  }
  if (T == 0) return false;
  return bad_stride(r->token_stride < r->width ? LONG_MAX : r->token_stride, why) ||
         bad_stride(read_stride(*r, T, H, bf16), why);
}

m4rt_rows dense(const void* data, int T, int H, int width) {
  return m4rt_rows{data, (long)T * H * width, token_stride(T, H, width), width, H, width};
}

int wide_keys(const la::Args& a) {
  for (int i = 0; i < a.roles; ++i)
    if (a.role[i].n > 64) return 2;
  return 1;
}

template <typename In>
void start_states(const la::Args& a, dim3 grid, hipStream_t st) {
  const dim3 block(64 * la::WAVES);
  if (wide_keys(a) == 1)
    hipLaunchKernelGGL((la::attention_states_kernel<In, 1>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((la::attention_states_kernel<In, 2>), grid, block, 0, st, a);
}

template <typename In, int NP, int NN>
void start_backward(const la::Args& a, dim3 grid, hipStream_t st) {
  const dim3 block(128 * la::WAVES);
  if (a.role[0].dots)
    hipLaunchKernelGGL((la::attention_backward_kernel<In, NP, NN, true>), grid, block, 0,
                       st, a);
  else
    hipLaunchKernelGGL((la::attention_backward_kernel<In, NP, NN, false>), grid, block, 0,
                       st, a);
}

template <typename In>
void start_outputs(const la::Args& a, dim3 grid, hipStream_t st) {
  const dim3 block(128 * la::WAVES);
  if (a.roles == 1) {
    if (a.role[0].n <= 64)
      hipLaunchKernelGGL((la::attention_kernel<In, 1>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((la::attention_kernel<In, 2>), grid, block, 0, st, a);
    return;
  }
  const bool wide_p = a.role[0].n > 64, wide_n = a.role[2].n > 64;
  if (wide_p)
    wide_n ? start_backward<In, 2, 2>(a, grid, st)
           : start_backward<In, 2, 1>(a, grid, st);
  else
    wide_n ? start_backward<In, 1, 2>(a, grid, st)
           : start_backward<In, 1, 1>(a, grid, st);
}

template <typename In>
int start_attention(const la::Args& a, hipStream_t st) {
  const unsigned x = (unsigned)((a.B * a.H + 7) / 8 * 8 * a.blocks);
  if (a.split) {
    int rc = api_launch("attention_states", st,
                        [&] { start_states<In>(a, dim3(x, a.NS), st); });
    if (rc) return rc;
    rc = api_launch("attention_carry", st, [&] {
      hipLaunchKernelGGL(la::carry_kernel, dim3(x, 4 * wide_keys(a)), dim3(64 * la::WAVES), 0, st,
                         a);
    });
    if (rc) return rc;
  }
  return api_launch("attention", st,
                    [&] { start_outputs<In>(a, dim3(x, a.split ? a.NS : 1), st); });
}

int run_attention(la::Args& a, const Shape& s, const Route& route, hipStream_t st) {
  a.blocks = 0;
  for (int i = 0; i < a.roles; ++i) a.blocks += a.role[i].tiles;
  a.B = s.B;
  a.T = s.T;
  a.H = s.H;
  a.NC = s.chunks();
  a.seg = segment(s, a.blocks);
  a.NS = route.segments;
  a.split = route.split;
  return s.bf16 ? start_attention<la::bf16_t>(a, st) : start_attention<float>(a, st);
}

// The step with as many loads in flight as its rows need.
template <typename In>
void start_step(const la::Step& a, bool whole, hipStream_t st) {
  const dim3 grid(a.B * a.H), block(la::STEP_THREADS);
  const int rows = la::STEP_THREADS >> a.span, passes = (a.N + rows - 1) / rows;
  if (!whole)
    hipLaunchKernelGGL((la::step_kernel<In, 1, 16>), grid, block, 0, st, a);
  else if (passes <= 4)
    hipLaunchKernelGGL((la::step_kernel<In, 4, 4>), grid, block, 0, st, a);
  else if (passes <= 8)
    hipLaunchKernelGGL((la::step_kernel<In, 4, 8>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((la::step_kernel<In, 4, 16>), grid, block, 0, st, a);
}

// The rows of a call as the kernels take them.
struct Operands {
  la::Rows q, k, v, d_output;
  Packing packing;
};

struct Backward {
  la::Role role[3];
  float *part[3], *dots_q, *dots_k;
  double* head;
};

int backward_tiles(const Shape& s) { return 2 * tiles_of(s.N) + tiles_of(s.P); }

// The forward's workspace: the segments' states of a split, packed rows.
size_t forward_workspace(const Shape& s, const m4rt_qkv& rows, const Route& route, void* base,
                         la::Role* role, Operands* x) {
  Carver c{static_cast<char*>(base)};
  take_states(c, s, s.N, tiles_of(s.P), route.split ? route.segments : 0, role);
  x->q = rows_of(rows.q, s.H, s.bf16);
  x->k = rows_of(rows.k, s.H, s.bf16);
  x->v = rows_of(rows.v, s.H, s.bf16);
  pack_rows(c, s, &x->q, rows.q.heads, &x->packing);
  pack_rows(c, s, &x->k, rows.k.heads, &x->packing);
  pack_rows(c, s, &x->v, rows.v.heads, &x->packing);
  return c.used;
}

// The backward's workspace: the segments' states (of dQ and dK for the decays'
// gradient too), float32 gradients of shared heads before their sums, the dots, the
// heads' sums, packed rows.
size_t backward_workspace(const Shape& s, const m4rt_qkv& rows, const Route& route,
                          const void* d_output, bool decays, void* base, Backward* out,
                          Operands* x) {
  Carver c{static_cast<char*>(base)};
  const int n[3] = {s.P, s.P, s.N}, p[3] = {s.N, s.N, s.P};
  const int heads[3] = {rows.q.heads, rows.k.heads, rows.v.heads};
  const size_t tokens = (size_t)s.B * s.T * s.H;
  const int count = route.segments;
  for (int i = 0; i < 3; ++i) {
    take_states(c, s, n[i], tiles_of(p[i]), route.split || (decays && i < 2) ? count : 0,
                &out->role[i]);
    out->part[i] = c.take<float>(heads[i] == s.H ? 0 : tokens * p[i]);
  }
  out->dots_q = c.take<float>(decays ? tokens * tiles_of(s.N) : 0);
  out->dots_k = c.take<float>(decays ? tokens * tiles_of(s.N) : 0);
  out->head = c.take<double>(decays ? (size_t)s.B * s.H * count : 0);
  x->q = rows_of(rows.q, s.H, s.bf16);
  x->k = rows_of(rows.k, s.H, s.bf16);
  x->v = rows_of(rows.v, s.H, s.bf16);
  x->d_output = rows_of(dense(d_output, s.T, s.H, s.P), s.H, s.bf16);
  pack_rows(c, s, &x->q, heads[0], &x->packing);
  pack_rows(c, s, &x->k, heads[1], &x->packing);
  pack_rows(c, s, &x->v, heads[2], &x->packing);
  pack_rows(c, s, &x->d_output, s.H, &x->packing);
  return c.used;
}

// The attention's shape from its rows, if they and it are sound, for the forward or
// the backward.
bool bad_attention(const m4rt_qkv* rows, int bf16, int B, int T, int H, bool backward, Shape* s,
                   std::string* why) {
  if (!rows) {
    *why = "a required pointer is NULL";
    return true;
  }
  *s = Shape{B, T, H, rows->q.width, rows->v.width, bf16};
  if (bad_shape(*s, backward ? backward_tiles(*s) : tiles_of(s->P), 128 * la::WAVES, why))
    return true;
  for (const m4rt_rows* r : {&rows->q, &rows->k, &rows->v})
    if (bad_rows(r, H, bf16, T, why)) return true;
  if (rows->q.width != rows->k.width) {
    *why = "q and k disagree in width";
    return true;
  }
  // The backward reads d_output too, dense, or copied if its address asks for that.
  const int piece = bf16 ? 8 : 4;
  return backward && bad_stride(token_stride(T, H, (s->P + piece - 1) / piece * piece), why);
}

}  // namespace

extern "C" {

size_t m4rt_attention_workspace_bytes(const m4rt_qkv* rows, int bf16, int B, int T, int H) {
  Shape s;
  std::string why;
  la::Role role{};
  Operands x{};
  if (bad_attention(rows, bf16, B, T, H, false, &s, &why)) return 0;
  return forward_workspace(s, *rows, attention_route(s, tiles_of(s.P)), nullptr, &role, &x);
}

size_t m4rt_attention_backward_workspace_bytes(const m4rt_qkv* rows, const void* d_output,
                                               int bf16, int B, int T, int H, int decays) {
  Shape s;
  std::string why;
  Backward w{};
  Operands x{};
  if (bad_attention(rows, bf16, B, T, H, true, &s, &why)) return 0;
  return backward_workspace(s, *rows, attention_route(s, backward_tiles(s)), d_output, decays,
                            nullptr, &w, &x);
}

int m4rt_attention_forward(const m4rt_qkv* rows, int bf16, const float* log_decay, int per_token,
                           const int* lengths, const float* initial, float scale, int B, int T,
                           int H, void* output, float* state, void* workspace,
                           size_t workspace_bytes, void* stream) {
  const char* name = "m4rt_attention_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    Shape s;
    std::string why;
    if (bad_attention(rows, bf16, B, T, H, false, &s, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!log_decay || !output) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    la::Args a{};
    la::Role& r = a.role[0];
    Operands x{};
    const Route route = attention_route(s, tiles_of(s.P));
    const size_t need = forward_workspace(s, *rows, route, workspace, &r, &x);
    if (bad_workspace(workspace, workspace_bytes, need, &why))
      return api_fail(M4MR_EINVAL, at + why);
    r.q = x.q;
    r.k = x.k;
    r.v = x.v;
    r.initial = la::States{const_cast<float*>(initial), s.P, 1};
    r.final = la::States{state, s.P, 1};
    r.out = output;
    r.out_f32 = !bf16;
    r.intra = r.inter = scale;
    r.update = 1.f;
    r.n = s.N;
    r.p = s.P;
    r.tiles = tiles_of(s.P);
    a.roles = 1;
    a.g = log_decay;
    a.gb = per_token ? (long)T * H : 0;
    a.gt = per_token ? H : 0;
    a.lengths = lengths;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = run_packing(x.packing, s, st);
    return rc ? rc : run_attention(a, s, route, st);
  });
}

int m4rt_attention_backward(const m4rt_qkv* rows, int bf16, const float* log_decay,
                            int per_token, const int* lengths, const float* initial, float scale,
                            int B, int T, int H, const void* d_output, const float* d_state, const float* state,
                            void* d_q, void* d_k, void* d_v, float* d_log_decay, float* d_initial,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4rt_attention_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    Shape s;
    std::string why;
    if (bad_attention(rows, bf16, B, T, H, true, &s, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!log_decay || !d_output || !d_q || !d_k || !d_v || (d_state && d_log_decay && !state))
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    const int heads[3] = {rows->q.heads, rows->k.heads, rows->v.heads};
    Backward w{};
    Operands x{};
    const Route route = attention_route(s, backward_tiles(s));
    const size_t need =
        backward_workspace(s, *rows, route, d_output, d_log_decay != nullptr, workspace, &w, &x);
    if (bad_workspace(workspace, workspace_bytes, need, &why))
      return api_fail(M4MR_EINVAL, at + why);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = run_packing(x.packing, s, st);
    if (rc) return rc;
    la::Args a{};
    void* outs[3] = {d_q, d_k, d_v};
    for (int i = 0; i < 3; ++i) {
      la::Role& r = a.role[i];
      r = w.role[i];
      const bool shared = heads[i] != H;
      r.out = shared ? (void*)w.part[i] : outs[i];
      r.out_f32 = !bf16 || shared;
      r.rev = i > 0;
      r.intra = scale;
      r.inter = i == 0 ? scale : 1.f;
      r.update = i == 0 ? 1.f : scale;
      r.n = i == 2 ? s.N : s.P;
      r.p = i == 2 ? s.P : s.N;
      r.tiles = tiles_of(r.p);
    }
    // dQ from the transposed state, dK and dV from the state's cotangent.
    la::Role &rdq = a.role[0], &rdk = a.role[1], &rdv = a.role[2];
    rdq.q = x.d_output, rdq.k = x.v, rdq.v = x.k;
    rdk.q = x.v, rdk.k = x.d_output, rdk.v = x.q;
    rdv.q = x.k, rdv.k = x.q, rdv.v = x.d_output;
    rdq.initial = la::States{const_cast<float*>(initial), 1, s.P};
    rdk.initial = la::States{const_cast<float*>(d_state), 1, s.P};
    rdv.initial = la::States{const_cast<float*>(d_state), s.P, 1};
    rdv.final = la::States{d_initial, s.P, 1};
    if (d_log_decay) {
      rdq.e = x.q, rdq.dots = w.dots_q;
      rdk.e = x.k, rdk.dots = w.dots_k;
    }
    a.roles = 3;
    a.g = log_decay;
    a.gb = per_token ? (long)T * H : 0;
    a.gt = per_token ? H : 0;
    a.lengths = lengths;
    rc = run_attention(a, s, route, st);
    if (rc) return rc;
    for (int i = 0; i < 3; ++i) {
      if (heads[i] == H) continue;
      const long count = (long)B * T * heads[i] * a.role[i].p;
      rc = api_launch("attention_share", st, [&] {
        const dim3 grid(element_blocks(count));
        const int share = H / heads[i];
        if (bf16)
          hipLaunchKernelGGL(la::share_sum_kernel<la::bf16_t>, grid, dim3(256), 0, st, w.part[i],
                             (long)B * T, H, share, a.role[i].p, static_cast<la::bf16_t*>(outs[i]));
        else
          hipLaunchKernelGGL(la::share_sum_kernel<float>, grid, dim3(256), 0, st, w.part[i],
                             (long)B * T, H, share, a.role[i].p, static_cast<float*>(outs[i]));
      });
      if (rc) return rc;
    }
    if (!d_log_decay) return (int)M4MR_OK;
    la::DecayGrad d{};
    d.dots_q = w.dots_q;
    d.dots_k = w.dots_k;
    d.starts_q = w.role[0].starts;
    d.starts_k = w.role[1].starts;
    d.tiles = tiles_of(s.N);
    d.slot = tiles_of(s.P) * la::TILE * la::TILE;
    d.seg = a.seg;
    d.NS = a.NS;
    d.g = log_decay;
    d.gb = a.gb;
    d.gt = a.gt;
    d.lengths = lengths;
    d.state = d_state ? state : nullptr;
    d.d_state = d_state;
    d.n = s.N;
    d.p = s.P;
    d.d_g = per_token ? d_log_decay : nullptr;
    d.head = per_token ? nullptr : w.head;
    d.B = B;
    d.T = T;
    d.H = H;
    rc = api_launch("attention_decay", st, [&] {
      hipLaunchKernelGGL(la::decay_grad_kernel, dim3(B * H, a.NS), dim3(la::GRAD_THREADS), 0, st,
                         d);
    });
    if (rc || per_token) return rc;
    return api_launch("attention_heads", st, [&] {
      hipLaunchKernelGGL(la::decay_heads_kernel, dim3(H), dim3(64), 0, st, w.head, B, H, a.NS,
                         d_log_decay);
    });
  });
}

int m4rt_attention_step(const m4rt_qkv* rows, int bf16, const float* log_decay, int per_token,
                        const uint8_t* active, float scale, int B, int H, const float* state,
                        float* new_state, void* output, void* stream) {
  const char* name = "m4rt_attention_step";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    if (!rows) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    const m4rt_rows *q = &rows->q, *k = &rows->k, *v = &rows->v;
    const Shape s{B, 1, H, q->width, v->width, bf16};
    std::string why;
    if (bad_shape(s, 1, la::STEP_THREADS, &why) || bad_rows(q, H, bf16, 0, &why) ||
        bad_rows(k, H, bf16, 0, &why) || bad_rows(v, H, bf16, 0, &why))
      return api_fail(M4MR_EINVAL, at + why);
    if (q->width != k->width) return api_fail(M4MR_EINVAL, at + "q and k disagree in width");
    if (!log_decay || !state || !new_state || !output)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    la::Step a{q->data, k->data, v->data, q->batch_stride, q->head_stride, k->batch_stride,
                     k->head_stride, v->batch_stride, v->head_stride, H / q->heads, H / k->heads,
                     H / v->heads, log_decay, per_token ? H : 0, active, state, new_state, output,
                     scale, B, H, s.N, s.P, 0};
    const uintptr_t states = reinterpret_cast<uintptr_t>(state) |
                             reinterpret_cast<uintptr_t>(new_state);
    if (states % 4) return api_fail(M4MR_EINVAL, at + "states must be aligned to 4 bytes");
    const bool whole = s.P % 4 == 0 && states % 16 == 0;
    while ((1 << a.span) < (whole ? s.P / 4 : s.P)) ++a.span;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return api_launch("attention_step", st, [&] {
      bf16 ? start_step<la::bf16_t>(a, whole, st) : start_step<float>(a, whole, st);
    });
  });
}

}  // extern "C"

// -------------------------------------------------------------- group norm --

namespace {

bool bad_norm(long M, int L, int C, int G, int act, std::string* why) {
  if (M <= 0 || L <= 0 || C <= 0 || G <= 0 || C % G) {
    *why = "M, L and C must be positive and G must divide C";
    return true;
  }
  if ((double)M * L * C > 1e15 || (long)L * C > INT_MAX || C > 1 << 23) {
    *why = "problem too large";
    return true;
  }
  if (act < gn::NONE || act > gn::GELU) {
    *why = "unknown activation";
    return true;
  }
  return false;
}

// Widest piece, in elements, that the channels of a group and the arrays'
// addresses allow.
int norm_vec(int D, int bf16, std::initializer_list<const void*> arrays) {
  uintptr_t at = 0;
  for (const void* p : arrays) at |= reinterpret_cast<uintptr_t>(p);
  const int size = bf16 ? 2 : 4;
  int vec = 16 / size;
  while (vec > 1 && (D % vec || at % (vec * size))) vec >>= 1;
  return vec;
}

// The route of a call: groups within a wave (one position, at most IT pieces a
// lane), or blocks over positions.  Grids depend on the sizes and the card.
struct NormPlan {
  int vec, pieces;  // pieces a lane holds; 0: position kernels
  dim3 grid;
  int threads, part_rows;
  bool whole;       // position kernels: in one launch
  size_t sums;      // floats of their partial statistics
};

NormPlan norm_plan(long M, int L, int C, int G, int vec, gn::Norm* a) {
  NormPlan p{};
  p.vec = vec;
  a->M = M;
  a->L = L;
  a->C = C;
  a->G = G;
  a->D = C / G;
  const int vecs = a->D / vec, cus = m4::api_compute_units();
  if (L == 1) {
    // Fewest idle lanes, then fewest pieces; at most 16 elements a lane.
    int best = 0;
    for (int lanes = 64; lanes >= 1; lanes >>= 1) {
      int pieces = (vecs + lanes - 1) / lanes;
      if (pieces == 3) pieces = 4;
      if (pieces > 4 || pieces * vec > 16) break;
      if (best == 0 || lanes * pieces < a->lanes * best) {
        a->lanes = lanes;
        best = pieces;
      }
    }
    if (best) {
      p.pieces = best;
      a->groups = std::min(G, gn::ROW_THREADS / a->lanes);
      const int across = a->groups * a->lanes;
      a->rows = (int)std::min<long>(gn::ROW_THREADS / across, M);
      p.threads = (a->rows * across + 63) / 64 * 64;
      const long most = (M + a->rows - 1) / a->rows;
      p.grid = dim3((unsigned)std::min<long>(most, 3L * cus), (G + a->groups - 1) / a->groups);
      p.part_rows = (int)p.grid.x;
      return p;
    }
  }
  a->vecs = vecs;
  a->subs = (vecs + gn::POS_THREADS - 1) / gn::POS_THREADS;
  a->span = a->subs > 1 ? 1 : std::min(G, gn::POS_THREADS / vecs);
  a->rows = a->subs > 1 ? 1 : std::max(1, std::min(L, gn::POS_THREADS / (vecs * a->span)));
  const int slots = (G * a->subs + a->span - 1) / a->span;
  // Parts of the positions, of 8 rows a thread up to 8 parts and of 16 beyond: they
  // depend on the sample alone, since the order of its sums does.  16 / 8 rows, forward
  // us: M1 L4000 C64 bfloat16 (3 / 7 parts) 24 / 17, M512 L196 C512 float32 (3 / 6, one
  // launch) 108 / 111, M8 L4000 C512 float32 (62 / 125) 39 / 51.
  const long rows = L / a->rows;
  a->parts = (int)std::max<long>(
      1, std::min<long>((2L * cus + slots - 1) / slots, std::max(std::min(8L, rows / 8), rows / 16)));
  if (a->subs > 1 && a->parts == 1) a->parts = std::min(L, 2);
  // A block takes a part, or whole samples where those are blocks enough for the card.
  p.whole = a->subs == 1 && (a->parts == 1 || M * slots >= 2L * cus);
  const int blocks = p.whole ? 1 : a->parts;
  // Blocks walk over samples past these (the column sums have a part for each).
  const long samples = std::min<long>(M, std::max(1L, 4L * cus / ((long)slots * blocks)));
  p.grid = dim3(blocks, (unsigned)samples, slots);
  p.threads = gn::POS_THREADS;
  p.part_rows = (int)samples * blocks;
  p.sums = a->parts == 1 && a->subs == 1 ? 0 : (size_t)M * a->parts * a->subs * G * 4;
  return p;
}

template <typename In, int V, int IT, bool BWD>
void start_rows(const gn::Norm& a, const NormPlan& p, hipStream_t st) {
  if constexpr (V * IT <= 16)
    hipLaunchKernelGGL((gn::norm_rows_kernel<In, V, IT, BWD>), p.grid, dim3(p.threads), 0, st, a);
}

template <typename In, int V, bool BWD>
void start_norm(const gn::Norm& a, const NormPlan& p, int phase, hipStream_t st) {
  if (p.pieces == 1) return start_rows<In, V, 1, BWD>(a, p, st);
  if (p.pieces == 2) return start_rows<In, V, 2, BWD>(a, p, st);
  if (p.pieces == 4) return start_rows<In, V, 4, BWD>(a, p, st);
  const dim3 block(p.threads);
  if (phase == gn::SUMS)
    hipLaunchKernelGGL((gn::norm_positions_kernel<In, V, BWD, gn::SUMS>), p.grid, block, 0, st, a);
  else if (phase == gn::APPLY)
    hipLaunchKernelGGL((gn::norm_positions_kernel<In, V, BWD, gn::APPLY>), p.grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((gn::norm_positions_kernel<In, V, BWD, gn::BOTH>), p.grid, block, 0, st, a);
}

template <bool BWD>
void launch_norm(const gn::Norm& a, const NormPlan& p, int bf16, int phase, hipStream_t st) {
  if (bf16) {
    if (p.vec == 8) return start_norm<gn::bf16_t, 8, BWD>(a, p, phase, st);
    if (p.vec == 4) return start_norm<gn::bf16_t, 4, BWD>(a, p, phase, st);
    if (p.vec == 2) return start_norm<gn::bf16_t, 2, BWD>(a, p, phase, st);
    return start_norm<gn::bf16_t, 1, BWD>(a, p, phase, st);
  }
  if (p.vec == 4) return start_norm<float, 4, BWD>(a, p, phase, st);
  if (p.vec == 2) return start_norm<float, 2, BWD>(a, p, phase, st);
  return start_norm<float, 1, BWD>(a, p, phase, st);
}

template <bool BWD>
int run_norm(const gn::Norm& a, const NormPlan& p, int bf16, hipStream_t st) {
  const char* name = BWD ? "norm_backward" : "norm";
  if (p.pieces || p.whole)
    return api_launch(name, st, [&] { launch_norm<BWD>(a, p, bf16, gn::BOTH, st); });
  int rc = api_launch(BWD ? "norm_backward_sums" : "norm_sums", st,
                      [&] { launch_norm<BWD>(a, p, bf16, gn::SUMS, st); });
  if (rc) return rc;
  return api_launch(name, st, [&] { launch_norm<BWD>(a, p, bf16, gn::APPLY, st); });
}

bool misaligned(int bf16, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % (bf16 ? 2 : 4)) return true;
  return false;
}

// The largest workspace over the widths of the pieces, which depend on
// addresses.
size_t norm_workspace(long M, int L, int C, int G, int bf16, bool backward) {
  size_t most = 0;
  for (int vec = bf16 ? 8 : 4; vec >= 1; vec >>= 1) {
    if ((C / G) % vec) continue;
    gn::Norm a{};
    const NormPlan p = norm_plan(M, L, C, G, vec, &a);
    const size_t part = backward ? align256((size_t)p.part_rows * 2 * C * sizeof(float)) : 0;
    most = std::max(most, part + align256(p.sums * sizeof(float)));
  }
  return most;
}

}  // namespace

extern "C" {

size_t m4rt_norm_workspace_bytes(long M, int L, int C, int G, int bf16, int backward) {
  std::string why;
  if (bad_norm(M, L, C, G, gn::NONE, &why)) return 0;
  return norm_workspace(M, L, C, G, bf16, backward);
}

int m4rt_norm_forward(const void* x, const float* weight, const float* bias, const void* gate,
                      int bf16, long M, int L, int C, int G, int activation, float eps, void* y,
                      float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4rt_norm_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_norm(M, L, C, G, activation, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!x || !y)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(bf16, {x, gate, y}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    if (bad_workspace(workspace, workspace_bytes, norm_workspace(M, L, C, G, bf16, false), &why))
      return api_fail(M4MR_EINVAL, at + why);
    gn::Norm a{};
    const NormPlan p = norm_plan(M, L, C, G, norm_vec(C / G, bf16, {x, gate, y}), &a);
    a.x = x;
    a.gate = gate;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.eps = eps;
    a.act = activation;
    a.stats = stats;
    a.sums = static_cast<float*>(workspace);
    return run_norm<false>(a, p, bf16, static_cast<hipStream_t>(stream));
  });
}

int m4rt_norm_backward(const void* x, const float* weight, const float* bias, const void* gate,
                       const void* d_output, const float* stats, int bf16, long M, int L, int C,
                       int G, int activation, float eps, void* d_x, float* d_weight, float* d_bias,
                       void* d_gate, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4rt_norm_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_norm(M, L, C, G, activation, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!x || !d_output || !stats)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(bf16, {x, gate, d_output, d_x, d_gate}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    if (bad_workspace(workspace, workspace_bytes, norm_workspace(M, L, C, G, bf16, true), &why))
      return api_fail(M4MR_EINVAL, at + why);
    gn::Norm a{};
    const NormPlan p =
        norm_plan(M, L, C, G, norm_vec(C / G, bf16, {x, gate, d_output, d_x, d_gate}), &a);
    Carver c{static_cast<char*>(workspace)};
    const bool columns = d_weight || d_bias;
    a.x = x;
    a.gate = gate;
    a.dy = d_output;
    a.weight = weight;
    a.bias = bias;
    a.dx = d_x;
    a.dgate = gate ? d_gate : nullptr;
    a.eps = eps;
    a.act = activation;
    a.stats = const_cast<float*>(stats);
    float* part = c.take<float>((size_t)p.part_rows * 2 * C);
    a.part = columns ? part : nullptr;
    a.sums = c.take<float>(p.sums);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = run_norm<true>(a, p, bf16, st);
    if (rc || !columns) return rc;
    return api_launch("norm_columns", st, [&] {
      hipLaunchKernelGGL(gn::norm_columns_kernel, dim3((2 * C + 15) / 16), dim3(1024), 0, st, part,
                         p.part_rows, C, d_weight, d_bias);
    });
  });
}

}  // extern "C"

// --------------------------------------------------------------- embedding --

namespace {

bool bad_embedding(long n, int rows, int width, std::string* why) {
  if (n <= 0 || rows <= 0 || width <= 0) {
    *why = "the tokens, rows and width must be positive";
    return true;
  }
  if (n > INT_MAX - (1 << 24) || rows > INT_MAX - 1 || (double)n * width > 1e12 ||
      (double)rows * width > 1e12) {
    *why = "problem too large";
    return true;
  }
  return false;
}

// Whether `blocks` of em::THREADS are more than a launch takes: under 2^32 threads.
bool bad_blocks(long blocks, std::string* why) {
  if (blocks < (1L << 32) / em::THREADS) return false;
  *why = "problem too large";
  return true;
}

int embedding_vec(int width, std::initializer_list<const void*> arrays) {
  uintptr_t at = 0;
  for (const void* p : arrays) at |= reinterpret_cast<uintptr_t>(p);
  int vec = 8;
  // 16-byte pieces of bfloat16, two of float32.
  while (vec > 1 && (width % vec || at % std::min(16, 4 * vec))) vec >>= 1;
  return vec;
}

// The backward's sort and chunks, and its workspace.
struct EmbeddingPlan {
  int passes, bits, tile, tiles, chunk, chunks;
  unsigned* counts[4];
  unsigned char* present;
  unsigned *keys[2], *tokens[2];
  float *head, *tail;
  size_t cleared;  // words from counts[1] on that the passes add up
};

size_t embedding_plan(long n, int rows, int width, void* base, EmbeddingPlan* p) {
  int bits = 1;
  while (bits < 32 && (unsigned)rows >> bits) ++bits;  // keys are 0..rows
  p->passes = (bits + em::MAX_DIGIT - 1) / em::MAX_DIGIT;
  p->bits = (bits + p->passes - 1) / p->passes;
  // Every tile reads all tiles' counts: at most 128 of them.
  p->tile = 1024;
  while ((n + p->tile - 1) / p->tile > 128) p->tile *= 2;
  p->tiles = (int)((n + p->tile - 1) / p->tile);
  // Short chunks fill the card, long ones leave fewer parts to join: sums + joins in
  // us in chunks of 16 and 64, of tokens of 768 into a float32 table: 4,096 22 + 8 and
  // 30 + 7, 16,384 24 + 12 and 29 + 8, 32,768 27 + 19 and 28 + 9; of 1,024 bfloat16:
  // 65,536 39 + 32 and 38 + 12, 131,071 84 + 64 and 82 + 20.
  p->chunk = n >= 65536 ? 64 : 16;
  p->chunks = (int)((n + p->chunk - 1) / p->chunk);
  Carver c{static_cast<char*>(base)};
  size_t first = 0;
  for (int i = 0; i < p->passes; ++i) {
    p->counts[i] = c.take<unsigned>((size_t)p->tiles << p->bits);
    if (i == 0) first = c.used;
  }
  p->present = c.take<unsigned char>(rows);
  p->cleared = (c.used - first) / sizeof(unsigned);
  for (int i = 0; i < 2; ++i) {
    // (Padded: a batch of rows may end past the last.)
    p->keys[i] = c.take<unsigned>(n + em::AHEAD);
    p->tokens[i] = c.take<unsigned>(n + em::AHEAD);
  }
  p->head = c.take<float>((size_t)p->chunks * width);
  p->tail = c.take<float>((size_t)p->chunks * width);
  return c.used;
}

// Blocks whose threads take four pieces of `rows` rows each.
long piece_blocks(long rows, int pieces) {
  return (rows * pieces + 4 * em::THREADS - 1) / (4 * em::THREADS);
}

template <typename In, typename Out, int V>
void start_lookup(const em::Lookup& a, hipStream_t st) {
  hipLaunchKernelGGL((em::lookup_kernel<In, Out, V>),
                     dim3((unsigned)piece_blocks(a.n, a.width / V)), dim3(em::THREADS), 0, st, a);
}

template <int V>
void launch_lookup(const em::Lookup& a, int table_bf16, int out_bf16, hipStream_t st) {
  if (table_bf16)
    out_bf16 ? start_lookup<em::bf16_t, em::bf16_t, V>(a, st)
             : start_lookup<em::bf16_t, float, V>(a, st);
  else
    out_bf16 ? start_lookup<float, em::bf16_t, V>(a, st) : start_lookup<float, float, V>(a, st);
}

// Blocks of waves that take 64 pieces of a chunk's columns each.
long chunk_blocks(long chunks, int pieces) {
  constexpr int waves = em::THREADS / 64;
  return (chunks * ((pieces + 63) / 64) + waves - 1) / waves;
}

template <typename In, typename Out, int V>
void start_sums(const em::Sum& a, hipStream_t st) {
  const long sums = chunk_blocks(a.chunks, a.width / V), zeros = piece_blocks(a.rows, a.width / V);
  hipLaunchKernelGGL((em::sum_kernel<In, Out, V>), dim3((unsigned)(sums + zeros)),
                     dim3(em::THREADS), 0, st, a, (unsigned)sums);
}

template <int V>
void launch_sums(const em::Sum& a, int table_bf16, int out_bf16, hipStream_t st) {
  if (table_bf16)
    out_bf16 ? start_sums<em::bf16_t, em::bf16_t, V>(a, st)
             : start_sums<float, em::bf16_t, V>(a, st);
  else
    out_bf16 ? start_sums<em::bf16_t, float, V>(a, st) : start_sums<float, float, V>(a, st);
}

template <int V>
void launch_join(const em::Sum& a, int table_bf16, hipStream_t st) {
  const dim3 grid((unsigned)chunk_blocks(a.chunks, a.width / V));
  if (table_bf16)
    hipLaunchKernelGGL((em::join_kernel<em::bf16_t, V>), grid, dim3(em::THREADS), 0, st, a);
  else
    hipLaunchKernelGGL((em::join_kernel<float, V>), grid, dim3(em::THREADS), 0, st, a);
}

#define EM_BY_VEC(vec, call)                 \
  do {                                       \
    if ((vec) == 8) call<8> EM_ARGS;         \
    else if ((vec) == 4) call<4> EM_ARGS;    \
    else if ((vec) == 2) call<2> EM_ARGS;    \
    else call<1> EM_ARGS;                    \
  } while (0)

}  // namespace

extern "C" {

int m4rt_embedding_forward(const void* ids, int ids_int64, const void* table, int table_bf16,
                           long n, int rows, int width, float scale, void* output, int output_bf16,
                           void* stream) {
  const char* name = "m4rt_embedding_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_embedding(n, rows, width, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!ids || !table || !output)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(table_bf16, {table}) || misaligned(output_bf16, {output}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    const em::Lookup a{ids, ids_int64, table, output, n, rows, width, scale};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int vec = embedding_vec(width, {table, output});
    if (bad_blocks(piece_blocks(n, width / vec), &why)) return api_fail(M4MR_EINVAL, at + why);
    return api_launch("embedding", st, [&] {
#define EM_ARGS (a, table_bf16, output_bf16, st)
      EM_BY_VEC(vec, launch_lookup);
#undef EM_ARGS
    });
  });
}

size_t m4rt_embedding_workspace_bytes(long n, int rows, int width) {
  std::string why;
  if (bad_embedding(n, rows, width, &why)) return 0;
  EmbeddingPlan p{};
  return embedding_plan(n, rows, width, nullptr, &p);
}

int m4rt_embedding_backward(const void* ids, int ids_int64, const void* d_output, int output_bf16,
                            long n, int rows, int width, float scale, void* d_table,
                            int table_bf16, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const char* name = "m4rt_embedding_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    std::string why;
    if (bad_embedding(n, rows, width, &why)) return api_fail(M4MR_EINVAL, at + why);
    if (!ids || !d_output || !d_table)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    if (misaligned(table_bf16, {d_table}) || misaligned(output_bf16, {d_output}))
      return api_fail(M4MR_EINVAL, at + "arrays must be aligned to their elements");
    EmbeddingPlan p{};
    if (bad_workspace(workspace, workspace_bytes, embedding_plan(n, rows, width, workspace, &p),
                      &why))
      return api_fail(M4MR_EINVAL, at + why);
    const int vec = embedding_vec(width, {d_output, d_table});
    if (bad_blocks(chunk_blocks(p.chunks, width / vec) + piece_blocks(rows, width / vec), &why))
      return api_fail(M4MR_EINVAL, at + why);
    hipStream_t st = static_cast<hipStream_t>(stream);
    em::Sort sort{};
    sort.ids = ids;
    sort.wide = ids_int64;
    sort.n = n;
    sort.rows = rows;
    sort.tile = p.tile;
    sort.tiles = p.tiles;
    sort.bits = p.bits;
    const em::Clear clear{reinterpret_cast<unsigned*>(p.passes > 1
                                                          ? reinterpret_cast<char*>(p.counts[1])
                                                          : reinterpret_cast<char*>(p.present)),
                          (long)p.cleared};
    int rc = api_launch("embedding_count", st, [&] {
      hipLaunchKernelGGL(em::count_kernel, dim3(p.tiles), dim3(em::THREADS), 0, st, sort,
                         p.counts[0], clear);
    });
    if (rc) return rc;
    for (int i = 0; i < p.passes; ++i) {
      const bool last = i + 1 == p.passes;
      sort.keys = i ? p.keys[(i - 1) & 1] : nullptr;
      sort.tokens = i ? p.tokens[(i - 1) & 1] : nullptr;
      sort.out_keys = p.keys[i & 1];
      sort.out_tokens = p.tokens[i & 1];
      sort.counts = p.counts[i];
      sort.next = last ? nullptr : p.counts[i + 1];
      sort.present = last ? p.present : nullptr;
      sort.shift = i * p.bits;
      sort.next_shift = sort.shift + p.bits;
      sort.next_bits = p.bits;
      rc = api_launch("embedding_scatter", st, [&] {
        hipLaunchKernelGGL(em::scatter_kernel, dim3(p.tiles), dim3(em::THREADS), 0, st, sort);
      });
      if (rc) return rc;
    }
    const int sorted = (p.passes - 1) & 1;
    const em::Sum sum{p.keys[sorted], p.tokens[sorted], p.present, d_output, d_table,
                      p.head, p.tail, n, rows, width, p.chunk, p.chunks, scale};
    rc = api_launch("embedding_sums", st, [&] {
#define EM_ARGS (sum, table_bf16, output_bf16, st)
      EM_BY_VEC(vec, launch_sums);
#undef EM_ARGS
    });
    if (rc) return rc;
    return api_launch("embedding_join", st, [&] {
#define EM_ARGS (sum, table_bf16, st)
      EM_BY_VEC(vec, launch_join);
#undef EM_ARGS
    });
  });
}

}  // extern "C"

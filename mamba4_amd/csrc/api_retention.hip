// C ABI of the retention layer's operators (include/mamba4_retention.h): the
// checks of the arguments and the launches.
#include <climits>
#include <cstdlib>
#include <cstring>

#include "../../include/mamba4_retention.h"
#include "api_common.hpp"
#include "linattn.hpp"

namespace la {
template <typename In, int NT, bool OUT>
__global__ void attention_kernel(Args);
__global__ void carry_kernel(Args);
__global__ void decay_grad_kernel(DecayGrad);
__global__ void decay_heads_kernel(const double*, int, int, float*);
template <typename Out>
__global__ void share_sum_kernel(const float*, long, int, int, int, Out*);
template <typename In>
__global__ void step_kernel(Step);
}  // namespace la

namespace {

using m4::api_fail;
using m4::api_launch;

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Consecutive pieces of one workspace (sizes only, if base is NULL).
struct Carver {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += align256(count * sizeof(T));
    return p;
  }
};

bool bad_workspace(const void* base, size_t given, size_t need, std::string* why) {
  if (need == 0) return false;
  if (!base || given < need) {
    *why = "workspace too small";
    return true;
  }
  if (reinterpret_cast<uintptr_t>(base) & 255) {
    *why = "workspace must be 256-byte aligned";
    return true;
  }
  return false;
}

// ------------------------------------------------------ linear attention --

struct Shape {
  int B, T, H, N, P, bf16;
  int chunks() const { return (T + la::C - 1) / la::C; }
  int segments() const { return (chunks() + la::SEG - 1) / la::SEG; }
};

bool bad_shape(const Shape& s, std::string* why) {
  if (s.B <= 0 || s.T <= 0 || s.H <= 0) {
    *why = "B, T and H must be positive";
    return true;
  }
  if (s.N <= 0 || s.P <= 0 || s.N > M4RT_MAX_WIDTH || s.P > M4RT_MAX_WIDTH) {
    *why = "key and value widths must be in 1.." + std::to_string(M4RT_MAX_WIDTH);
    return true;
  }
  // Grids: blocks of at most six tiles a (b, h), segments along y.
  if ((double)s.B * s.H * 6 + 64 > INT_MAX / 2 || s.segments() > 65535 || s.T > INT_MAX - 4096) {
    *why = "problem too large";
    return true;
  }
  return false;
}

int tiles_of(int width) { return (width + la::TILE - 1) / la::TILE; }

// Whether the sequences are split into segments (their states formed first,
// then carried, then all walked at once) instead of walked from end to end.
// M4RT_ATTENTION = "walk" or "split" overrides the choice; the bits are the same.
bool attention_splits(const Shape& s, int blocks) {
  if (s.segments() < 2) return false;
  if (const char* mode = std::getenv("M4RT_ATTENTION")) {
    if (std::strcmp(mode, "walk") == 0) return false;
    if (std::strcmp(mode, "split") == 0) return true;
  }
  return (long)s.B * s.H * blocks < 2L * m4::api_compute_units();
}

// A split run's states of one role (n keys wide, `tiles` blocks of values).
void take_states(Carver& c, const Shape& s, int n, int tiles, bool split, la::Role* role) {
  const size_t slots = split ? (size_t)tiles * s.B * s.H * s.segments() : 0;
  role->starts = c.take<float>(slots * tiles_of(n) * la::TILE * la::TILE);
  role->decays = c.take<float>(slots);
}

// Rows as the kernels take them: how many elements a load may take at once
// (16 bytes, or the 4 of a bfloat16 pair, else one element).
la::Rows rows_of(const m4rt_rows& r, int H, int bf16) {
  la::Rows x{r.data, r.batch_stride, r.token_stride, r.head_stride, H / r.heads, r.width, 1};
  const uintptr_t at = reinterpret_cast<uintptr_t>(r.data);
  const int size = bf16 ? 2 : 4;
  for (int vec : {16 / size, 4 / size}) {
    if (at % (vec * size) == 0 && r.batch_stride % vec == 0 && r.token_stride % vec == 0 &&
        r.head_stride % vec == 0 && r.width % vec == 0) {
      x.vec = vec;
      break;
    }
  }
  return x;
}

bool bad_rows(const m4rt_rows* r, int H, int bf16, bool tokens, std::string* why) {
  if (!r || !r->data) {
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
  if (tokens && (r->token_stride < r->width || r->token_stride > INT_MAX / (4 * la::C))) {
    *why = "a token stride must be at least the width, and 64 of it below 2^31 bytes";
    return true;
  }
  return false;
}

m4rt_rows dense(const void* data, int T, int H, int width) {
  return m4rt_rows{data, (long)T * H * width, (long)H * width, width, H, width};
}

int wide_keys(const la::Args& a) {
  for (int i = 0; i < a.roles; ++i)
    if (a.role[i].n > 64) return 2;
  return 1;
}

template <typename In, int NT, bool OUT>
void start_attention(const la::Args& a, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((la::attention_kernel<In, NT, OUT>), grid, dim3(la::THREADS), 0, st, a);
}

template <bool OUT>
void launch_attention(const la::Args& a, int bf16, dim3 grid, hipStream_t st) {
  const int nt = wide_keys(a);
  if (bf16) {
    nt == 1 ? start_attention<la::bf16_t, 1, OUT>(a, grid, st)
            : start_attention<la::bf16_t, 2, OUT>(a, grid, st);
  } else {
    nt == 1 ? start_attention<float, 1, OUT>(a, grid, st)
            : start_attention<float, 2, OUT>(a, grid, st);
  }
}

int run_attention(la::Args& a, const Shape& s, bool split, hipStream_t st) {
  a.blocks = 0;
  for (int i = 0; i < a.roles; ++i) a.blocks += a.role[i].tiles;
  a.B = s.B;
  a.T = s.T;
  a.H = s.H;
  a.NC = s.chunks();
  a.NS = s.segments();
  const unsigned x = (unsigned)((s.B * s.H + 7) / 8 * 8 * a.blocks);
  if (split) {
    int rc = api_launch("attention_states", st,
                        [&] { launch_attention<false>(a, s.bf16, dim3(x, a.NS), st); });
    if (rc) return rc;
    rc = api_launch("attention_carry", st, [&] {
      hipLaunchKernelGGL(la::carry_kernel, dim3(x, 4 * wide_keys(a)), dim3(la::THREADS), 0, st, a);
    });
    if (rc) return rc;
  }
  return api_launch("attention", st, [&] {
    launch_attention<true>(a, s.bf16, dim3(x, split ? a.NS : 1), st);
  });
}

struct Backward {
  la::Role role[3];
  float *part[3], *dots_q, *dots_k;
  double* head;
};

int backward_tiles(const Shape& s) { return 2 * tiles_of(s.N) + tiles_of(s.P); }

// The backward's workspace: split states, float32 gradients of shared heads
// before their sums, the dots, the heads' sums.
size_t backward_workspace(const Shape& s, const int heads[3], void* base, Backward* out) {
  Carver c{static_cast<char*>(base)};
  const int n[3] = {s.P, s.P, s.N}, p[3] = {s.N, s.N, s.P};
  const size_t rows = (size_t)s.B * s.T * s.H;
  const bool split = attention_splits(s, backward_tiles(s));
  for (int i = 0; i < 3; ++i) {
    take_states(c, s, n[i], tiles_of(p[i]), split, &out->role[i]);
    out->part[i] = c.take<float>(heads[i] == s.H ? 0 : rows * p[i]);
  }
  out->dots_q = c.take<float>(rows * tiles_of(s.N));
  out->dots_k = c.take<float>(rows * tiles_of(s.N));
  out->head = c.take<double>((size_t)s.B * s.H);
  return c.used;
}

}  // namespace

extern "C" {

size_t m4rt_attention_workspace_bytes(int B, int T, int H, int N, int P, int bf16) {
  const Shape s{B, T, H, N, P, bf16};
  std::string why;
  if (bad_shape(s, &why)) return 0;
  Carver c{nullptr};
  la::Role role{};
  take_states(c, s, N, tiles_of(P), attention_splits(s, tiles_of(P)), &role);
  return c.used;
}

int m4rt_attention_forward(const m4rt_rows* q, const m4rt_rows* k, const m4rt_rows* v, int bf16,
                           const float* log_decay, int per_token, const int* lengths,
                           const float* initial, float scale, int B, int T, int H, void* output,
                           float* state, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4rt_attention_forward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    const Shape s{B, T, H, q ? q->width : 0, v ? v->width : 0, bf16};
    std::string why;
    if (bad_shape(s, &why) || bad_rows(q, H, bf16, true, &why) || bad_rows(k, H, bf16, true, &why) ||
        bad_rows(v, H, bf16, true, &why))
      return api_fail(M4MR_EINVAL, at + why);
    if (q->width != k->width) return api_fail(M4MR_EINVAL, at + "q and k disagree in width");
    if (!log_decay || !output) return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    la::Args a{};
    la::Role& r = a.role[0];
    const bool split = attention_splits(s, tiles_of(s.P));
    Carver c{static_cast<char*>(workspace)};
    take_states(c, s, s.N, tiles_of(s.P), split, &r);
    if (bad_workspace(workspace, workspace_bytes, c.used, &why))
      return api_fail(M4MR_EINVAL, at + why);
    r.q = rows_of(*q, H, bf16);
    r.k = rows_of(*k, H, bf16);
    r.v = rows_of(*v, H, bf16);
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
    return run_attention(a, s, split, static_cast<hipStream_t>(stream));
  });
}

size_t m4rt_attention_backward_workspace_bytes(int B, int T, int H, int q_heads, int k_heads,
                                               int v_heads, int N, int P, int bf16) {
  const Shape s{B, T, H, N, P, bf16};
  const int heads[3] = {q_heads, k_heads, v_heads};
  std::string why;
  if (bad_shape(s, &why)) return 0;
  Backward w{};
  return backward_workspace(s, heads, nullptr, &w);
}

int m4rt_attention_backward(const m4rt_rows* q, const m4rt_rows* k, const m4rt_rows* v, int bf16,
                            const float* log_decay, int per_token, const int* lengths,
                            const float* initial, float scale, int B, int T, int H,
                            const void* d_output, const float* d_state, const float* state,
                            void* d_q, void* d_k, void* d_v, float* d_log_decay, float* d_initial,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "m4rt_attention_backward";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    const Shape s{B, T, H, q ? q->width : 0, v ? v->width : 0, bf16};
    std::string why;
    if (bad_shape(s, &why) || bad_rows(q, H, bf16, true, &why) || bad_rows(k, H, bf16, true, &why) ||
        bad_rows(v, H, bf16, true, &why))
      return api_fail(M4MR_EINVAL, at + why);
    if (q->width != k->width) return api_fail(M4MR_EINVAL, at + "q and k disagree in width");
    if (!log_decay || !d_output || !d_q || !d_k || !d_v || (d_state && d_log_decay && !state))
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    const int heads[3] = {q->heads, k->heads, v->heads};
    Backward w{};
    const size_t need = backward_workspace(s, heads, workspace, &w);
    if (bad_workspace(workspace, workspace_bytes, need, &why))
      return api_fail(M4MR_EINVAL, at + why);
    const m4rt_rows cot = dense(d_output, T, H, s.P);
    const la::Rows rq = rows_of(*q, H, bf16), rk = rows_of(*k, H, bf16),
                   rv = rows_of(*v, H, bf16), ro = rows_of(cot, H, bf16);
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
    rdq.q = ro, rdq.k = rv, rdq.v = rk;
    rdk.q = rv, rdk.k = ro, rdk.v = rq;
    rdv.q = rk, rdv.k = rq, rdv.v = ro;
    rdq.initial = la::States{const_cast<float*>(initial), 1, s.P};
    rdk.initial = la::States{const_cast<float*>(d_state), 1, s.P};
    rdv.initial = la::States{const_cast<float*>(d_state), s.P, 1};
    rdv.final = la::States{d_initial, s.P, 1};
    if (d_log_decay) {
      rdq.e = rq, rdq.dots = w.dots_q;
      rdk.e = rk, rdk.dots = w.dots_k;
    }
    a.roles = 3;
    a.g = log_decay;
    a.gb = per_token ? (long)T * H : 0;
    a.gt = per_token ? H : 0;
    a.lengths = lengths;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = run_attention(a, s, attention_splits(s, backward_tiles(s)), st);
    if (rc) return rc;
    for (int i = 0; i < 3; ++i) {
      if (heads[i] == H) continue;
      const long count = (long)B * T * heads[i] * a.role[i].p;
      rc = api_launch("attention_share", st, [&] {
        const dim3 grid((unsigned)((count + 255) / 256));
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
    d.tiles_q = d.tiles_k = tiles_of(s.N);
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
      hipLaunchKernelGGL(la::decay_grad_kernel, dim3(B * H), dim3(1024), 0, st, d);
    });
    if (rc || per_token) return rc;
    return api_launch("attention_heads", st, [&] {
      hipLaunchKernelGGL(la::decay_heads_kernel, dim3((H + 63) / 64), dim3(64), 0, st, w.head, B, H,
                         d_log_decay);
    });
  });
}

int m4rt_attention_step(const m4rt_rows* q, const m4rt_rows* k, const m4rt_rows* v, int bf16,
                        const float* log_decay, int per_token, const uint8_t* active, float scale,
                        int B, int H, const float* state, float* new_state, void* output,
                        void* stream) {
  const char* name = "m4rt_attention_step";
  return m4::api_entry(name, [&] {
    const std::string at = std::string(name) + ": ";
    const Shape s{B, 1, H, q ? q->width : 0, v ? v->width : 0, bf16};
    std::string why;
    if (bad_shape(s, &why) || bad_rows(q, H, bf16, false, &why) ||
        bad_rows(k, H, bf16, false, &why) || bad_rows(v, H, bf16, false, &why))
      return api_fail(M4MR_EINVAL, at + why);
    if (q->width != k->width) return api_fail(M4MR_EINVAL, at + "q and k disagree in width");
    if (!log_decay || !state || !new_state || !output)
      return api_fail(M4MR_EINVAL, at + "a required pointer is NULL");
    const la::Step a{q->data, k->data, v->data, q->batch_stride, q->head_stride, k->batch_stride,
                     k->head_stride, v->batch_stride, v->head_stride, H / q->heads, H / k->heads,
                     H / v->heads, log_decay, per_token ? H : 0, active, state, new_state, output,
                     scale, B, H, s.N, s.P};
    hipStream_t st = static_cast<hipStream_t>(stream);
    return api_launch("attention_step", st, [&] {
      if (bf16)
        hipLaunchKernelGGL(la::step_kernel<la::bf16_t>, dim3(B * H), dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL(la::step_kernel<float>, dim3(B * H), dim3(256), 0, st, a);
    });
  });
}

}  // extern "C"

// Embedding lookup with a scale, and its gradient by sorted tokens, for gfx950.
//
//   out_i = scale table[id_i],   dtable[r] = scale * sum of dy_i over id_i = r.
// An id outside the table gives a zero row and adds to none.
//
// The lookup moves rows in 16-byte pieces.  The gradient sorts the tokens by
// id (stable, so that a row's terms are added in the order of the tokens and the
// bits are the same on every run), then cuts the sorted tokens into chunks of
// equal length, however often an id occurs: each chunk sums its runs of equal
// ids in float32 and stores the rows that begin and end in it; parts of rows
// that span chunks are joined by a last kernel in order, a row's by one wave for each 64
// pieces.  Rows of ids that do not occur are zeroed by the same launch as the sums.
//
// Sort: passes of at most 9 bits over tiles of tokens.  A pass's tile counts are
// complete before it starts (the first pass's by the counting kernel, the next
// one's added up by the scatter before it, integers, so in any order); each
// tile sums the counts that precede it itself, which spares the scans their own
// launches.
#include <hip/hip_runtime.h>

#include "embed.hpp"

namespace em {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned pack(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}
__device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// V consecutive elements: as loaded, and as float32; written rounded.
template <typename T, int V>
struct Piece;
template <int V>
struct Piece<float, V> {
  typedef float raw __attribute__((ext_vector_type(V)));
  raw r;
  __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const raw*>(p); }
  __device__ __forceinline__ float get(int i) const { return r[i]; }
  __device__ __forceinline__ void touch() {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float x = r[i];
      asm volatile("" : "+v"(x));
      r[i] = x;
    }
  }
};
template <int V>
struct Piece<bf16_t, V> {
  typedef unsigned raw __attribute__((ext_vector_type(V / 2)));
  raw r;
  __device__ __forceinline__ void load(const bf16_t* p) { r = *reinterpret_cast<const raw*>(p); }
  __device__ __forceinline__ float get(int i) const {
    return i & 1 ? high(r[i / 2]) : low(r[i / 2]);
  }
  __device__ __forceinline__ void touch() {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      unsigned x = r[i];
      asm volatile("" : "+v"(x));
      r[i] = x;
    }
  }
};
template <>
struct Piece<bf16_t, 1> {
  bf16_t r;
  __device__ __forceinline__ void load(const bf16_t* p) { r = *p; }
  __device__ __forceinline__ float get(int) const { return __uint_as_float((unsigned)r << 16); }
  __device__ __forceinline__ void touch() {
    unsigned x = r;
    asm volatile("" : "+v"(x));
    r = (bf16_t)x;
  }
};
template <int V>
__device__ __forceinline__ void write(float* p, const float (&v)[V]) {
  typedef float raw __attribute__((ext_vector_type(V)));
  raw r;
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = v[i];
  *reinterpret_cast<raw*>(p) = r;
}
template <int V>
__device__ __forceinline__ void write(bf16_t* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = (bf16_t)pack(v[0], 0.f);
  } else {
    typedef unsigned raw __attribute__((ext_vector_type(V / 2)));
    raw r;
#pragma unroll
    for (int i = 0; i < V; i += 2) r[i / 2] = pack(v[i], v[i + 1]);
    *reinterpret_cast<raw*>(p) = r;
  }
}

// The id of token i, or `rows` for one outside the table.
__device__ __forceinline__ unsigned key_of(const void* ids, int wide, long i, int rows) {
  const long id = wide ? static_cast<const long*>(ids)[i] : (long)static_cast<const int*>(ids)[i];
  return id >= 0 && id < rows ? (unsigned)id : (unsigned)rows;
}

// Each thread moves four pieces, 256 apart, of the block's 1024.  Bound by memory:
// 131,071 rows of 1,024 bfloat16 75 us (268 MB written, 3.6 TB/s, as much read, the
// frequent rows from the caches).
template <typename In, typename Out, int V>
__global__ __launch_bounds__(THREADS) void lookup_kernel(Lookup a) {
  const int vecs = a.width / V;
  const long first = (long)blockIdx.x * (4 * THREADS), row0 = first / vecs;
  const unsigned rest = (unsigned)(first - row0 * vecs);
  const In* table = static_cast<const In*>(a.table);
  Out* out = static_cast<Out*>(a.out);
  // Every load is issued before the first use, unknown ids' from row 0.
  Piece<In, V> x[4];
  long at[4];
  bool known[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned item = rest + threadIdx.x + THREADS * j, step = item / vecs;
    const unsigned v = item - step * vecs;
    const long i = row0 + step;
    at[j] = i < a.n ? i * a.width + v * V : -1;
    const unsigned key = key_of(a.ids, a.wide, min(i, a.n - 1), a.rows);
    known[j] = key < (unsigned)a.rows;
    x[j].load(table + (long)(known[j] ? key : 0) * a.width + v * V);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (at[j] < 0) continue;
    float y[V];
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = known[j] ? x[j].get(e) * a.scale : 0.f;
    write<V>(out + at[j], y);
  }
}

// Tile counts of the first pass's digits; clears what the passes add up.
__global__ __launch_bounds__(THREADS) void count_kernel(Sort a, unsigned* counts, Clear clear) {
  __shared__ unsigned bins[BINS];
  const int size = 1 << a.bits;
  for (int d = threadIdx.x; d < size; d += THREADS) bins[d] = 0;
  for (long i = (long)blockIdx.x * THREADS + threadIdx.x; i < clear.count;
       i += (long)gridDim.x * THREADS)
    clear.words[i] = 0;
  __syncthreads();
  const long first = (long)blockIdx.x * a.tile;
  for (int k = threadIdx.x; k < a.tile; k += THREADS)
    if (first + k < a.n) {
      const unsigned key = key_of(a.ids, a.wide, first + k, a.rows);
      atomicAdd(&bins[(key >> a.shift) & (size - 1)], 1u);
    }
  __syncthreads();
  for (int d = threadIdx.x; d < size; d += THREADS) counts[(long)blockIdx.x * size + d] = bins[d];
}

// Lanes whose digit is this lane's, among the lanes that have one.
__device__ __forceinline__ unsigned long peers(unsigned digit, int bits, bool have) {
  unsigned long mask = __ballot(have);
  for (int b = 0; b < bits; ++b) {
    const unsigned long set = __ballot((digit >> b) & 1);
    mask &= (digit >> b) & 1 ? set : ~set;
  }
  return mask;
}

// One pass: each wave ranks a quarter of the tile in order, 64 pairs at a
// time; equal digits keep their order.  A tile of 64 ROUNDS pairs a wave holds
// them in registers; longer ones repeat that.  Bound by latency: 10 us for 16,384
// tokens, 19 for 131,071.
constexpr int ROUNDS = 4;

__global__ __launch_bounds__(THREADS) void scatter_kernel(Sort a) {
  __shared__ unsigned place[THREADS / 64][BINS], total[2][BINS], before[BINS];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, size = 1 << a.bits;
  const int per = a.tile / (THREADS / 64);
  const long first = (long)blockIdx.x * a.tile + w * per;
  const unsigned long below = (1ul << lane) - 1;
  auto fetch = [&](int k, unsigned (&key)[ROUNDS]) {
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const long i = min(first + k + 64 * j + lane, a.n - 1);
      key[j] = a.keys ? a.keys[i] : key_of(a.ids, a.wide, i, a.rows);
    }
  };
  unsigned key[ROUNDS], rank[ROUNDS];
  unsigned long same[ROUNDS];  // lanes with this lane's digit
  fetch(0, key);
  for (int d = tid; d < (THREADS / 64) * BINS; d += THREADS) (&place[0][0])[d] = 0;
  // This tile's part in the digits: all tiles' counts, and those before it.
  for (int d = tid; d < size; d += THREADS) {
    unsigned all = 0, mine = 0;
#pragma unroll 16
    for (int t = 0; t < a.tiles; ++t) {
      const unsigned c = a.counts[(long)t * size + d];
      all += c;
      mine += t < (int)blockIdx.x ? c : 0;
    }
    total[0][d] = all;
    before[d] = mine;
  }
  __syncthreads();
  // Ranks within the wave's quarter.
  auto count = [&](int k) {
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const bool have = first + k + 64 * j + lane < a.n;
      const unsigned digit = (key[j] >> a.shift) & (size - 1);
      const unsigned long mask = peers(digit, a.bits, have);
      const unsigned seen = __popcll(mask & below);
      same[j] = mask;
      rank[j] = place[w][digit] + seen;
      __builtin_amdgcn_wave_barrier();
      if (have && seen == 0) place[w][digit] += __popcll(mask);
      __builtin_amdgcn_wave_barrier();
    }
  };
  for (int k = 0; k < per; k += 64 * ROUNDS) {
    if (k) fetch(k, key);
    count(k);
  }
  // Exclusive sums of the totals over the digits.
  int from = 0;
  for (int s = 1; s < size; s <<= 1) {
    for (int d = tid; d < size; d += THREADS)
      total[from ^ 1][d] = total[from][d] + (d >= s ? total[from][d - s] : 0);
    from ^= 1;
    __syncthreads();
  }
  for (int d = tid; d < size; d += THREADS) {
    unsigned at = (d > 0 ? total[from][d - 1] : 0) + before[d];
    for (int i = 0; i < THREADS / 64; ++i) {
      const unsigned c = place[i][d];
      place[i][d] = at;
      at += c;
    }
  }
  __syncthreads();
  const bool once = per == 64 * ROUNDS;  // the ranks are still at hand
  for (int k = 0; k < per; k += 64 * ROUNDS) {
    if (!once) {
      fetch(k, key);
      count(k);
    }
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const long i = first + k + 64 * j + lane;
      const bool have = i < a.n;
      const unsigned digit = (key[j] >> a.shift) & (size - 1);
      const unsigned at = once && have ? place[w][digit] + rank[j] : rank[j];
      if (a.next) {
        // One addition for the lanes that share the first one's id and tile: a
        // frequent id's would meet at one address.
        const unsigned tile = at / a.tile;
        const int lead = __ffsll((unsigned long long)same[j]) - 1;
        const unsigned lead_key = __shfl(key[j], lead), lead_tile = __shfl(tile, lead);
        const bool with = have && key[j] == lead_key && tile == lead_tile;
        const unsigned long group = __ballot(with) & same[j];
        unsigned* counter = &a.next[((long)tile << a.next_bits) +
                                    ((key[j] >> a.next_shift) & ((1 << a.next_bits) - 1))];
        if (have && lane == lead) atomicAdd(counter, (unsigned)__popcll(group));
        if (have && !with) atomicAdd(counter, 1u);
      }
      if (!have) continue;
      a.out_keys[at] = key[j];
      a.out_tokens[at] = a.tokens ? a.tokens[i] : (unsigned)i;
      if (a.present && key[j] < (unsigned)a.rows) a.present[key[j]] = 1;
    }
  }
}

// The sorted ids and tokens, which no kernel that reads them so writes.
typedef const __attribute__((address_space(4))) unsigned* Scalars;

// Every load of x is issued before this point: without it the compiler moves
// them to their uses behind branches, one wait each.
template <typename P, int N>
__device__ __forceinline__ void in_flight(P (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i].touch();
}

// A wave's chunk, and the lane's piece of the columns.
struct Place {
  int chunk, piece;
};
__device__ __forceinline__ Place place_of(int vecs) {
  const unsigned slices = (vecs + 63) / 64;
  const unsigned wave =
      __builtin_amdgcn_readfirstlane(blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6));
  const unsigned chunk = wave / slices;
  return Place{(int)chunk, (int)(64 * (wave - chunk * slices) + (threadIdx.x & 63))};
}

// Sums of runs: a wave takes 64 pieces of the columns of one chunk.  The
// blocks from `sum_blocks` on zero the rows that do not occur (blocks of both kinds
// in turn took longer).  Bound by memory: 131,071 rows of 1,024 bfloat16 into 50,257,
// 371 MB in 95 us, 3.9 TB/s.
template <typename In, typename Out, int V>
__global__ __launch_bounds__(THREADS) void sum_kernel(Sum a, unsigned sum_blocks) {
  const int vecs = a.width / V;
  const unsigned rows = (unsigned)a.rows;
  Out* dw = static_cast<Out*>(a.dw);
  if (blockIdx.x >= sum_blocks) {
    const long first = (long)(blockIdx.x - sum_blocks) * (4 * THREADS), row0 = first / vecs;
    const unsigned rest = (unsigned)(first - row0 * vecs);
    const float zero[V] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned item = rest + threadIdx.x + THREADS * j, step = item / vecs;
      const long r = row0 + step;
      if (r < a.rows && !a.present[r]) write<V>(dw + r * a.width + (item - step * vecs) * V, zero);
    }
    return;
  }
  // A wave: 64 pieces of one chunk's columns, so that ids and tokens are scalars.
  const Place at = place_of(vecs);
  if (at.chunk >= a.chunks) return;
  const long chunk = at.chunk;
  const int column = at.piece * V;
  const bool on = at.piece < vecs;
  const In* dy = static_cast<const In*>(a.dy) + (on ? column : 0);
  const Scalars keys = (Scalars)a.keys, tokens = (Scalars)a.tokens;
  const long s = chunk * a.chunk, e = min(s + a.chunk, a.n);
  unsigned current = keys[s];
  bool from_before = s > 0 && keys[s - 1] == current;
  float acc[V] = {};
  auto store = [&](unsigned key) {
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = a.scale * acc[i];
    if (on) write<V>(dw + (long)key * a.width + column, x);
  };
  auto keep = [&](float* parts) {
    if (on) write<V>(parts + chunk * a.width + column, acc);
  };
  // Loads without a condition, so that they are in flight together; what they
  // read past the chunk (the arrays are padded) or for unknown ids is not added.
  for (long i = s; i < e; i += AHEAD) {
    unsigned key[AHEAD];
    Piece<In, V> x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      key[j] = keys[i + j];
      const long token = key[j] < rows ? tokens[i + j] : 0u;
      x[j].load(dy + min(token, a.n - 1) * a.width);
    }
    in_flight(x);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i + j < e && key[j] != current) {
        if (from_before)
          keep(a.head);
        else
          store(current);
        from_before = false;
        current = key[j];
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.f;
      }
      if (i + j < e && current < rows) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += x[j].get(k);
      }
    }
  }
  if (current >= rows) return;
  if (from_before)
    keep(a.head);
  else if (e < a.n && keys[e] == current)
    keep(a.tail);
  else
    store(current);
}

// Rows whose run goes on past the chunk it begins in: its parts in order, so the most
// frequent row sets the time: 131,071 tokens of 1,024 bfloat16 14 us with random ids, 16
// with text's frequencies, 169 with all of one id.
template <typename Out, int V>
__global__ __launch_bounds__(THREADS) void join_kernel(Sum a) {
  const int vecs = a.width / V;
  const Place at = place_of(vecs);
  if (at.chunk >= a.chunks) return;
  const long chunk = at.chunk;
  const bool on = at.piece < vecs;
  const int column = on ? at.piece * V : 0;
  const Scalars keys = (Scalars)a.keys;
  const long s = chunk * a.chunk, e = s + a.chunk;
  if (e >= a.n) return;
  const unsigned key = keys[e - 1];
  if (key >= (unsigned)a.rows || keys[e] != key) return;
  if (s > 0 && keys[s - 1] == key) return;
  Piece<float, V> tail;
  tail.load(a.tail + chunk * a.width + column);
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = tail.get(k);
  // The run's parts, 64 at a time: where it ends, then the sums.
  constexpr int PARTS = 16;
  bool more = true;
  for (long c = chunk + 1; more; c += 64) {
    const long end = (c + (threadIdx.x & 63) + 1) * a.chunk;
    const unsigned then = a.keys[min(end, a.n - 1)];
    const unsigned long goes_on = __ballot(end < a.n && then == key);
    more = ~goes_on == 0;
    const int parts = more ? 64 : __ffsll((unsigned long long)~goes_on);
    for (int first = 0; first < parts; first += PARTS) {
      Piece<float, V> x[PARTS];
#pragma unroll
      for (int j = 0; j < PARTS; ++j)
        x[j].load(a.head + min(c + first + j, (long)a.chunks - 1) * a.width + column);
      in_flight(x);
#pragma unroll
      for (int j = 0; j < PARTS; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k)
          acc[k] = first + j < parts ? acc[k] + x[j].get(k) : acc[k];
    }
  }
  if (!on) return;
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] *= a.scale;
  write<V>(static_cast<Out*>(a.dw) + (long)key * a.width + column, acc);
}

#define EM_TYPES(In, Out, V)                                         \
  template __global__ void lookup_kernel<In, Out, V>(Lookup);        \
  template __global__ void sum_kernel<In, Out, V>(Sum, unsigned);
#define EM_ALL(V)                                            \
  EM_TYPES(float, float, V)                                  \
  EM_TYPES(float, bf16_t, V)                                 \
  EM_TYPES(bf16_t, float, V)                                 \
  EM_TYPES(bf16_t, bf16_t, V)
#define EM_JOIN(V)                                           \
  template __global__ void join_kernel<float, V>(Sum);       \
  template __global__ void join_kernel<bf16_t, V>(Sum);
EM_ALL(8)
EM_ALL(4)
EM_ALL(2)
EM_ALL(1)
EM_JOIN(8)
EM_JOIN(4)
EM_JOIN(2)
EM_JOIN(1)

}  // namespace em

// Arguments of the embedding's kernels, shared by the host entry points and
// embed.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace em {

typedef unsigned short bf16_t;

constexpr int THREADS = 256;
constexpr int AHEAD = 8;               // rows a thread loads at a time
constexpr int MAX_DIGIT = 9;          // bits of a sorting pass
constexpr int BINS = 1 << MAX_DIGIT;  // most bins of a pass

struct Lookup {
  const void* ids;
  int wide;         // ids are int64 (else int32)
  const void* table;
  void* out;
  long n;
  int rows, width;
  float scale;
};

// The sort's passes: pairs (key, token) by the digit of `bits` bits at
// `shift`; tiles of `tile` pairs.
struct Sort {
  const void* ids;       // first pass: the ids themselves
  int wide;
  const unsigned *keys, *tokens;  // later passes
  unsigned *out_keys, *out_tokens;
  const unsigned* counts;  // this pass: [tiles][bins]
  unsigned* next;          // the next pass's counts, added up here, or NULL
  unsigned char* present;  // last pass: ids that occur, or NULL
  long n;
  int rows, tile, tiles;
  int shift, bits, next_shift, next_bits;
};

struct Clear {
  unsigned* words;
  long count;
};

struct Sum {
  const unsigned *keys, *tokens;  // sorted
  const unsigned char* present;
  const void* dy;
  void* dw;
  float *head, *tail;  // [chunks][width] parts of rows that span chunks
  long n;
  int rows, width, chunk, chunks;
  float scale;
};

}  // namespace em

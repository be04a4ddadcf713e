// Internal interface of the 8-bit key/value cache (mnb_kv*.hip).
#pragma once

#include "mnb_kernels.h"
#include "../../include/mnb_kv.h"

#include <algorithm>

namespace mnb {
namespace kv {

struct Cache {
  uint8_t *codes[2];  // keys, values: [pages][heads][page][dim]
  float *scales[2];   // [pages][heads]
  uint32_t pages;
  int32_t heads, page_shift, dim;
};

struct Batch {
  const int32_t *table, *lengths, *starts;
  int32_t sequences, width, tokens, each;  // each: rows of a sequence where starts is NULL
  int32_t max_tokens;
};

struct Rows {
  const void *x;
  int64_t token_stride, head_stride;
};

// The rows of sequence s, in bounds whatever starts and lengths hold.
struct Span {
  int32_t row, count;  // first row, rows: row + count <= tokens
  int32_t first;       // position of the first row, perhaps below 0
  int32_t end;         // behind the last position that a row has and the table reaches
};

__host__ __device__ inline Span SpanOf(const Batch &b, int s, int page_shift) {
  Span r;
  if (b.starts != nullptr) {
    r.row = b.starts[s] < 0 ? 0 : b.starts[s] < b.tokens ? b.starts[s] : b.tokens;
    const int32_t to = b.starts[s + 1] < b.tokens ? b.starts[s + 1] : b.tokens;
    r.count = to > r.row ? to - r.row : 0;
  } else {
    r.row = s * b.each;
    r.count = b.each;
  }
  const int32_t length = b.lengths[s] > 0 ? b.lengths[s] : 0;
  const int32_t reach = b.width << page_shift;
  r.first = length - r.count;
  r.end = length < reach ? length : reach;
  return r;
}

// Ragged sequences share a launch: of workgroups `unit` 0 .. UnitsOf - 1, each sequence
// has those from its first row times `rows`, in blocks of 2^shift, plus `more` for every sequence
// before it. That are no fewer than its own rows touch (more: 1 where they are counted from the
// sequence's first, 2 where blocks lie anywhere), and the launch grows with the
// rows and the sequences, not with their product.
struct Units {
  int32_t rows, shift, more;
};

inline int64_t UnitsOf(const Batch &b, const Units &u) {
  return (static_cast<int64_t>(b.tokens) * u.rows >> u.shift) +
         static_cast<int64_t>(b.sequences) * u.more;
}

#ifdef __HIPCC__
// The sequence that has this unit, and its first one. All lanes of a wavefront call it: they
// look at 64 sequences at a time.
__device__ inline int SequenceOf(const Batch &b, const Units &u, int64_t unit, int64_t *first) {
  const auto from = [&](int s) {
    const int row = min(max(b.starts[s], 0), b.tokens);
    return (static_cast<int64_t>(row) * u.rows >> u.shift) + static_cast<int64_t>(s) * u.more;
  };
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = b.sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const int before = __popcll(__ballot(s < hi && from(min(s, hi - 1)) <= unit));
    lo += max(before - 1, 0) * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  *first = from(lo);
  return lo;
}
#endif

// Page of a sequence's position block p < width, or a number that is no page's.
__host__ __device__ inline uint32_t PageOf(const Batch &b, int s, int p) {
  return static_cast<uint32_t>(b.table[static_cast<int64_t>(s) * b.width + p]);
}

__host__ __device__ inline int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

hipError_t LaunchAppend(const Cache &c, const Batch &b, int32_t x_type, const Rows &k,
                        const Rows &v, hipStream_t s);

struct Attend {
  Cache cache;
  Batch batch;
  Rows q;
  int32_t q_heads;
  float scale;
  int32_t window;  // 0: none
  void *y;         // [tokens][q_heads][dim]
};

size_t AttendWorkBytes(const Cache &c, const Batch &b, int32_t q_heads, int32_t x_type);
hipError_t LaunchAttend(const Attend &a, int32_t x_type, void *work, hipStream_t s);

} // namespace kv
} // namespace mnb

// Attention over the 8-bit key/value cache.
//
// Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T, so that a
// query is a column of every MFMA: lane l of a 16 x 16 result holds rows 4 (l / 16)
// .. + 3 of column l % 16, and the softmax's maximum, sum and rescaling of a query
// are that lane's own. The rows of S^T that a lane holds are the tokens that it
// then supplies as P^T's operand, in whatever order, as long as V^T's operand
// has the same: P stays in its registers.
//
// e4m3 codes are exact in fp16, so the products are fp16 MFMAs on the codes
// themselves. A page's key scale multiplies its scores. Its value scale w goes
// into the exponent: with y = s log2(e) + log2(w) and m near the maximum of y so far,
// P = 2^(y - m + 12) is the token's weight times its value scale, with full fp16
// precision down to 2^-25 of the largest; the sum of the weights alone takes P / w. Then
// O / l needs no further scale. m is the maximum that earlier tiles left, and a factor of 2
// above it, until a tile has weights that fp16 might not hold.
// Queries are scaled by a power of two to below 2^15 and rounded to one fp16 term
// (exact for fp16, and for bf16 down to 2^-31 of the row's largest magnitude) or,
// fp32, to two (22 bits). P is two terms (22 bits) for fp32 and fp16 results: one, of 11
// bits, is as coarse as an fp16 result itself, and made its error 1.4 times its own
// rounding's (2048 tokens over 16384: 733 us, 552 with one; a token of each of 32 sequences
// there 193 and 194). It is one for bf16, whose results have 8 bits: there it adds 1%.
#include "mnb_kv.h"
#include "mnb_values.h"

#include <type_traits>

namespace mnb {
namespace kv {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float floatx16v __attribute__((ext_vector_type(16)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;          // tokens of a step
constexpr int kWaves = 4;          // of a workgroup: each takes every fourth tile of its part
constexpr int kThreads = 64 * kWaves;
constexpr float kInf = __builtin_inff();
constexpr float kShift = 12.0f;    // P is 2^12 where y is m

// The weights' sums count P / w in units of 2^16. P is below 65504 / 4 on average (Fits), so
// 2^30 tokens of the least scale, 2^-100, stay below 2^128, and one of the largest that append
// makes, 2^120, whose P is 2^11, is 2^-125. (An exponent that an instruction can hold: as a
// factor it took two registers more, and 16 drafted tokens of 8 sequences at 16384 121 us for 113.)
__device__ __forceinline__ float InSumUnits(float v) { return ldexpf(v, -16); }

template <typename T>
constexpr int Terms() { return sizeof(T) == 4 ? 2 : 1; }

// Terms of a weight.
template <typename T>
constexpr int WeightTerms() { return std::is_same<T, __bf16>::value ? 1 : 2; }

// Two codes' words -> the eight values, in order.
__device__ __forceinline__ half8v Widen8(uint32_t lo, uint32_t hi) {
  const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(lo), 1.0f, false);
  const half2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(lo), 1.0f, true);
  const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(hi), 1.0f, false);
  const half2v d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(hi), 1.0f, true);
  return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Byte j of out[i] is byte i of in[j]: a 4 x 4 transposition of bytes.
__device__ __forceinline__ void Transpose4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
  const uint32_t ab = __builtin_amdgcn_perm(in[1], in[0], 0x05010400);  // b0 of 0, 1, b1 of 0, 1
  const uint32_t AB = __builtin_amdgcn_perm(in[1], in[0], 0x07030602);  // b2, b3
  const uint32_t cd = __builtin_amdgcn_perm(in[3], in[2], 0x05010400);
  const uint32_t CD = __builtin_amdgcn_perm(in[3], in[2], 0x07030602);
  out[0] = __builtin_amdgcn_perm(cd, ab, 0x05040100);
  out[1] = __builtin_amdgcn_perm(cd, ab, 0x07060302);
  out[2] = __builtin_amdgcn_perm(CD, AB, 0x05040100);
  out[3] = __builtin_amdgcn_perm(CD, AB, 0x07060302);
}

// 0x80 in the place of each NaN code (0x7F or 0xFF), 0 in the others'.
__device__ __forceinline__ uint32_t NanTops(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

// The larger of lanes l and l ^ 32, l and l ^ 16, without a round trip through LDS: of a
// register swapped with itself one result has the lower lanes' values everywhere, the other
// the upper ones'.
__device__ __forceinline__ float MaxHalves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float MaxRows(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The largest of the lanes with the same column of a 16 x 16 result.
__device__ __forceinline__ float MaxGroups(float v) { return MaxHalves(MaxRows(v)); }

__device__ __forceinline__ float SumGroups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ float Exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// A page of zeros may have the scale 0: its values are 0, its tokens weigh what they do.
__device__ __forceinline__ float ValueScale(float w) { return w == 0.0f ? 0x1p-64f : w; }

// log2 of a positive scale: an integer exactly for a power of two.
__device__ __forceinline__ float Log2Scale(float w) {
  int e;
  const float m = frexpf(w, &e);  // w = m 2^e, 0.5 <= m < 1
  return static_cast<float>(e - 1) + log2f(2.0f * m);
}

// What a page's scales add to the scores of its tokens: log2 of the values', or something that
// is not below infinity where they are no numbers (a negative one of values is none).
__device__ __forceinline__ float ScoreAdd(float key, float value) {
  return fabsf(key) < kInf ? Log2Scale(value) : __builtin_nanf("");
}
__device__ __forceinline__ bool NoScale(float add) { return !(add < kInf); }

// The power of two by which a row of queries with this largest magnitude is
// multiplied; fp16 rows are taken as they are.
template <typename T>
__device__ __forceinline__ int QueryShift(uint32_t top) {
  return std::is_same<T, _Float16>::value ? 0 : SplitExponent(__uint_as_float(top), 14);
}

// What turns a dot product of such a row with key codes into log2 of a weight, but for
// the codes' scale. Its sign is in the queries, so that the largest product is the largest
// weight; it is never 0, so that an unseen token's -inf stays that.
__device__ __forceinline__ float QueryScale(float scale, int shift) {
  return ldexpf(fabsf(scale) * 1.44269504f, -shift);
}

__device__ __forceinline__ float ScoreScale(float query, float key) {
  return fmaxf(query * key, 0x1p-126f);
}

template <int TERMS>
__device__ __forceinline__ void SplitQuery(const float (&f)[8], int shift, float sign,
                                           half8v (&q)[TERMS]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = ldexpf(f[e] * sign, shift);
    const _Float16 hi = static_cast<_Float16>(v);
    q[0][e] = hi;
    if constexpr (TERMS == 2) {
      const float rest = v - static_cast<float>(hi);
      q[1][e] = static_cast<_Float16>(rest == rest ? rest : 0.0f);  // an infinity has none
    }
  }
}

// Whether fp16 holds all weights that add up to these sums; a NaN fails too, as it does
// in a row's first tile.
__device__ __forceinline__ bool Fits(const float (&sum)[4]) {
  return fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3])) <= 65504.0f &&
         sum[0] + sum[1] + sum[2] + sum[3] < kInf;
}

__device__ __forceinline__ float FromLane(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// The weights 2^(scale s + add) of eight scores as fp16 terms, and their sum before that rounding:
// beside a page of far larger values a page's weights may be lost for the values'
// sum, but never for their own.
template <int TERMS>
__device__ __forceinline__ float Weights(const float (&s)[8], float scale, float add,
                                         half8v (&p)[TERMS]) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = Exp2(fmaf(s[i], scale, add));
    sum += w;
    const _Float16 hi = static_cast<_Float16>(w);
    p[0][i] = hi;
    if constexpr (TERMS == 2) p[1][i] = static_cast<_Float16>(w - static_cast<float>(hi));
  }
  return sum;
}

// The same number, of which the compiler knows nothing.
__device__ __forceinline__ uint32_t Opaque(uint32_t v) {
  __asm__ volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ half8v ReadLds(uint32_t at) {
  return *(const __attribute__((address_space(3))) half8v *)at;
}

template <typename V>
__device__ __forceinline__ void WriteLds(uint32_t at, V v) {
  *(__attribute__((address_space(3))) V *)at = v;
}

// The tokens that a tile of rows looks at, and how they are shared out.
struct Reach {
  int pmin, pmax;    // positions of its first and last row
  int begin, end;    // tokens, begin a multiple of kTile
};

__device__ __forceinline__ Reach ReachOf(const Span &span, int rows_first, int rows_last,
                                         int window) {
  Reach r;
  r.pmin = span.first + rows_first;
  r.pmax = span.first + rows_last;
  r.end = min(r.pmax + 1, span.end);
  r.begin = window > 0 && r.pmin >= window ? (r.pmin - window + 1) / kTile * kTile : 0;
  return r;
}

// Parts of rows, of `splits` shares of the keys: sums [dim], maximum and sum of weights.
struct Parts {
  float *sums;
  float2 *ml;
  int splits;
};

// Sequences with at most `few` rows to a cache head are AttendSplitKernel's, whose parts
// lie [split][sequence][few_tokens][q_heads]; the others AttendTileKernel's, [split][token]
// [q_heads].
struct Work {
  Parts part, tile_part;
  int64_t few;
  int32_t few_tokens;
};

// Rows of a sequence to a cache head.
__device__ __forceinline__ int64_t RowsOf(const Attend &a, const Span &span) {
  return static_cast<int64_t>(min(span.count, a.batch.max_tokens)) * (a.q_heads / a.cache.heads);
}

// A row's place among the parts, of split 0, and the distance to the next split's.
__device__ __forceinline__ int64_t PartOf(const Attend &a, const Work &w, int s, int i, int head) {
  return (static_cast<int64_t>(s) * w.few_tokens + i) * a.q_heads + head;
}
__device__ __forceinline__ int64_t PartStep(const Attend &a, const Work &w) {
  return static_cast<int64_t>(a.batch.sequences) * w.few_tokens * a.q_heads;
}
__device__ __forceinline__ int64_t TilePartStep(const Attend &a) {
  return static_cast<int64_t>(a.batch.tokens) * a.q_heads;
}

// Tiles of `per` rows, a power of two, of ragged sequences.
__host__ __device__ inline Units RowUnits(const Cache &c, int q_heads, int per) {
  return {q_heads / c.heads, 31 - __builtin_clz(per), 1};
}

// Few rows: each key and value is read once, by one wavefront, from memory straight into
// the registers that the MFMAs take, with no LDS between; the row's heads and drafted
// tokens share it. DP: head_dim rounded up to 64, 128 or 256; MT: tiles of 16 queries.
// grid (heads x row tiles x splits, sequences), or (row tiles of all sequences x heads x
// splits) where row_tiles is 0. A row is a token's query head of this cache head: row r is
// token r / group, head r % group.
// Memory bounds it: 32 sequences at 16384 tokens, 8 heads of 128, bf16, take 188 us (1.08 GB,
// 5.7 TB/s; a copy reaches 4.7), 16 drafted tokens of 8 sequences there 114 with widening and
// weights in the way, one wavefront on a SIMD and, bf16, 20 spilled registers. One sequence at
// 8192 tokens has a workgroup on each CU, each with two tiles a wavefront: 8.3 us, of which 3.6
// are its bytes'.
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kThreads) void AttendSplitKernel(Attend a, Work work, int row_tiles,
                                                              int64_t unit0) {
  constexpr int kTerms = Terms<T>(), kWeights = WeightTerms<T>();
  constexpr int KS = DP / 64;      // 16-byte pieces of a key that a lane holds
  constexpr int VD = DP / 16;      // values of a token that a lane holds, tiles of O^T
  constexpr int VW = VD / 4;       // the same in words
  const Cache &c = a.cache;
  const int split = blockIdx.x % work.part.splits, rest = blockIdx.x / work.part.splits;
  int s = blockIdx.y, h, tile;
  if (row_tiles > 0) {
    h = rest / row_tiles;
    tile = rest - h * row_tiles;
  } else {  // units of ragged sequences
    h = rest % c.heads;
    const int64_t unit = unit0 + rest / c.heads;
    int64_t first;
    s = SequenceOf(a.batch, RowUnits(a.cache, a.q_heads, 16 * MT), unit, &first);
    tile = static_cast<int>(unit - first);
    if (tile < 0) return;
  }
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span span = SpanOf(a.batch, s, c.page_shift);
  const int group = a.q_heads / c.heads;
  const int64_t rows = RowsOf(a, span);
  const int64_t row0 = static_cast<int64_t>(tile) * (16 * MT);
  if (row0 >= rows || rows > work.few) return;
  const int64_t row1 = min(row0 + 16 * MT, rows) - 1;
  const Reach reach = ReachOf(span, static_cast<int>(row0 / group), static_cast<int>(row1 / group),
                              a.window);
  const int tiles = reach.end > reach.begin ? (reach.end - reach.begin + kTile - 1) / kTile : 0;
  const int each = (tiles + work.part.splits - 1) / work.part.splits;
  const int tile1 = min(tiles, (split + 1) * each);

  // Queries. A lane's values for the two MFMAs of piece j are the halves of 16
  // neighbouring ones, as its codes of a key are.
  half8v q[MT][KS][2][kTerms];
  float cq[MT];   // what turns a dot product with key codes into log2 weights
  int pos[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t r = row0 + 16 * t + col;
    const bool there = r < rows;
    const int i = there ? static_cast<int>(r / group) : 0;
    const int g = there ? static_cast<int>(r - static_cast<int64_t>(i) * group) : 0;
    pos[t] = there ? span.first + i : -1;
    const T *x = static_cast<const T *>(a.q.x) + (span.row + i) * a.q.token_stride +
                 (h * group + g) * a.q.head_stride;
    float f[KS][2][8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int d = 64 * j + 16 * grp + 8 * half;
        Load8<T, true>(x + d, there ? c.dim - d : 0, f[j][half]);
        top = max(top, TopBits(f[j][half]));
      }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
    const int shift = QueryShift<T>(top);
    cq[t] = QueryScale(a.scale, shift);
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        SplitQuery<kTerms>(f[j][half], shift, sign, q[t][j][half]);
  }

  floatx4v o[MT][VD];
  float m[MT], l[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    m[t] = -kInf;
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < VD; ++d) o[t][d] = floatx4v{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // A tile is four groups of 16 tokens, each of one page; lanes 16 j .. look up group j's
  // page and scales. Keys are asked for as soon as the last tile's are multiplied,
  // values likewise, into the same registers, and pages a tile earlier.
  uint4v kw[4][KS];
  uint32_t vw[4][4][VW];
  uint32_t id[4];  // pages of what kw holds or will hold, ~0 for none
  float sk = 1.0f, sv = 1.0f;
  const uint32_t dim = c.dim, slots = (1u << c.page_shift) - 1;
  const uint32_t head = static_cast<uint32_t>(h << c.page_shift) * dim;
  const uint32_t apart = static_cast<uint32_t>(c.heads << c.page_shift) * dim;
  const int32_t *table = a.batch.table + static_cast<int64_t>(s) * a.batch.width;
  // Past head_dim the query is 0: any of a key's codes will do; and rows of O^T lie there
  // that are not stored.
  uint32_t koff[KS];
#pragma unroll
  for (int j = 0; j < KS; ++j)
    koff[j] = col * dim + (64 * j + 16 * grp < dim ? 64 * j + 16 * grp : 0);
  const uint32_t voff = 4 * grp * dim + (VD * col < dim ? VD * col : 0);
  const auto find = [&](int step) {
    const int tok = reach.begin + kTile * step + 16 * grp;
    const uint32_t page = table[min(tok, reach.end - 1) >> c.page_shift];
    return step < tile1 && tok < reach.end && page < c.pages ? page : ~0u;
  };
  const auto spread = [&](uint32_t page) {
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) id[sub] = __builtin_amdgcn_readlane(page, 16 * sub);
  };
  const auto where = [&](int step, int sub) {  // codes before a group's; page 0's for none
    const uint32_t slot = (reach.begin + kTile * step + 16 * sub) & slots;
    return static_cast<int64_t>(id[sub] != ~0u ? id[sub] : 0) * apart + (head + slot * dim);
  };
  const auto load_keys = [&](int step) {
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      const uint8_t *k = c.codes[0] + where(step, sub);
#pragma unroll
      for (int j = 0; j < KS; ++j) kw[sub][j] = *reinterpret_cast<const uint4v *>(k + koff[j]);
    }
  };
  const auto load_values = [&](int step) {
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      const uint8_t *v = c.codes[1] + where(step, sub);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(v + (voff + i * dim));
#pragma unroll
        for (int x = 0; x < VW; ++x) vw[sub][i][x] = w[x];
      }
    }
  };
  const auto load_scales = [&](uint32_t page) {
    const int64_t at = static_cast<int64_t>(page != ~0u ? page : 0) * c.heads + h;
    sk = c.scales[0][at];
    sv = c.scales[1][at];
  };
  int step = split * each + wave;
  uint32_t page = ~0u, next = ~0u;  // this lane's group's, of this and the next tile
  if (step < tile1) {
    page = find(step);
    next = find(step + kWaves);
    spread(page);
    load_keys(step);
    load_scales(page);
    load_values(step);
  }
  for (; step < tile1; step += kWaves) {
    const int t0 = reach.begin + kTile * step;
    floatx4v acc[MT][4];
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t][sub] = floatx4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const half8v kf = Widen8(kw[sub][j][2 * half], kw[sub][j][2 * half + 1]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
              acc[t][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[t][j][half][term],
                                                                   acc[t][sub], 0, 0, 0);
        }
    }
    // The scales' part in scores and weights, made by the lanes that hold them.
    const bool there = page != ~0u;
    const float value = ValueScale(sv);
    const float lane_ks = there ? sk : 1.0f;
    float lane_ev = there ? ScoreAdd(sk, value) : -kInf;
    float lane_inv = there ? InSumUnits(1.0f / value) : 0.0f;
    // Some row does not see some token.
    const bool edge = !__all(there) || t0 + kTile - 1 > reach.pmin || t0 + kTile > reach.end ||
                      (a.window > 0 && t0 <= reach.pmax - a.window);
    // Scales that are no numbers reach the rows that see their tokens, through the scores.
    const uint64_t none = edge ? __ballot(NoScale(lane_ev)) : 0;
    if (none != 0 && NoScale(lane_ev)) lane_ev = lane_inv = 0.0f;
    float ks[4], ev[4], inv[4];
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      ks[sub] = FromLane(lane_ks, 16 * sub);
      ev[sub] = FromLane(lane_ev, 16 * sub);
      inv[sub] = FromLane(lane_inv, 16 * sub);
    }
    const bool more = step + kWaves < tile1;
    if (more) {
      spread(next);
      load_keys(step + kWaves);
      load_scales(next);
    }
    page = next;
    // Before the next values: loads end in their order, and the wait for this one must
    // not be one for those.
    if (more) next = find(step + 2 * kWaves);

    half8v p[MT][2][kWeights];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (edge) {
        const int hi = min(pos[t], reach.end - 1) - (t0 + 4 * grp);
        const int lo = a.window > 0 ? pos[t] - a.window - (t0 + 4 * grp) : -64;
#pragma unroll
        for (int sub = 0; sub < 4; ++sub)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = 16 * sub + i;
            const bool seen = tok <= hi && tok > lo && ev[sub] != -kInf;
            acc[t][sub][i] = seen ? acc[t][sub][i] : -kInf;
          }
        __asm__ volatile("");  // a branch, not selects
        if (none != 0) {
#pragma unroll
          for (int sub = 0; sub < 4; ++sub)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((none >> (16 * sub) & 1) != 0 && acc[t][sub][i] != -kInf)
                acc[t][sub][i] = __builtin_nanf("");
        }
      }
      float scale[4], part[4];
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) scale[sub] = ScoreScale(cq[t], ks[sub]);
      const auto make = [&](float top) {
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
          const float add = ev[sub] - top + kShift;
          part[sub] = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = Exp2(fmaf(acc[t][sub][i], scale[sub], add));
            part[sub] += w;
            const _Float16 hi = static_cast<_Float16>(w);
            p[t][sub >> 1][0][4 * (sub & 1) + i] = hi;
            if constexpr (kWeights == 2)
              p[t][sub >> 1][1][4 * (sub & 1) + i] =
                  static_cast<_Float16>(w - static_cast<float>(hi));
          }
        }
      };
      make(m[t]);
      if (__any(!Fits(part))) {
        float top = -kInf;
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
          const float most = fmaxf(fmaxf(acc[t][sub][0], acc[t][sub][1]),
                                   fmaxf(acc[t][sub][2], acc[t][sub][3]));
          top = fmaxf(top, fmaf(most, scale[sub], ev[sub]));
        }
        top = fmaxf(m[t], MaxGroups(top) + 1.0f);
        const float use = top == -kInf ? 0.0f : top;
        const float alpha = Exp2(m[t] - use);
        m[t] = top;
        make(use);
        l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < VD; ++d) o[t][d] *= alpha;
      }
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) l[t] = fmaf(part[sub], inv[sub], l[t]);
    }

#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {
      if (edge) {
        // A weight of 0 does not undo a NaN: values of tokens that no row sees are
        // cleared, and NaN values that some rows may see are kept apart.
        uint32_t nan = 0;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = t0 + 32 * pair + 16 * x + 4 * grp + i;
            const bool seen = tok < reach.end && ev[2 * pair + x] != -kInf &&
                              (a.window == 0 || tok > reach.pmin - a.window);
#pragma unroll
            for (int y = 0; y < VW; ++y) {
              vw[2 * pair + x][i][y] = seen ? vw[2 * pair + x][i][y] : 0u;
              nan |= NanTops(vw[2 * pair + x][i][y]);
            }
          }
        if (__any(nan != 0)) {
          half8v seen[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                seen[t][4 * x + i] = acc[t][2 * pair + x][i] == -kInf
                                         ? static_cast<_Float16>(0.0f)
                                         : static_cast<_Float16>(1.0f);
#pragma unroll
          for (int y = 0; y < VW; ++y) {
            uint32_t flag[2][4], turned[2][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t &w = vw[2 * pair + x][i][y];
                const uint32_t bytes = (NanTops(w) >> 7) * 0xFFu;
                w &= ~bytes;
                flag[x][i] = bytes & 0x38383838u;  // 1.0
              }
              Transpose4(flag[x], turned[x]);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const half8v f = Widen8(turned[0][b], turned[1][b]);
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                floatx4v count = {0.0f, 0.0f, 0.0f, 0.0f};
                count = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, seen[t], count, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (count[i] > 0.0f) o[t][4 * y + b][i] = __builtin_nanf("");
              }
            }
          }
        }
      }
#pragma unroll
      for (int y = 0; y < VW; ++y) {
        uint32_t turned[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t in[4] = {vw[2 * pair + x][0][y], vw[2 * pair + x][1][y],
                                  vw[2 * pair + x][2][y], vw[2 * pair + x][3][y]};
          Transpose4(in, turned[x]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const half8v vf = Widen8(turned[0][b], turned[1][b]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int term = 0; term < kWeights; ++term)
              o[t][4 * y + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[t][pair][term],
                                                                       o[t][4 * y + b], 0, 0, 0);
        }
      }
    }
    if (more) load_values(step + kWaves);
  }

  // The wavefronts' parts, one tile of 16 rows at a time. A lane holds values VD (4 grp
  // + i) + d of its row.
  __shared__ float sums[kWaves][16][DP + 4];
  __shared__ float2 ml[kWaves][16];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const float total = SumGroups(l[t]);
    if (t > 0) __syncthreads();
    if (grp == 0) ml[wave][col] = make_float2(m[t], total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < VD; d += 4) {
        floatx4v v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[t][d + e][i];
        *reinterpret_cast<floatx4v *>(&sums[wave][col][VD * (4 * grp + i) + d]) = v;
      }
    __syncthreads();
    // Sixteen threads to a row, VD values each.
    const int r = threadIdx.x >> 4, d0 = VD * (threadIdx.x & 15);
    const int64_t row = row0 + 16 * t + r;
    if (row >= rows || d0 >= c.dim) continue;
    float top = -kInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w][r].x);
    const float use = top == -kInf ? 0.0f : top;
    float sum = 0.0f, v[VD];
#pragma unroll
    for (int d = 0; d < VD; ++d) v[d] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (ml[w][r].y == 0.0f) continue;  // saw nothing
      const float by = Exp2(ml[w][r].x - use);
      sum = fmaf(ml[w][r].y, by, sum);
#pragma unroll
      for (int d = 0; d < VD; ++d) v[d] = fmaf(sums[w][r][d0 + d], by, v[d]);
    }
    const int i = static_cast<int>(row / group), g = static_cast<int>(row - static_cast<int64_t>(i) * group);
    const int64_t at = static_cast<int64_t>(span.row + i) * a.q_heads + h * group + g;
    if (work.part.splits == 1) {
      const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
      T *y = static_cast<T *>(a.y) + at * c.dim + d0;
#pragma unroll
      for (int d = 0; d < VD; ++d) y[d] = static_cast<T>(InSumUnits(v[d]) * by);
    } else {
      const int64_t part = PartOf(a, work, s, i, h * group + g) + split * PartStep(a, work);
      if (d0 == 0) work.part.ml[part] = make_float2(top, sum);
      float *y = work.part.sums + part * c.dim + d0;
      if (sum != 0.0f)
#pragma unroll
        for (int d = 0; d < VD; ++d) y[d] = v[d];
    }
  }
}

// Many rows: 32 queries to a wavefront, NW wavefronts to a workgroup, on tiles of 64
// tokens that the workgroup widens to fp16 once, in LDS, for all of them. MFMAs of
// 32 x 32 halve what a product reads of LDS; V is laid out transposed, in the order
// of tokens that a lane's weights have. The next tile's codes are in registers
// while a tile is multiplied, and are widened into the other half of LDS.
// grid (row tiles x splits x heads, sequences), or (row tiles of all sequences x splits x
// heads) where row_tiles is 0: heads lie next to each other, so that a
// head's workgroups share an XCD's cache where there are eight; late rows, which see
// the most keys, come first.
// The matrix instructions bound it: 2048 bf16 tokens of 32 heads of 128 over 16384 keys take
// 549 us, 0.94 PFLOP/s (a large library product reaches 1.2). The weights, their exponentials
// first, take nearly as long as a tile's products, and run on the SIMD's other wavefront
// meanwhile; with the halves of a workgroup not half a step apart it took 772.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void AttendTileKernel(Attend a, Work work, int row_tiles,
                                                             int64_t unit0) {
  constexpr int kTerms = Terms<T>(), kWeights = WeightTerms<T>();
  constexpr int kThreadsT = 64 * NW;
  constexpr int KP = DP / 16;                  // 16-code pieces of a key, steps of Q K^T
  constexpr int DT = DP / 32;                  // tiles of O^T
  constexpr int kUnits = 4 * DP;               // 16-byte pieces of a tile's keys, of its values
  constexpr int kEach = (kUnits + kThreadsT - 1) / kThreadsT;
  constexpr int kMask = DP / 8 < 16 ? DP / 8 - 1 : 15;
  const Cache &c = a.cache;
  const int h = blockIdx.x % a.cache.heads, rest = blockIdx.x / a.cache.heads;
  const int split = rest % work.tile_part.splits;
  int s = blockIdx.y, late = rest / work.tile_part.splits;  // tiles behind this one
  if (row_tiles == 0) {  // units of ragged sequences
    const int64_t unit = unit0 + late;
    int64_t first;
    s = SequenceOf(a.batch, RowUnits(a.cache, a.q_heads, 32 * NW), unit, &first);
    late = static_cast<int>(unit - first);
  }
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Span span = SpanOf(a.batch, s, c.page_shift);
  const int group = a.q_heads / c.heads;
  const int64_t rows = RowsOf(a, span);
  const int tile = static_cast<int>(CeilDiv(rows, 32 * NW)) - 1 - late;
  if (tile < 0 || late < 0 || rows <= work.few) return;
  const int64_t row0 = static_cast<int64_t>(tile) * (32 * NW);
  const int64_t row1 = min(row0 + 32 * NW, rows) - 1;
  const Reach reach = ReachOf(span, static_cast<int>(row0 / group), static_cast<int>(row1 / group),
                              a.window);
  const int tiles = reach.end > reach.begin ? (reach.end - reach.begin + kTile - 1) / kTile : 0;
  const int each = (tiles + work.tile_part.splits - 1) / work.tile_part.splits;
  const int tile0 = split * each, tile1 = min(tiles, tile0 + each);

  // Two tiles of keys, [token][unit ^ token], and two of values, [d][unit ^ (d / 4) ^ d],
  // units of eight values: neighbouring lanes' units lie in different banks.
  constexpr uint32_t kHalf = kTile * DP * 2;
  __shared__ __attribute__((aligned(256))) uint8_t tiles_of[4 * kHalf];
  // Of 16 tokens: the keys' scale, log2 and inverse (in sum units) of the values'.
  __shared__ float4 info[4][4];
  // NaN values are kept apart: a tile's tokens that have one, by d, and whether any has.
  // Four tiles' records, for one is made while readers of others are behind.
  __shared__ uint32_t nans[4][DP][2], any_nan[4];

  const uint32_t base = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)tiles_of));

  // This wavefront's rows.
  const int64_t r0 = row0 + 32 * wave, r = r0 + col;
  const bool there = r < rows;
  const int i0 = there ? static_cast<int>(r / group) : 0;
  const int g = there ? static_cast<int>(r - static_cast<int64_t>(i0) * group) : 0;
  const int pos = there ? span.first + i0 : -1;
  const int pmin = __builtin_amdgcn_readfirstlane(span.first + static_cast<int>(r0 / group));
  const int pmax = __builtin_amdgcn_readfirstlane(
      span.first + static_cast<int>(min(r0 + 31, rows - 1) / group));
  half8v q[KP][kTerms];
  float cq;
  {
    const T *x = static_cast<const T *>(a.q.x) + (span.row + i0) * a.q.token_stride +
                 (h * group + g) * a.q.head_stride;
    float f[KP][8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KP; ++j) {
      const int d = 16 * j + 8 * half;
      Load8<T, true>(x + d, there ? c.dim - d : 0, f[j]);
      top = max(top, TopBits(f[j]));
    }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
    const int shift = QueryShift<T>(top);
    cq = QueryScale(a.scale, shift);
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int j = 0; j < KP; ++j) SplitQuery<kTerms>(f[j], shift, sign, q[j]);
  }

  // What a thread brings of each tile: 16 codes of a key, four of four tokens' values. All
  // that a wavefront brings at a time is of one group of 16 tokens, and so of one page.
  // Values are brought a tile later than keys, when their weights are made.
  uint4v kw[kEach];
  uint32_t vw[kEach][4];
  uint32_t id[kEach];                           // page of the group's next keys; ~0: none
  uint32_t kid[kEach], vid[kEach];              // of the keys and the values that are held
  int64_t kfrom[kEach], vfrom[kEach];           // where their group begins
  float sk[kEach], sv[kEach];                   // the keys' page's scales
  int grp[kEach];
  uint32_t koff[kEach], voff[kEach], kto[kEach], vto[kEach];
  const uint32_t dim = c.dim, slots = (1u << c.page_shift) - 1;
  const int64_t head = static_cast<int64_t>(h << c.page_shift) * dim;
  const int32_t *table = a.batch.table + static_cast<int64_t>(s) * a.batch.width;
  // The index of a vector load whose address is the same in all lanes: a scalar load
  // would be waited for with the next read of LDS.
  const uint32_t lane0 = Opaque(0);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const uint32_t u = tid + k * kThreadsT;
    grp[k] = __builtin_amdgcn_readfirstlane(u / DP);
    kid[k] = vid[k] = ~0u;
    kfrom[k] = vfrom[k] = 0;
    const uint32_t kt = u / KP, kd = 16 * (u % KP), quad = u / (DP / 4), vd = 4 * (u % (DP / 4));
    koff[k] = kt % 16 * dim + (kd < dim ? kd : 0);
    voff[k] = 4 * (quad % 4) * dim + (vd < dim ? vd : 0);
    // The key's second unit is its first ^ 1. Four tokens 4 quad .. of a group of 16 are the
    // first or the second half of the eight that a lane with half = quad % 2 has
    // weights of; value vd + e goes e rows further, to unit ^ e.
    kto[k] = (kt * (DP / 8) + (2 * (u % KP) ^ (kt & kMask))) * 16;
    vto[k] = 2 * kHalf + 8 * (quad / 2 % 2) +
             16 * (vd * (kTile / 8) + ((2 * (quad / 4) + quad % 2) ^ (((vd >> 2) ^ vd) & 7)));
  }
  const auto find = [&](int n) {  // the pages of tile n
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int tok = reach.begin + kTile * n + 16 * grp[k];
      const int32_t *at = table + (min(tok, reach.end - 1) >> c.page_shift);
      id[k] = tok < reach.end ? at[lane0] : ~0u;
    }
  };
  const auto load_keys = [&](int n) {  // and their scales; of page 0 where there are none
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      vid[k] = kid[k];
      vfrom[k] = kfrom[k];
      kid[k] = __builtin_amdgcn_readfirstlane(id[k]);
      const uint32_t page = kid[k] < c.pages ? kid[k] : 0;
      const uint32_t slot = (reach.begin + kTile * n + 16 * grp[k]) & slots;
      kfrom[k] = static_cast<int64_t>(page) * (static_cast<uint32_t>(c.heads << c.page_shift) * dim) +
                 head + slot * dim;
      if (kUnits % kThreadsT != 0 && grp[k] >= 4) break;
      kw[k] = *reinterpret_cast<const uint4v *>(c.codes[0] + kfrom[k] + koff[k]);
      if ((64 * wave + k * kThreadsT) % DP == 0) {
        const int64_t at = static_cast<int64_t>(page) * c.heads + h;
        sk[k] = c.scales[0][at + lane0];
        sv[k] = c.scales[1][at + lane0];
      }
    }
  };
  const auto load_values = [&]() {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (kUnits % kThreadsT != 0 && grp[k] >= 4) break;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vw[k][e] = *reinterpret_cast<const uint32_t *>(c.codes[1] + vfrom[k] + (voff[k] + e * dim));
    }
  };
  const auto store_keys = [&](int n) {  // into half n & 1 of the keys' LDS
    const uint32_t off = base + (n & 1 ? kHalf : 0);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (kUnits % kThreadsT != 0 && grp[k] >= 4) break;
      const bool good = kid[k] < c.pages;
      if (!good) kw[k] = uint4v{0, 0, 0, 0};  // no NaN: the info's -inf does the rest
      WriteLds(off + kto[k], Widen8(kw[k][0], kw[k][1]));
      WriteLds((off + kto[k]) ^ 16, Widen8(kw[k][2], kw[k][3]));
      if ((64 * wave + k * kThreadsT) % DP == 0 && lane == 0) {
        const float value = ValueScale(sv[k]);
        info[n & 3][grp[k]] =
            good ? make_float4(sk[k], ScoreAdd(sk[k], value), InSumUnits(1.0f / value), 0.0f)
                 : make_float4(1.0f, -kInf, 0.0f, 0.0f);
      }
    }
  };
  const auto store_values = [&](int n) {
    const int t0 = reach.begin + kTile * n;
    const uint32_t off = base + (n & 1 ? kHalf : 0);
    const bool part_seen = t0 + kTile > reach.end || (a.window > 0 && t0 <= reach.pmin - a.window);
    // Some rows see a token that others do not: elsewhere NaN may go the way of all values.
    const bool mixed = t0 + kTile - 1 > reach.pmin ||
                       (a.window > 0 && t0 <= reach.pmax - a.window);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (kUnits % kThreadsT != 0 && grp[k] >= 4) break;
      // A weight of 0 does not undo a NaN: values of tokens that no row sees are cleared.
      const bool good = vid[k] < c.pages;
      if (part_seen || !good) {
        const uint32_t u = Opaque(tid) + k * kThreadsT;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = t0 + static_cast<int>(4 * (u / (DP / 4))) + e;
          const bool seen = good && tok < reach.end &&
                            (a.window == 0 || tok > reach.pmin - a.window);
          vw[k][e] = seen ? vw[k][e] : 0u;
        }
      }
      uint32_t nan = 0;
      if (mixed)
        nan = NanTops(vw[k][0]) | NanTops(vw[k][1]) | NanTops(vw[k][2]) | NanTops(vw[k][3]);
      if (nan != 0) {
        const uint32_t u = Opaque(tid) + k * kThreadsT;
        any_nan[n & 3] = 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t tops = NanTops(vw[k][e]);
          const int tok = 4 * (u / (DP / 4)) + e;
#pragma unroll 1
          for (int x = 0; x < 4; ++x)
            if ((tops >> (8 * x)) & 0x80u)
              atomicOr(&nans[n & 3][4 * (u % (DP / 4)) + x][tok >> 5], 1u << (tok & 31));
          vw[k][e] &= ~((tops >> 7) * 0xFFu);
        }
      }
      uint32_t turned[4];
      Transpose4(vw[k], turned);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const half2v lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(turned[e]), 1.0f,
                                                                   false);
        const half2v hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(turned[e]), 1.0f,
                                                                   true);
        WriteLds(((off + vto[k]) ^ (16 * e)) + e * (kTile * 2), half4v{lo[0], lo[1], hi[0], hi[1]});
      }
    }
  };
  const auto clear = [&](int n) {  // the record of tile n's NaN, by one wavefront
    for (int d = lane; d < DP; d += 64) nans[n & 3][d][0] = nans[n & 3][d][1] = 0;
    any_nan[n & 3] = 0;
  };

  floatx16v o[DT], sc[2];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  half8v p[4][kWeights];
  float m = -kInf, l = 0.0f;

  // Where this lane reads: the other tokens, values and half lie at constant distances.
  uint32_t kat[KP], vat[4];
#pragma unroll
  for (int k = 0; k < KP; ++k)
    kat[k] = base + (col * (DP / 8) + ((2 * k + half) ^ (col & kMask))) * 16;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    vat[j] = base + 2 * kHalf +
             (col * (kTile / 8) + ((2 * j + half) ^ (((col >> 2) ^ col) & 7))) * 16;

  // sc = K(n) Q^T and o += V(n - 1)^T P^T, or the first alone. Left to itself the compiler
  // waits for each operand when it reads it (40 MFMAs' time); here kAhead are on their way.
  const auto multiply = [&](auto values, int n) {
    constexpr int kFirst = 2 * KP, kAll = kFirst + (decltype(values)::value ? 4 * DT : 0);
    constexpr int kAhead = 6;
    const uint32_t koff = n & 1 ? kHalf : 0, voff = kHalf - koff;
    half8v x[kAhead];
    const auto read = [&](int i) {
      if (i < kFirst)
        x[i % kAhead] = ReadLds(kat[i >> 1] + koff + (i & 1) * (32 * DP * 2));
      else
        x[i % kAhead] = ReadLds(vat[(i - kFirst) / DT] + voff +
                                (i - kFirst) % DT * (32 * kTile * 2));
    };
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[j][e] = 0.0f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(i);
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i < kFirst) {
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
          sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i % kAhead], q[i >> 1][term],
                                                             sc[i & 1], 0, 0, 0);
      } else {
        const int j = (i - kFirst) / DT, d = (i - kFirst) % DT;
#pragma unroll
        for (int term = 0; term < kWeights; ++term)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i % kAhead], p[j][term], o[d], 0, 0, 0);
      }
      if (i + kAhead < kAll) read(i + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // This lane's row sees token j of tile n, where it is of a page, if low < j <= high.
  const auto high = [&](int n) { return min(pos, reach.end - 1) - (reach.begin + kTile * n); };
  const auto low = [&](int n) {
    return a.window > 0 ? pos - a.window - (reach.begin + kTile * n) : -1;
  };
  const auto weights = [&](int n) {  // p, l and m from sc
    const int t0 = reach.begin + kTile * n;
    float4 in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) in[j] = info[n & 3][j];
    // Whether some row does not see some token.
    if (t0 + kTile - 1 > pmin || t0 + kTile > reach.end ||
        (a.window > 0 && t0 <= pmax - a.window)) {
      const int hi = high(n) - 4 * half, lo = low(n) - 4 * half;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int tok = 32 * j + 8 * (e >> 2) + (e & 3);
          sc[j][e] = tok <= hi && tok > lo ? sc[j][e] : -kInf;
        }
      __asm__ volatile("");  // a branch: as selects this would take as long as the rest
      // Scales that are no numbers reach the rows that see their tokens, through the scores.
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (NoScale(in[j].y)) {
#pragma unroll
          for (int e = 8 * (j & 1); e < 8 * (j & 1) + 8; ++e)
            sc[j >> 1][e] = sc[j >> 1][e] == -kInf ? -kInf : __builtin_nanf("");
          in[j].y = in[j].z = 0.0f;
        }
    }
    float scale[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) scale[j] = ScoreScale(cq, in[j].x);
    float part[4];
    const auto make = [&](float top) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = sc[j >> 1][8 * (j & 1) + e];
        part[j] = Weights<kWeights>(y, scale[j], in[j].y - top + kShift, p[j]);
      }
    };
    make(m);
    if (__any(!Fits(part))) {
      __asm__ volatile("");
      float top = -kInf;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float most = -kInf;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, sc[j >> 1][8 * (j & 1) + e]);
        top = fmaxf(top, fmaf(most, scale[j], in[j].y));
      }
      top = MaxHalves(top) + 1.0f;
      const float next = fmaxf(m, top), use = next == -kInf ? 0.0f : next;
      const float alpha = Exp2(m - use);
      m = next;
      make(use);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) l = fmaf(part[j], in[j].z, l);
    // Made here, not where they are used: there the matrix instructions would wait, and what
    // they are made of would take registers.
    __asm__ volatile("" : "+v"(l));
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int term = 0; term < kWeights; ++term) __asm__ volatile("" : "+v"(p[j][term]));
  };
  const auto spoil = [&](int n) {  // NaN values of tile n, to the rows that see them
    if (any_nan[n & 3] != 0) {
      const auto to = [](int j) {  // the tokens up to j
        return j < 0 ? uint64_t{0} : j >= 63 ? ~uint64_t{0} : (uint64_t{2} << j) - 1;
      };
      const uint64_t seen = to(high(n)) & ~to(low(n));
      const uint32_t sees[2] = {static_cast<uint32_t>(seen), static_cast<uint32_t>(seen >> 32)};
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t *w = nans[n & 3][32 * d + 8 * (e >> 2) + 4 * half + (e & 3)];
          if (((w[0] & sees[0]) | (w[1] & sees[1])) != 0) o[d][e] = __builtin_nanf("");
          __builtin_amdgcn_sched_barrier(0);  // one condition at a time: all would take 128 SGPRs
        }
    }
  };

  if (tile0 < tile1) {
    // Where a SIMD has two of the wavefronts, one multiplies while the other makes
    // weights and widens codes: the second is half a step behind, and so, to be in time
    // for the first, brings its share of a tile a step ahead.
    const bool second = NW == 8 && wave >= 4;
    if (wave == 0)
      for (int n = 0; n < 4; ++n) clear(n);
    find(tile0);
    load_keys(tile0);
    find(tile0 + 1);
    __syncthreads();
    store_keys(tile0);
    load_keys(tile0 + 1);
    load_values();
    find(tile0 + 2);
    int ahead = tile0;
    const auto bring = [&]() {  // the keys of tile ahead + 1, the values of tile ahead
      store_keys(ahead + 1);
      store_values(ahead);
      load_keys(ahead + 2);
      load_values();
      find(ahead + 3);
      ++ahead;
    };
    __syncthreads();
    if (second) {
      bring();
      __syncthreads();
    }
    multiply(std::false_type{}, tile0);
    for (int n = tile0; n < tile1; ++n) {
      __syncthreads();
      weights(n);
      bring();
      if (wave == 0 && any_nan[(n + 2) & 3] != 0) clear(n + 2);
      __syncthreads();
      multiply(std::true_type{}, n + 1);  // the scores of tile1 are not used
      spoil(n);
    }
    if (NW == 8 && !second) __syncthreads();
  }
  if (!there) return;
  l += __shfl_xor(l, 32);
  const int64_t at = static_cast<int64_t>(span.row + i0) * a.q_heads + h * group + g;
  const float by = work.tile_part.splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t part = split * TilePartStep(a) + at;
  if (work.tile_part.splits > 1 && half == 0) work.tile_part.ml[part] = make_float2(m, l);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d0 = 32 * d + 8 * (e >> 2) + 4 * half;
      if (d0 >= c.dim) continue;
      if (work.tile_part.splits > 1) {
        *reinterpret_cast<floatx4v *>(work.tile_part.sums + part * c.dim + d0) =
            floatx4v{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
      } else {
        typedef T Vec __attribute__((ext_vector_type(4)));
        Vec y;
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = static_cast<T>(InSumUnits(o[d][e + x]) * by);
        *reinterpret_cast<Vec *>(static_cast<T *>(a.y) + at * c.dim + d0) = y;
      }
    }
}

// Joins the splits of a row. PER threads to a row, four values of it each; where one
// row has more threads than its width, they take every n-th split. All parts of a row
// are asked for at once: it is bound by two trips to memory, 4 us. A workgroup per row
// (PER 256) is sooner for few rows of many splits (attention of one token over 8192: 11.1 us in
// all, 12.5 with a wavefront), a wavefront (PER 64) for many rows (3500: 37.0, 41.7).
template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void JoinKernel(Attend a, Work work, int64_t row0) {
  const int64_t row = row0 + static_cast<int64_t>(blockIdx.x) * (kThreads / PER) +
                      __builtin_amdgcn_readfirstlane(threadIdx.x / PER);
  const int token = static_cast<int>(row / a.q_heads);
  if (token >= a.batch.tokens) return;  // PER 256: all threads
  int s = 0;
  if (a.batch.starts == nullptr) {
    s = token / a.batch.each;
  } else {  // the last sequence that starts at this token or before
    for (int to = a.batch.sequences; to - s > 1;) {
      const int mid = (s + to) / 2;
      if (a.batch.starts[mid] <= token) s = mid;
      else to = mid;
    }
  }
  const Span span = SpanOf(a.batch, s, a.cache.page_shift);
  const int i = token - span.row;
  if (i < 0 || i >= min(span.count, a.batch.max_tokens)) return;
  const bool tile = RowsOf(a, span) > work.few;
  const Parts &parts = tile ? work.tile_part : work.part;
  const int splits = parts.splits;
  if (splits == 1) return;  // written where it was computed
  const int head = static_cast<int>(row - static_cast<int64_t>(token) * a.q_heads);
  const int64_t at = tile ? row : PartOf(a, work, s, i, head);
  const int64_t step = tile ? TilePartStep(a) : PartStep(a, work);
  const int dim = a.cache.dim, lane = threadIdx.x & 63;
  const int wide = dim <= 64 ? 16 : dim <= 128 ? 32 : 64;  // threads that hold a row
  const int t = threadIdx.x % PER, first = t / wide, stride = PER / wide, d = 4 * (t % wide);
  // Every wavefront finds the maximum: a lane per split, 64 at most.
  float2 ml = lane < splits ? parts.ml[lane * step + at] : make_float2(-kInf, 0.0f);
  float top = ml.x;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float use = top == -kInf ? 0.0f : top;
  const float by = ml.y == 0.0f ? 0.0f : Exp2(ml.x - use);
  float sum = ml.y * by;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
  floatx4v v = {0.0f, 0.0f, 0.0f, 0.0f};
  const float *part = parts.sums + at * dim + (d < dim ? d : 0);
  for (int s0 = 0; s0 < splits; s0 += 4 * stride) {
    floatx4v p[4];  // asked for before it is known which splits saw anything
#pragma unroll
    for (int x = 0; x < 4; ++x)
      p[x] = *reinterpret_cast<const floatx4v *>(
          part + min(s0 + x * stride + first, splits - 1) * step * dim);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i0 = s0 + x * stride + first;
      const float w = __shfl(by, i0 & 63);
      if (i0 >= splits || w == 0.0f) continue;  // it saw nothing, and wrote nothing
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(p[x][e], w, v[e]);
    }
  }
  for (int off = wide; off < 64; off *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], off);
  if constexpr (PER > 64) {
    __shared__ floatx4v sums[PER / 64][64];
    sums[threadIdx.x >> 6][lane] = v;
    __syncthreads();
    if (threadIdx.x >= wide) return;
#pragma unroll
    for (int w = 1; w < PER / 64; ++w) v += sums[w][lane];
  } else if (lane >= wide) {
    return;
  }
  if (d >= dim) return;
  const float over = sum == 0.0f ? 0.0f : 1.0f / sum;
  T *y = static_cast<T *>(a.y) + row * dim + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(InSumUnits(v[e]) * over);
}

// How a call is launched: for sequences of at most `few` rows to a cache head
// AttendSplitKernel with mt tiles of 16, for others AttendTileKernel with `waves`
// wavefronts. Of sequences that all have as many rows only one of the two has any (mt or
// waves is 0), ragged ones may have both.
struct Plan {
  int mt = 0, row_tiles = 0, splits = 1;
  int waves = 0, tile_row_tiles = 0, tile_splits = 1;
  int64_t few = 0;
  int32_t few_tokens = 0;
};

Plan PlanOf(const Cache &c, const Batch &b, int32_t q_heads, int32_t x_type) {
  Plan p;
  const int64_t group = q_heads / c.heads, rows = b.max_tokens * group;
  const bool fp32 = x_type == MNB_TYPE_FLOAT, tiles = c.dim <= 128;
  // Up to 64 rows AttendSplitKernel is as fast as AttendTileKernel over long caches (16 drafted
  // tokens of 8 sequences at 16384: 114 and 112 us) and starts sooner. Two tiles of fp32
  // queries 256 wide leave no registers for the keys.
  const int most_mt = fp32 ? (tiles ? 2 : 1) : tiles ? 4 : 2;
  const int64_t key_tiles = CeilDiv(static_cast<int64_t>(b.width) << c.page_shift, kTile);
  const auto parts = [&](int64_t groups, int64_t goal, int64_t least) {
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(64, key_tiles / least));
    return static_cast<int>(std::min(most, std::max<int64_t>(1, goal / groups)));
  };
  int64_t few = rows;
  if (tiles && rows > 16 * most_mt) {
    // Where ragged sequences are long or short, the short ones are taken to be decoded. Tokens of
    // more than 32 rows are sooner in the launch that there is for the prompts (48 heads on one,
    // 8 sequences at 2000 tokens beside a prompt of 200: 56 us, 65 apart; 64 on each of two, 64
    // sequences at 16000: 517, 715): then nothing is left for AttendSplitKernel, and it is not
    // launched.
    p.few = few = b.starts == nullptr || group > 32 ? 0 : group <= 16 ? 16 : 32;
    // Eight wavefronts share a tile's widening (2048 tokens over 16384: 549 us, 631 with
    // four); 128 rows leave half of them without any (4 x 32 tokens over 8192: 46 us, 58 with
    // eight). fp32 keeps four: ragged calls, few long tiles, gain from narrow ones (a prompt of
    // 200 beside 8 decoded sequences at 2000: 55 us, 76 with eight), prompts alone would from
    // wide ones (1024 tokens over 8192: 358 us, 335; at head_dim 64 227, 176).
    p.waves = rows > 128 && !fp32 ? 8 : 4;
    const int64_t per = 32 * p.waves;
    p.tile_row_tiles = static_cast<int>(CeilDiv(rows, per));
    const int64_t filled = b.starts == nullptr ? b.sequences * p.tile_row_tiles
                                               : CeilDiv(b.tokens * group, per);
    // One workgroup of eight wavefronts fits a CU, or two of four, or one of 128-wide fp32 or
    // fp16 (301 and 259 registers). Four tiles
    // at least are worth a part (32 to 128 tokens of one sequence over 4096: 25 to 33 us, 30 to
    // 36 with eight, 27 to 32 with two); eight of fp32 (128 tokens: 39 us, 51 with four).
    p.tile_splits = parts(filled * c.heads, fp32 || p.waves == 8 ? 256 : 512, fp32 ? 8 : 4);
  } else {
    p.few = INT64_MAX;
  }
  p.few_tokens = static_cast<int32_t>(few / group);
  if (few > 0) {
    p.mt = static_cast<int>(std::min<int64_t>(most_mt, CeilDiv(few, 16)));
    p.row_tiles = static_cast<int>(CeilDiv(few, 16 * p.mt));
    // Three workgroups to a CU, where mt 1 lets two stay at a time and others one: short calls
    // do not depend on it, long ones want as many as stay or fewer, those that divide badly
    // more (for one, two, three and six to a CU, us: 16 drafted tokens of 8 sequences at 16384
    // 80, 96, 114, 127; a token of 32 there 185, 193, 193, 195; of 16 at 8192 and head_dim 256,
    // 16 heads on 4, 51, 56, 62, 87; of 12 at 8192 43, 40, 39, 41). A part's sums are as large
    // as mt tiles of keys for each of its wavefronts.
    p.splits = parts(static_cast<int64_t>(b.sequences) * c.heads * p.row_tiles, 3 * 256,
                     kWaves * p.mt);
  }
  return p;
}

// Ragged sequences' units, `each` workgroups to one, so many at a time that a grid's
// threads stay below 2^32.
template <typename L>
hipError_t InUnits(const Attend &a, const Units &u, unsigned each, const L &launch) {
  const int64_t units = UnitsOf(a.batch, u), most = (1 << 22) / each;
  for (int64_t i = 0; i < units; i += most) {
    const hipError_t e = launch(dim3(each * static_cast<unsigned>(std::min(most, units - i))), 0, i);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int DP, int MT>
hipError_t Split(const Attend &a, const Work &w, const Plan &p, hipStream_t s) {
  const unsigned each = static_cast<unsigned>(a.cache.heads) * p.splits;
  const auto launch = [&](dim3 grid, int row_tiles, int64_t unit0) {
    hipLaunchKernelGGL((AttendSplitKernel<T, DP, MT>), grid, dim3(kThreads), 0, s, a, w, row_tiles,
                       unit0);
    return hipGetLastError();
  };
  if (a.batch.starts == nullptr || p.row_tiles == 1)
    return launch(dim3(each * p.row_tiles, a.batch.sequences), p.row_tiles, 0);
  return InUnits(a, RowUnits(a.cache, a.q_heads, 16 * MT), each, launch);
}

template <typename T, int DP, int NW>
hipError_t Tile(const Attend &a, const Work &w, const Plan &p, hipStream_t s) {
  const unsigned each = static_cast<unsigned>(a.cache.heads) * p.tile_splits;
  const auto launch = [&](dim3 grid, int row_tiles, int64_t unit0) {
    hipLaunchKernelGGL((AttendTileKernel<T, DP, NW>), grid, dim3(64 * NW), 0, s, a, w, row_tiles,
                       unit0);
    return hipGetLastError();
  };
  if (a.batch.starts == nullptr)
    return launch(dim3(each * p.tile_row_tiles, a.batch.sequences), p.tile_row_tiles, 0);
  return InUnits(a, RowUnits(a.cache, a.q_heads, 32 * NW), each, launch);
}

template <typename T, int DP>
hipError_t LaunchDim(const Attend &a, const Work &w, const Plan &p, hipStream_t s) {
  hipError_t e = hipSuccess;
  if constexpr (DP <= 128) {
    if (p.waves == 4) e = Tile<T, DP, 4>(a, w, p, s);
    if constexpr (Terms<T>() == 1)
      if (p.waves == 8) e = Tile<T, DP, 8>(a, w, p, s);
  }
  if (e != hipSuccess) return e;
  if constexpr (DP <= 128 && Terms<T>() == 1) {
    if (p.mt == 3) return Split<T, DP, 3>(a, w, p, s);
    if (p.mt == 4) return Split<T, DP, 4>(a, w, p, s);
  }
  if constexpr (DP <= 128 || Terms<T>() == 1)
    if (p.mt == 2) return Split<T, DP, 2>(a, w, p, s);
  if (p.mt == 1) return Split<T, DP, 1>(a, w, p, s);
  return e;
}

// Where a call's parts lie in the workspace.
struct Layout {
  size_t ml = 0, tile_sums = 0, tile_ml = 0, total = 0;
};

Layout LayoutOf(const Cache &c, const Batch &b, int32_t q_heads, const Plan &p) {
  Layout l;
  const auto round = [](size_t v) { return (v + 255) / 256 * 256; };
  const auto rows = [&](int splits, size_t tokens) {
    return splits > 1 ? static_cast<size_t>(splits) * tokens * q_heads : 0;
  };
  const size_t few = rows(p.splits, static_cast<size_t>(b.sequences) * p.few_tokens);
  const size_t many = rows(p.tile_splits, b.tokens);
  l.ml = round(few * c.dim * sizeof(float));
  l.tile_sums = l.ml + round(few * sizeof(float2));
  l.tile_ml = l.tile_sums + round(many * c.dim * sizeof(float));
  l.total = l.tile_ml + round(many * sizeof(float2));
  return l;
}

template <typename T>
hipError_t LaunchT(const Attend &a, int32_t x_type, void *work, hipStream_t s) {
  const Plan p = PlanOf(a.cache, a.batch, a.q_heads, x_type);
  const Layout l = LayoutOf(a.cache, a.batch, a.q_heads, p);
  char *const at = static_cast<char *>(work);
  const Work w{{reinterpret_cast<float *>(at), reinterpret_cast<float2 *>(at + l.ml), p.splits},
               {reinterpret_cast<float *>(at + l.tile_sums),
                reinterpret_cast<float2 *>(at + l.tile_ml), p.tile_splits},
               p.few,
               p.few_tokens};
  const hipError_t e = a.cache.dim <= 64    ? LaunchDim<T, 64>(a, w, p, s)
                       : a.cache.dim <= 128 ? LaunchDim<T, 128>(a, w, p, s)
                                            : LaunchDim<T, 256>(a, w, p, s);
  const int splits = std::max(p.splits, p.tile_splits);
  if (e != hipSuccess || splits == 1) return e;
  // Rows at a time, so that a grid's threads stay below 2^32.
  const int64_t rows = static_cast<int64_t>(a.batch.tokens) * a.q_heads, most = int64_t{1} << 23;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = std::min(most, rows - r);
    if (splits > 8 && rows <= 1024)
      hipLaunchKernelGGL((JoinKernel<T, kThreads>), dim3(static_cast<unsigned>(n)), dim3(kThreads),
                         0, s, a, w, r);
    else
      hipLaunchKernelGGL((JoinKernel<T, 64>), dim3(static_cast<unsigned>(CeilDiv(n, kWaves))),
                         dim3(kThreads), 0, s, a, w, r);
    const hipError_t j = hipGetLastError();
    if (j != hipSuccess) return j;
  }
  return hipSuccess;
}

} // namespace

size_t AttendWorkBytes(const Cache &c, const Batch &b, int32_t q_heads, int32_t x_type) {
  return LayoutOf(c, b, q_heads, PlanOf(c, b, q_heads, x_type)).total;
}

hipError_t LaunchAttend(const Attend &a, int32_t x_type, void *work, hipStream_t s) {
  switch (x_type) {
  case MNB_TYPE_FLOAT16: return LaunchT<_Float16>(a, x_type, work, s);
  case MNB_TYPE_BFLOAT16: return LaunchT<__bf16>(a, x_type, work, s);
  default: return LaunchT<float>(a, x_type, work, s);
  }
}

} // namespace kv
} // namespace mnb

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
// into the exponent: with y = s log2(e) + log2(w) and m the running maximum of y,
// P = 2^(y - m + 14) is the token's weight times its value scale, at most 2^14 and
// with full fp16 precision down to 2^-28 of the largest; the sum of the weights
// alone takes P / w. Then O / l needs no further scale.
// Queries are scaled by a power of two to below 2^15 and rounded to one fp16 term
// (exact for fp16, and for bf16 down to 2^-31 of the row's largest magnitude) or,
// fp32, to two (22 bits); P likewise is one term or, fp32, two.
#include "mnb_kv.h"
#include "mnb_values.h"

#include <type_traits>

namespace mnb {
namespace kv {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;          // tokens of a step
constexpr int kWaves = 4;          // of a workgroup: each takes every fourth tile of its part
constexpr int kThreads = 64 * kWaves;
constexpr float kInf = __builtin_inff();
constexpr float kShift = 14.0f;    // P's largest value is 2^14

template <typename T>
constexpr int Terms() { return sizeof(T) == 4 ? 2 : 1; }

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

// 0xFF in the place of each NaN code (0x7F or 0xFF).
__device__ __forceinline__ uint32_t NanBytes(uint32_t w) {
  const uint32_t top = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  return (top >> 7) * 0xFFu;
}

__device__ __forceinline__ float MaxGroups(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float SumGroups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ float Exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// log2 of a positive scale: an integer exactly for a power of two.
__device__ __forceinline__ float Log2Scale(float w) {
  int e;
  const float m = frexpf(w, &e);  // w = m 2^e, 0.5 <= m < 1
  return static_cast<float>(e - 1) + log2f(2.0f * m);
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

// A part of a row: parts[split][row][dim] sums, ml[split][row] = {maximum, sum}.
struct Work {
  float *parts;
  float2 *ml;
  int splits;
};

// DP: head_dim rounded up to 64, 128 or 256; MT: tiles of 16 queries.
// grid (splits, heads x row tiles, sequences). A row is a token's query head of
// this cache head: row r is token r / group, head r % group.
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kThreads) void AttendSplitKernel(Attend a, Work work, int row_tiles) {
  constexpr int kTerms = Terms<T>();
  constexpr int KS = DP / 64;      // 16-byte pieces of a key that a lane holds
  constexpr int VD = DP / 16;      // values of a token that a lane holds, tiles of O^T
  constexpr int VW = VD / 4;       // the same in words
  const Cache &c = a.cache;
  const int s = blockIdx.z, split = blockIdx.x;
  const int h = blockIdx.y / row_tiles, tile = blockIdx.y - h * row_tiles;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span span = SpanOf(a.batch, s, c.page_shift);
  const int group = a.q_heads / c.heads;
  const int64_t rows = static_cast<int64_t>(span.count) * group;
  const int64_t row0 = static_cast<int64_t>(tile) * (16 * MT);
  if (row0 >= rows) return;
  const int64_t row1 = min(row0 + 16 * MT, rows) - 1;
  const Reach reach = ReachOf(span, static_cast<int>(row0 / group), static_cast<int>(row1 / group),
                              a.window);
  const int tiles = reach.end > reach.begin ? (reach.end - reach.begin + kTile - 1) / kTile : 0;
  const int each = (tiles + work.splits - 1) / work.splits;
  const int tile1 = min(tiles, (split + 1) * each);

  // Queries. A lane's values for the two MFMAs of piece j are the halves of 16
  // neighbouring ones, as its codes of a key are.
  half8v q[MT][KS][2][kTerms];
  float cq[MT];   // what turns a dot product with key codes into log2 weights
  int pos[MT];
  int64_t out[MT];  // row of Y, -1 for none
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t r = row0 + 16 * t + col;
    const bool there = r < rows;
    const int i = there ? static_cast<int>(r / group) : 0, g = static_cast<int>(r - static_cast<int64_t>(i) * group);
    pos[t] = there ? span.first + i : -1;
    out[t] = there ? static_cast<int64_t>(span.row + i) * a.q_heads + h * group + g : -1;
    const T *x = static_cast<const T *>(a.q.x) + (span.row + i) * a.q.token_stride +
                 (h * group + (there ? g : 0)) * a.q.head_stride;
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
    int shift = 0;
    if constexpr (!std::is_same<T, _Float16>::value) {
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      shift = RangeExponent(__uint_as_float(top), 14);
    }
    cq[t] = ldexpf(a.scale * 1.44269504f, -shift);
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = ldexpf(f[j][half][e], shift);
          const _Float16 hi = static_cast<_Float16>(v);
          q[t][j][half][0][e] = hi;
          if constexpr (kTerms == 2)
            q[t][j][half][1][e] = static_cast<_Float16>(v - static_cast<float>(hi));
        }
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

  for (int step = split * each + wave; step < tile1; step += kWaves) {
    const int t0 = reach.begin + kTile * step;
    // Every token is seen by every row, unless the tile lies at an edge.
    bool edge = t0 + kTile - 1 > reach.pmin || t0 + kTile > reach.end ||
                (a.window > 0 && t0 <= reach.pmax - a.window);
    uint4v kw[4][KS];
    uint32_t vw[4][4][VW];
    float ks[4], ev[4], inv[4];
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      const int ts = t0 + 16 * sub;
      uint32_t id = ts < reach.end ? PageOf(a.batch, s, ts >> c.page_shift) : ~0u;
      const bool good = id < c.pages;
      edge |= !good;
      id = good ? id : 0u;  // in bounds; nothing of it counts
      const int64_t at = static_cast<int64_t>(id) * c.heads + h;
      const int slot = ts & ((1 << c.page_shift) - 1);
      const int64_t base = ((at << c.page_shift) + slot) * c.dim;
      const uint8_t *kp = c.codes[0] + base + col * c.dim;
      const uint8_t *vp = c.codes[1] + base + 4 * grp * c.dim;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        // Past head_dim the query is 0: any of this key's codes will do.
        const int d = 64 * j + 16 * grp;
        kw[sub][j] = *reinterpret_cast<const uint4v *>(kp + (d < c.dim ? d : 0));
      }
      // Past head_dim lie rows of O^T that are not stored.
      const int d = VD * col < c.dim ? VD * col : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(vp + i * c.dim + d);
#pragma unroll
        for (int x = 0; x < VW; ++x) vw[sub][i][x] = w[x];
      }
      const float sk = c.scales[0][at], sv = c.scales[1][at];
      ks[sub] = good ? sk : 0.0f;
      ev[sub] = good ? Log2Scale(sv) : -kInf;
      inv[sub] = good ? 1.0f / sv : 0.0f;
    }

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

    half8v p[MT][2][kTerms];
    bool grew = false;
    float alpha[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float top = -kInf;
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        const float scale = cq[t] * ks[sub];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = fmaf(acc[t][sub][i], scale, ev[sub]);
          if (edge) {
            const int tok = t0 + 16 * sub + 4 * grp + i;
            const bool seen = tok <= pos[t] && tok < reach.end && ev[sub] != -kInf &&
                              (a.window == 0 || tok > pos[t] - a.window);
            y = seen ? y : -kInf;
          }
          acc[t][sub][i] = y;
          top = fmaxf(top, y);
        }
      }
      top = fmaxf(m[t], MaxGroups(top));
      const float use = top == -kInf ? 0.0f : top;
      alpha[t] = Exp2(m[t] - use);
      grew |= top != m[t];
      m[t] = top;
      float sum = 0.0f;
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = Exp2(acc[t][sub][i] - (use - kShift));
          part += w;
          const _Float16 hi = static_cast<_Float16>(w);
          p[t][sub >> 1][0][4 * (sub & 1) + i] = hi;
          if constexpr (kTerms == 2)
            p[t][sub >> 1][1][4 * (sub & 1) + i] =
                static_cast<_Float16>(w - static_cast<float>(hi));
        }
        sum = fmaf(part, inv[sub], sum);
      }
      l[t] = fmaf(l[t], alpha[t], sum);
    }
    if (__any(grew)) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int d = 0; d < VD; ++d) o[t][d] *= alpha[t];
    }

#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {
      uint32_t w[2][4][VW];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int y = 0; y < VW; ++y) w[x][i][y] = vw[2 * pair + x][i][y];
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
              w[x][i][y] = seen ? w[x][i][y] : 0u;
              nan |= NanBytes(w[x][i][y]);
            }
          }
        if (__any(nan != 0)) {
          half8v seen[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int tok = t0 + 32 * pair + 16 * x + 4 * grp + i;
                seen[t][4 * x + i] = acc[t][2 * pair + x][i] == -kInf || tok > pos[t]
                                         ? static_cast<_Float16>(0.0f)
                                         : static_cast<_Float16>(1.0f);
              }
#pragma unroll
          for (int y = 0; y < VW; ++y) {
            uint32_t flag[2][4], turned[2][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t bytes = NanBytes(w[x][i][y]);
                w[x][i][y] &= ~bytes;
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
          const uint32_t in[4] = {w[x][0][y], w[x][1][y], w[x][2][y], w[x][3][y]};
          Transpose4(in, turned[x]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const half8v vf = Widen8(turned[0][b], turned[1][b]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
              o[t][4 * y + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[t][pair][term],
                                                                       o[t][4 * y + b], 0, 0, 0);
        }
      }
    }
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
    if (work.splits == 1) {
      const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
      T *y = static_cast<T *>(a.y) + at * c.dim + d0;
#pragma unroll
      for (int d = 0; d < VD; ++d) y[d] = static_cast<T>(v[d] * by);
    } else {
      const int64_t part = static_cast<int64_t>(split) * a.batch.tokens * a.q_heads + at;
      if (d0 == 0) work.ml[part] = make_float2(top, sum);
      float *y = work.parts + part * c.dim + d0;
      if (sum != 0.0f)
#pragma unroll
        for (int d = 0; d < VD; ++d) y[d] = v[d];
    }
  }
}

// Joins the splits of a row: one wavefront per row, four values of it a lane.
template <typename T>
__global__ __launch_bounds__(kThreads) void JoinKernel(Attend a, Work work) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  const Span span = SpanOf(a.batch, blockIdx.y, a.cache.page_shift);
  if (i >= static_cast<int64_t>(span.count) * a.q_heads) return;
  const int64_t row = static_cast<int64_t>(span.row) * a.q_heads + i;
  const int64_t step = static_cast<int64_t>(a.batch.tokens) * a.q_heads;
  const int d = 4 * (threadIdx.x & 63);
  const bool there = d < a.cache.dim;
  float top = -kInf;
  for (int s = 0; s < work.splits; ++s) top = fmaxf(top, work.ml[s * step + row].x);
  const float use = top == -kInf ? 0.0f : top;
  float sum = 0.0f;
  floatx4v v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < work.splits; ++s) {
    const float2 ml = work.ml[s * step + row];
    if (ml.y == 0.0f) continue;
    const float by = Exp2(ml.x - use);
    sum = fmaf(ml.y, by, sum);
    if (!there) continue;
    const floatx4v part =
        *reinterpret_cast<const floatx4v *>(work.parts + (s * step + row) * a.cache.dim + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(part[e], by, v[e]);
  }
  if (!there) return;
  const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
  T *y = static_cast<T *>(a.y) + row * a.cache.dim + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(v[e] * by);
}

// How a call is launched.
struct Plan {
  int mt, row_tiles, splits;
};

Plan PlanOf(const Cache &c, const Batch &b, int32_t q_heads, int32_t x_type) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(b.max_tokens) * (q_heads / c.heads);
  // Two tiles of fp32 queries 256 wide leave no registers for the keys.
  p.mt = rows > 16 && (c.dim <= 128 || x_type != MNB_TYPE_FLOAT) ? 2 : 1;
  p.row_tiles = static_cast<int>(CeilDiv(rows, 16 * p.mt));
  // Workgroups for three on each CU, each with a tile for every wavefront at least.
  const int64_t groups = static_cast<int64_t>(b.sequences) * c.heads * p.row_tiles;
  const int64_t tiles = CeilDiv(static_cast<int64_t>(b.width) << c.page_shift, kTile);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(64, tiles / kWaves));
  p.splits = static_cast<int>(std::min(most, std::max<int64_t>(1, 3 * 256 / groups)));
  return p;
}

template <typename T, int DP, int MT>
hipError_t Split(const Attend &a, const Work &w, const Plan &p, hipStream_t s) {
  const dim3 grid(p.splits, static_cast<unsigned>(a.cache.heads * p.row_tiles), a.batch.sequences);
  hipLaunchKernelGGL((AttendSplitKernel<T, DP, MT>), grid, dim3(kThreads), 0, s, a, w,
                     p.row_tiles);
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t SplitDim(const Attend &a, const Work &w, const Plan &p, hipStream_t s) {
  if constexpr (DP <= 128 || Terms<T>() == 1)
    if (p.mt == 2) return Split<T, DP, 2>(a, w, p, s);
  return Split<T, DP, 1>(a, w, p, s);
}

size_t Round256(size_t v) { return (v + 255) / 256 * 256; }

size_t PartBytes(const Cache &c, const Batch &b, int32_t q_heads, int splits) {
  return Round256(sizeof(float) * splits * b.tokens * q_heads * c.dim);
}

template <typename T>
hipError_t LaunchT(const Attend &a, int32_t x_type, void *work, hipStream_t s) {
  const Plan p = PlanOf(a.cache, a.batch, a.q_heads, x_type);
  const Work w{static_cast<float *>(work),
               reinterpret_cast<float2 *>(static_cast<char *>(work) +
                                          PartBytes(a.cache, a.batch, a.q_heads, p.splits)),
               p.splits};
  hipError_t e = a.cache.dim <= 64    ? SplitDim<T, 64>(a, w, p, s)
                 : a.cache.dim <= 128 ? SplitDim<T, 128>(a, w, p, s)
                                      : SplitDim<T, 256>(a, w, p, s);
  if (e != hipSuccess || p.splits == 1) return e;
  const dim3 grid(static_cast<unsigned>(
                      CeilDiv(static_cast<int64_t>(a.batch.max_tokens) * a.q_heads, kWaves)),
                  a.batch.sequences);
  hipLaunchKernelGGL((JoinKernel<T>), grid, dim3(kThreads), 0, s, a, w);
  return hipGetLastError();
}

} // namespace

size_t AttendWorkBytes(const Cache &c, const Batch &b, int32_t q_heads, int32_t x_type) {
  const Plan p = PlanOf(c, b, q_heads, x_type);
  if (p.splits == 1) return 0;
  return PartBytes(c, b, q_heads, p.splits) + sizeof(float2) * p.splits * b.tokens * q_heads;
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

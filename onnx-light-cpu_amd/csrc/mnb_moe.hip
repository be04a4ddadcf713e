// The mixture-of-experts layer for few tokens on 4-bit weights.
//
// A layer of few tokens is bound by reading the weights of the experts that
// they meet, 4.25 bits a value; what a CU does per weight has to stay small.
// The products are exact integers on the int8 MFMA:
//
//   x = 2^s (256^2 d2 + 256 d1 + d0), digits in [-128, 127] (two digits for
//   16-bit activations), one power of two for each block of 128 values,
//   w = scale (q - z), q - 8 in the high half of a byte: one mask per four
//   weights and no conversion.
//
// A token's digits are neighbouring columns of one MFMA tile: 16 columns hold
// five tokens of three digits or eight of two, so the digits cost no extra
// matrix instruction, and the rows of a tile are 16 weight rows. A weight
// block's sums S = 16 sum (q - 8) d are exact (below 2^21), as is S - 16 (z - 8)
// sum d; they are scaled and added up in fp32, column by column, and the
// columns of a token join after the last block.
//
// Four launches: logits and the fixed-point tokens; the choice; gate/up with
// the activation, whose rows leave in fixed point; down with the weighted sum
// over the experts. No atomics: every sum has one fixed order.
#include "mnb_moe.h"

#include <algorithm>

namespace mnb {
namespace moe {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// Columns of a tile per digit: the tokens of one column group.
template <int ND>
constexpr int kTokens = ND == 3 ? 5 : 8;

// ---- fixed point ---------------------------------------------------------------

// Eight values of a unit, k = 8 i .. 8 i + 7 for lane i of 16, into digits: row
// d at dig + d * stride (the unit's 128 bytes; the eight of lane i lie at
// 32 (i % 4) + 8 (i / 4), the order in which the weight layout takes them), the
// unit's power of two at *xs, and per digit and weight block the sum of its
// digits, times 16, at sd + d * sd_stride (folds words).
template <int ND>
__device__ __forceinline__ void StoreDigits(const float (&x)[8], int8_t *dig, int64_t stride,
                                            float *xs, float *sd, int64_t sd_stride, int folds) {
  const int i = threadIdx.x & 15;
  // As integers, magnitudes order like their values, infinity above them and NaN on top.
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1)
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 16)));
  const bool finite = top < 0x7F800000u;
  // 2^e <= amax < 2^(e + 1), at least 2^-90: smaller values count against that.
  // The largest magnitude becomes at most 2^22 (2^14 for two digits), so that
  // the top digit with its carries stays in a byte.
  const int e = finite ? max(static_cast<int>(top >> 23) - 127, -90) : 0;
  constexpr int kBits = ND == 3 ? 21 : 13;
  int n[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    n[j] = finite ? static_cast<int>(rintf(ldexpf(x[j], kBits - e))) : 0;
  const int lanes = 16 / folds;  // per weight block
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    uint32_t lo = 0, hi = 0;
    int sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int digit = d + 1 < ND ? static_cast<int>(static_cast<int8_t>(n[j])) : n[j];
      n[j] = (n[j] - digit) >> 8;
      sum += digit;
      const uint32_t b = static_cast<uint32_t>(digit) & 0xFFu;
      if (j < 4) lo |= b << (8 * j);
      else hi |= b << (8 * (j - 4));
    }
    *reinterpret_cast<uint2 *>(dig + d * stride + 32 * (i & 3) + 8 * (i >> 2)) =
        make_uint2(lo, hi);
    for (int off = 1; off < lanes; off <<= 1) sum += __shfl_xor(sum, off, 16);
    if (i % lanes == 0) sd[d * sd_stride + i / lanes] = 16.0f * static_cast<float>(sum);
  }
  // Digit d counts 256^d units of 2^(e - kBits); the 16 of the weights' bytes is here too.
  if (i == 0) *xs = finite ? ldexpf(1.0f, e - kBits - 4) : __uint_as_float(0x7FC00000u);
}

// Rows in fixed point: digits [rows][ND][units * 128], powers of two [rows][units],
// digit sums [rows][ND][units * folds].
struct Fixed {
  int8_t *dig;
  float *xs, *sd;
  int64_t units;
};

template <int ND>
__device__ __forceinline__ void StoreUnit(const Fixed &f, int64_t row, int64_t unit, int folds,
                                          const float (&x)[8]) {
  StoreDigits<ND>(x, f.dig + row * ND * f.units * kUnit + unit * kUnit, f.units * kUnit,
                  f.xs + row * f.units + unit, f.sd + (row * ND * f.units + unit) * folds,
                  f.units * folds, folds);
}

// ---- first launch: the tokens in fixed point and the logits ----------------------

// Workgroups 0 .. router_wgs - 1: one expert and up to RT tokens each, sums in
// 64 bits (the choice is a comparison of sums: it shall not hang on their
// order). The others: 16 lanes per (token, unit).
template <int ND, int RT, typename T>
__global__ __launch_bounds__(256) void MoePrepKernel(const T *__restrict__ X,
                                                     const float *__restrict__ R, float *logits,
                                                     Fixed fx, int tokens, int64_t H, int E,
                                                     int folds, int router_wgs) {
  const int tid = threadIdx.x;
  if (static_cast<int>(blockIdx.x) < router_wgs) {
    const int e = static_cast<int>(blockIdx.x) % E, t0 = static_cast<int>(blockIdx.x) / E * RT;
    const float *r = R + static_cast<int64_t>(e) * H;
    const T *x[RT];
    double sum[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      x[t] = X + static_cast<int64_t>(min(t0 + t, tokens - 1)) * H;
      sum[t] = 0.0;
    }
    for (int64_t k = tid; k < H; k += 256) {
      const double w = static_cast<double>(r[k]);
#pragma unroll
      for (int t = 0; t < RT; ++t) sum[t] = fma(w, static_cast<double>(static_cast<float>(x[t][k])), sum[t]);
    }
    __shared__ double red[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) sum[t] += __shfl_xor(sum[t], off, 64);
      if ((tid & 63) == 0) red[t][tid >> 6] = sum[t];
    }
    __syncthreads();
    if (tid < RT && t0 + tid < tokens)
      logits[static_cast<int64_t>(t0 + tid) * E + e] =
          static_cast<float>((red[tid][0] + red[tid][1]) + (red[tid][2] + red[tid][3]));
    return;
  }
  const int64_t item = static_cast<int64_t>(static_cast<int>(blockIdx.x) - router_wgs) * 16 + tid / 16;
  if (item >= tokens * fx.units) return;
  const int64_t row = item / fx.units, unit = item - row * fx.units;
  const int64_t k0 = unit * kUnit + 8 * (tid & 15);
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = k0 + j < H ? static_cast<float>(X[row * H + k0 + j]) : 0.0f;
  StoreUnit<ND>(fx, row, unit, folds, x);
}

// ---- second launch: the choice ------------------------------------------------

// Order-preserving bits of a logit, NaN as -inf.
__device__ __forceinline__ uint32_t Key(float l) {
  const uint32_t b = __float_as_uint(l != l ? -__builtin_inff() : l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One workgroup per token: an expert's place is the number of experts before
// it, by key and then by index.
__global__ __launch_bounds__(256) void MoeRouteKernel(const float *__restrict__ logits,
                                                      int32_t *pair_expert, float *pair_weight,
                                                      int32_t *ids, float *weights, int E, int k,
                                                      bool normalize) {
  __shared__ uint32_t key[kMaxExperts];
  __shared__ float best[kMaxTopK];
  __shared__ int32_t who[kMaxTopK];
  __shared__ float red[4];
  const int tid = threadIdx.x, t = blockIdx.x;
  const float *l = logits + static_cast<int64_t>(t) * E;
  // -0 and 0 are equal logits.
  for (int e = tid; e < E; e += 256) key[e] = Key(l[e] + 0.0f);
  __syncthreads();
  for (int e = tid; e < E; e += 256) {
    const uint32_t me = key[e];
    int place = 0;
    for (int j = 0; j < E; ++j) place += (key[j] > me || (key[j] == me && j < e)) ? 1 : 0;
    if (place < k) {
      best[place] = l[e] != l[e] ? -__builtin_inff() : l[e];
      who[place] = e;
    }
  }
  __syncthreads();
  float total = 0.0f;
  const float top = best[0];
  if (normalize) {
    for (int j = 0; j < k; ++j) total += expf(best[j] - top);
  } else {
    float s = 0.0f;
    for (int e = tid; e < E; e += 256) s += expf((l[e] != l[e] ? -__builtin_inff() : l[e]) - top);
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    total = (red[0] + red[1]) + (red[2] + red[3]);
  }
  if (tid < k) {
    const float p = expf(best[tid] - top) / total;
    pair_expert[t * k + tid] = who[tid];
    pair_weight[t * k + tid] = p;
    if (ids) ids[t * k + tid] = who[tid];
    if (weights) weights[t * k + tid] = p;
  }
}

// ---- the products ---------------------------------------------------------------

// One unit of R records of a row group with GC column groups.
template <int ND, int R, int GC, int F, bool ZP>
struct Stream {
  struct Unit {
    uint4 w[R];
    float4 s[R][F];
    uint32_t z[R][F];
    intx4 d[GC][2];
    float xs[GC], sd[GC][F];
  };
  // Per lane: the record, scale and zero-point bytes of the first unit; per
  // column group the digits, powers and sums of this lane's column.
  const uint8_t *rec;
  const float *scales;
  const int8_t *zeros;
  const int8_t *dig[GC];
  const float *xs[GC], *sd[GC];

  __device__ __forceinline__ void Rows(const Matrix &m, int64_t matrix, int64_t group, int lane) {
    const int64_t first = (matrix * m.groups + group) * m.units * R;
    const int q = lane >> 4;
    rec = m.rec + first * kRec + lane * 16;
    scales = m.scales + (first * 4 + q) * F * 4;
    if constexpr (ZP) zeros = m.zeros + (first * 4 + q) * F * 4;
  }
  __device__ __forceinline__ void Column(int g, const Fixed &f, int64_t row, int d, int lane) {
    dig[g] = f.dig + (row * ND + d) * f.units * kUnit + 32 * (lane >> 4);
    xs[g] = f.xs + row * f.units;
    if constexpr (ZP) sd[g] = f.sd + (row * ND + d) * f.units * F;
  }
  __device__ __forceinline__ void Load(int64_t u, Unit &o) const {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      o.w[r] = *reinterpret_cast<const uint4 *>(rec + (u * R + r) * kRec);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        o.s[r][f] = *reinterpret_cast<const float4 *>(scales + ((u * R + r) * 4 * F + f) * 4);
        if constexpr (ZP)
          o.z[r][f] = *reinterpret_cast<const uint32_t *>(zeros + ((u * R + r) * 4 * F + f) * 4);
      }
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      const intx4 *p = reinterpret_cast<const intx4 *>(dig[g] + u * kUnit);
      o.d[g][0] = p[0];
      o.d[g][1] = p[1];
      o.xs[g] = xs[g][u];
      if constexpr (ZP) {
#pragma unroll
        for (int f = 0; f < F; ++f) o.sd[g][f] = sd[g][u * F + f];
      }
    }
  }
  static __device__ __forceinline__ long Long(int lo, int hi) {
    return static_cast<long>((static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) |
                             static_cast<uint32_t>(lo));
  }
  // acc[r][g][v] += row 4 q + v, this lane's column.
  static __device__ __forceinline__ void Multiply(const Unit &o, floatx4 (&acc)[R][GC], int lane) {
    const bool low = lane < 32;  // lane groups of the first 16 values of each 32
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t w[4] = {o.w[r].x, o.w[r].y, o.w[r].z, o.w[r].w};
      int a[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[2 * i] = static_cast<int>((w[i] << 4) & 0xF0F0F0F0u);
        a[2 * i + 1] = static_cast<int>(w[i] & 0xF0F0F0F0u);
      }
      const intx4 a0{a[0], a[1], a[2], a[3]}, a1{a[4], a[5], a[6], a[7]};
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        const intx4 b0 = o.d[g][0], b1 = o.d[g][1];
        floatx4 part{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < F; ++f) {
          intx4 sum{0, 0, 0, 0};
          if constexpr (F == 1) {
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b0, sum, 0, 0, 0);
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b1, sum, 0, 0, 0);
          } else if constexpr (F == 2) {
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(f == 0 ? a0 : a1, f == 0 ? b0 : b1, sum, 0,
                                                        0, 0);
          } else {
            const int i = F == 4 ? f : f / 2;
            const intx4 b = i < 2 ? b0 : b1;
            int lo = b[2 * (i & 1)], hi = b[2 * (i & 1) + 1];
            if constexpr (F == 8) {  // half of the 32 values
              const bool mine = low == (f % 2 == 0);
              lo = mine ? lo : 0;
              hi = mine ? hi : 0;
            }
            sum = __builtin_amdgcn_mfma_i32_16x16x32_i8(Long(a[2 * i], a[2 * i + 1]), Long(lo, hi),
                                                        sum, 0, 0, 0);
          }
          const float s[4] = {o.s[r][f].x, o.s[r][f].y, o.s[r][f].z, o.s[r][f].w};
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float t = static_cast<float>(sum[v]);
            if constexpr (ZP) {
              const int z = static_cast<int8_t>(o.z[r][f] >> (8 * v));
              t = fmaf(-static_cast<float>(z), o.sd[g][f], t);  // exact
            }
            part[v] = fmaf(t, s[v], part[v]);
          }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[r][g][v] = fmaf(part[v], o.xs[g], acc[r][g][v]);
      }
    }
  }
  // Units u0, u0 + step, .. below u1.
  __device__ __forceinline__ void Run(int64_t u0, int64_t u1, int64_t step,
                                      floatx4 (&acc)[R][GC], int lane) const {
    if (u0 >= u1) return;
    Unit x, y;
    Load(u0, x);
    for (int64_t u = u0; u < u1; u += 2 * step) {
      Load(u + step < u1 ? u + step : u, y);
      Multiply(x, acc, lane);
      if (u + step < u1) {
        Load(u + 2 * step < u1 ? u + 2 * step : u, x);
        Multiply(y, acc, lane);
      }
    }
  }
};

// The sum of a token's digit columns, in the column of digit 0 (garbage in the
// others): v holds this lane's column times 256^digit.
template <int ND>
__device__ __forceinline__ float JoinDigits(float v) {
  const int b = __float_as_int(v);
  if constexpr (ND == 2) {  // columns t and 8 + t
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(b, 0x128, 0xF, 0xF, true));  // row_ror:8
  } else {  // columns t, 5 + t, 10 + t
    const float m = __int_as_float(__builtin_amdgcn_mov_dpp(b, 0x105, 0xF, 0xF, true));  // row_shl:5
    const float h = __int_as_float(__builtin_amdgcn_mov_dpp(b, 0x10A, 0xF, 0xF, true));  // row_shl:10
    return (h + m) + v;
  }
}

template <int ND>
__device__ __forceinline__ float DigitWeight(int digit) {
  return digit == 0 ? 1.0f : digit == 1 ? 256.0f : 65536.0f;
}

// What the choice gives each launch of experts: entry i of min(tokens * top_k,
// experts) is an expert with the pairs (token * top_k + place) that chose it.
struct Entries {
  int32_t *expert;  // [entries]
  int32_t *count;   // 0: an expert that another entry has, or nobody chose
  int32_t *pair;    // [entries][kMaxTokens]
};

// The pairs that chose an expert, in order: every thread of the first wavefront.
__device__ __forceinline__ int CollectPairs(const int32_t *pair_expert, int pairs, int e,
                                            int32_t *out) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int p0 = 0; p0 < pairs; p0 += 64) {
    const int p = p0 + lane;
    const bool mine = p < pairs && pair_expert[p] == e;
    const uint64_t mask = __ballot(mine);
    if (mine) out[n + __popcll(mask & ((uint64_t{1} << lane) - 1))] = p;
    n += __popcll(mask);
  }
  return n;
}

// Third launch: workgroup (b, i) the 128 channels of block b of entry i's
// expert, KS runs of the units for each of 8 wavefronts' 16 channels.
template <int ND, int GC, int F, bool ZP, int KS>
__global__ __launch_bounds__(512 * KS) void MoeGateUpKernel(Matrix m, Fixed fx, Fixed fh,
                                                            const int32_t *__restrict__ pair_expert,
                                                            Entries entries, int pairs, int top_k,
                                                            bool by_expert) {
  constexpr int kT = kTokens<ND>;
  __shared__ int32_t list[kMaxTokens];
  __shared__ int32_t shared_n;
  __shared__ float part[KS > 1 ? (KS - 1) * 8 : 1][2 * GC][64][4];
  __shared__ float hidden[GC * kT][kUnit];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int entry = blockIdx.y;
  const int e = by_expert ? entry : pair_expert[entry];
  if (wave == 0) {
    int n = CollectPairs(pair_expert, pairs, e, list);
    // Of the pairs that share an expert the first one works.
    if (!by_expert && list[0] != entry) n = 0;
    if (lane == 0) shared_n = n;
    if (blockIdx.x == 0) {
      if (lane == 0) {
        entries.expert[entry] = e;
        entries.count[entry] = n;
      }
      if (lane < n) entries.pair[entry * kMaxTokens + lane] = list[lane];
    }
  }
  __syncthreads();
  const int n = shared_n;
  if (n == 0) return;
  const int cg = wave & 7, ks = wave >> 3;
  const int c = lane & 15, q = lane >> 4;
  const int digit = min(c / kT, ND - 1), slot = c % kT;
  const float weight = c < ND * kT ? DigitWeight<ND>(digit) : 0.0f;
  Stream<ND, 2, GC, F, ZP> stream;
  stream.Rows(m, e, static_cast<int64_t>(blockIdx.x) * 8 + cg, lane);
  const int64_t run = CeilDiv(m.units, KS);
  for (int t0 = 0; t0 < n; t0 += GC * kT) {
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      const int i = t0 + g * kT + slot;
      stream.Column(g, fx, list[i < n ? i : 0] / top_k, digit, lane);
    }
    floatx4 acc[2][GC];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int g = 0; g < GC; ++g) acc[r][g] = floatx4{0.f, 0.f, 0.f, 0.f};
    stream.Run(ks * run, min(m.units, (ks + 1) * run), 1, acc, lane);
    if constexpr (KS > 1) {
      if (ks > 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int g = 0; g < GC; ++g)
            *reinterpret_cast<floatx4 *>(part[(ks - 1) * 8 + cg][r * GC + g][lane]) = acc[r][g];
      }
      __syncthreads();
    }
    if (ks == 0) {
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        float4 h;
        float *hv = &h.x;
#pragma unroll
        for (int r = 0; r < 2; ++r)
          for (int s = 1; s < KS; ++s)
            acc[r][g] += *reinterpret_cast<const floatx4 *>(part[(s - 1) * 8 + cg][r * GC + g][lane]);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float gate = JoinDigits<ND>(acc[0][g][v] * weight);
          const float up = JoinDigits<ND>(acc[1][g][v] * weight);
          hv[v] = SiluMul(gate, up);
        }
        if (c < kT) *reinterpret_cast<float4 *>(&hidden[g * kT + c][16 * cg + 4 * q]) = h;
      }
    }
    __syncthreads();
    for (int i = tid / 16; i < GC * kT; i += 32 * KS) {
      if (t0 + i < n) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = hidden[i][8 * (tid & 15) + j];
        StoreUnit<ND>(fh, list[t0 + i], blockIdx.x, F, x);
      }
    }
    __syncthreads();
  }
}

// Fourth launch: a workgroup takes 16 columns of Y and all experts. Its wavefronts
// share the list of (entry, unit) items in equal runs and keep sums of their own,
// which join in order.
constexpr int kDownWaves = 8;

template <int ND, int GC, int F, bool ZP, typename T>
__global__ __launch_bounds__(64 * kDownWaves) void MoeDownKernel(
    Matrix m, Fixed fh, Entries entries, const float *__restrict__ pair_weight, T *__restrict__ Y,
    int n_entries, int tokens, int top_k, int64_t H) {
  constexpr int kT = kTokens<ND>;
  extern __shared__ float sums[];  // [kDownWaves][tokens][16]
  __shared__ int32_t active[kMaxExperts];
  __shared__ int32_t shared_n;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (wave == 0) {
    int n = 0;
    for (int i0 = 0; i0 < n_entries; i0 += 64) {
      const int i = i0 + lane;
      const bool on = i < n_entries && entries.count[i] > 0;
      const uint64_t mask = __ballot(on);
      if (on) active[n + __popcll(mask & ((uint64_t{1} << lane) - 1))] = i;
      n += __popcll(mask);
    }
    if (lane == 0) shared_n = n;
  }
  float *mine = sums + static_cast<int64_t>(wave) * tokens * 16;
  for (int i = lane; i < tokens * 16; i += 64) mine[i] = 0.0f;
  __syncthreads();
  const int64_t items = shared_n * m.units;
  const int64_t i0 = items * wave / kDownWaves, i1 = items * (wave + 1) / kDownWaves;
  const int c = lane & 15, q = lane >> 4;
  const int digit = min(c / kT, ND - 1), slot = c % kT;
  const float weight = c < ND * kT ? DigitWeight<ND>(digit) : 0.0f;
  for (int64_t i = i0; i < i1;) {
    const int entry = active[i / m.units];
    const int64_t u0 = i % m.units, u1 = min(m.units, u0 + (i1 - i));
    const int32_t *list = entries.pair + entry * kMaxTokens;
    const int n = entries.count[entry];
    Stream<ND, 1, GC, F, ZP> stream;
    stream.Rows(m, entries.expert[entry], blockIdx.x, lane);
    for (int t0 = 0; t0 < n; t0 += GC * kT) {
      int pair[GC];
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        const int j = t0 + g * kT + slot;
        pair[g] = list[j < n ? j : 0];
        stream.Column(g, fh, pair[g], digit, lane);
      }
      floatx4 acc[1][GC];
#pragma unroll
      for (int g = 0; g < GC; ++g) acc[0][g] = floatx4{0.f, 0.f, 0.f, 0.f};
      stream.Run(u0, u1, 1, acc, lane);
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        float y[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = JoinDigits<ND>(acc[0][g][v] * weight);
        if (c < kT && t0 + g * kT + c < n) {
          const float p = pair_weight[pair[g]];
          float4 *at = reinterpret_cast<float4 *>(mine + (pair[g] / top_k) * 16 + 4 * q);
          float4 s = *at;
          s.x = fmaf(p, y[0], s.x);
          s.y = fmaf(p, y[1], s.y);
          s.z = fmaf(p, y[2], s.z);
          s.w = fmaf(p, y[3], s.w);
          *at = s;
        }
      }
    }
    i += u1 - u0;
  }
  __syncthreads();
  for (int i = tid; i < tokens * 16; i += 64 * kDownWaves) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 16 + (i & 15);
    if (n >= H) continue;
    float y = sums[i];
    for (int w = 1; w < kDownWaves; ++w) y += sums[w * tokens * 16 + i];
    Y[(i >> 4) * H + n] = static_cast<T>(y);
  }
}

// ---- weight layout -----------------------------------------------------------------

// One thread per 16 bytes of a record.
__global__ __launch_bounds__(256) void MoeRecordKernel(const uint8_t *__restrict__ B,
                                                       uint8_t *__restrict__ rec, int64_t N,
                                                       int64_t K, int64_t row_bytes, int64_t groups,
                                                       int64_t units, int r, int R, int64_t total) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int lane = static_cast<int>(i & 63);
  const int64_t unit_id = i >> 6;  // (matrix, group, unit)
  const int64_t u = unit_id % units, mg = unit_id / units, matrix = mg / groups,
                group = mg - matrix * groups;
  const int64_t n = group * 16 + (lane & 15);
  uint32_t out[4] = {0, 0, 0, 0};
  if (n < N) {
    const uint8_t *row = B + (matrix * N + n) * row_bytes;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int64_t k = u * kUnit + 32 * w + 8 * (lane >> 4);
      if (k >= K) continue;
      uint32_t v = *reinterpret_cast<const uint32_t *>(row + k / 2) ^ 0x88888888u;
      if (k + 8 > K) v &= (1u << (4 * (K - k))) - 1u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[w] |= ((v >> (4 * j)) & 15u) << (8 * j) | ((v >> (4 * j + 16)) & 15u) << (8 * j + 4);
    }
  }
  reinterpret_cast<uint4 *>(rec)[(unit_id * R + r) * 64 + lane] =
      make_uint4(out[0], out[1], out[2], out[3]);
}

// One thread per scale: [4 q][folds][4] of a record.
__global__ __launch_bounds__(256) void MoeScaleKernel(const float *__restrict__ S,
                                                      const uint8_t *__restrict__ Z,
                                                      float *__restrict__ scales,
                                                      int8_t *__restrict__ zeros, int64_t N,
                                                      int64_t nb, int64_t groups, int64_t units,
                                                      int folds, int block_size, int r, int R,
                                                      int64_t total) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int per = 16 * folds;
  const int at = static_cast<int>(i % per);
  const int v = at & 3, f = at / 4 % folds, q = at / (4 * folds);
  const int64_t unit_id = i / per;
  const int64_t u = unit_id % units, mg = unit_id / units, matrix = mg / groups,
                group = mg - matrix * groups;
  const int64_t n = group * 16 + 4 * q + v;
  const int64_t b = block_size >= kUnit ? u * kUnit / block_size : u * folds + f;
  float s = 0.0f;
  int z = 8;
  if (n < N && b < nb) {
    s = S[(matrix * N + n) * nb + b];
    if (Z) z = (Z[(matrix * N + n) * ((nb + 1) / 2) + b / 2] >> (4 * (b & 1))) & 15;
  }
  const int64_t o = (unit_id * R + r) * per + at;
  scales[o] = s;
  if (Z) zeros[o] = static_cast<int8_t>(z - 8);
}

// ---- launches ------------------------------------------------------------------------

struct Work {
  Fixed fx, fh;
  float *logits;
  int32_t *pair_expert;
  float *pair_weight;
  Entries entries;
  size_t bytes;
};

Work Split(const Layer &l, int T, int ND, void *base) {
  Work w;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *p = static_cast<char *>(base) + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const size_t pairs = static_cast<size_t>(T) * l.top_k;
  auto fixed = [&](size_t rows, int64_t units) {
    Fixed f;
    f.units = units;
    f.dig = reinterpret_cast<int8_t *>(take(rows * ND * units * kUnit));
    f.xs = reinterpret_cast<float *>(take(rows * units * 4));
    f.sd = reinterpret_cast<float *>(take(rows * ND * units * l.folds * 4));
    return f;
  };
  w.fx = fixed(T, l.gate_up.units);
  w.fh = fixed(pairs, l.down.units);
  w.logits = reinterpret_cast<float *>(take(static_cast<size_t>(T) * l.experts * 4));
  w.pair_expert = reinterpret_cast<int32_t *>(take(pairs * 4));
  w.pair_weight = reinterpret_cast<float *>(take(pairs * 4));
  const size_t entries = std::min<size_t>(pairs, l.experts);
  w.entries.expert = reinterpret_cast<int32_t *>(take(entries * 4));
  w.entries.count = reinterpret_cast<int32_t *>(take(entries * 4));
  w.entries.pair = reinterpret_cast<int32_t *>(take(entries * kMaxTokens * 4));
  w.bytes = at;
  return w;
}

template <int ND, int GC, int F, bool ZP, typename T>
hipError_t LaunchExperts(const Layer &l, const Work &w, int tokens, void *Y, hipStream_t s) {
  const int pairs = tokens * l.top_k;
  const int entries = std::min(pairs, l.experts);
  const dim3 grid(static_cast<unsigned>(l.gate_up.groups / 8), static_cast<unsigned>(entries));
  hipLaunchKernelGGL((MoeGateUpKernel<ND, GC, F, ZP, 1>), grid, dim3(512), 0, s, l.gate_up, w.fx,
                     w.fh, w.pair_expert, w.entries, pairs, l.top_k, pairs >= l.experts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const size_t lds = static_cast<size_t>(kDownWaves) * tokens * 16 * sizeof(float);
  hipLaunchKernelGGL((MoeDownKernel<ND, GC, F, ZP, T>), dim3(static_cast<unsigned>(l.down.groups)),
                     dim3(64 * kDownWaves), lds, s, l.down, w.fh, w.entries, w.pair_weight,
                     static_cast<T *>(Y), entries, tokens, l.top_k, l.hidden);
  return hipGetLastError();
}

template <int ND, int GC, bool ZP, typename T>
hipError_t LaunchFolds(const Layer &l, const Work &w, int tokens, void *Y, hipStream_t s) {
  switch (l.folds) {
  case 1: return LaunchExperts<ND, GC, 1, ZP, T>(l, w, tokens, Y, s);
  case 2: return LaunchExperts<ND, GC, 2, ZP, T>(l, w, tokens, Y, s);
  case 4: return LaunchExperts<ND, GC, 4, ZP, T>(l, w, tokens, Y, s);
  default: return LaunchExperts<ND, GC, 8, ZP, T>(l, w, tokens, Y, s);
  }
}

template <typename T>
hipError_t LaunchLayerT(const Layer &l, int tokens, const void *X, const float *logits, void *Y,
                        int32_t *ids, float *weights, void *work, hipStream_t s) {
  constexpr int ND = sizeof(T) == 4 ? 3 : 2;
  const Work w = Split(l, tokens, ND, work);
  constexpr int kRT = 4;
  const int router_wgs =
      logits ? 0 : l.experts * (tokens == 1 ? 1 : static_cast<int>(CeilDiv(tokens, kRT)));
  const unsigned prep =
      static_cast<unsigned>(router_wgs + CeilDiv(tokens * l.gate_up.units, 16));
  if (tokens == 1)
    hipLaunchKernelGGL((MoePrepKernel<ND, 1, T>), dim3(prep), dim3(256), 0, s,
                       static_cast<const T *>(X), l.router, w.logits, w.fx, tokens, l.hidden,
                       l.experts, l.folds, router_wgs);
  else
    hipLaunchKernelGGL((MoePrepKernel<ND, kRT, T>), dim3(prep), dim3(256), 0, s,
                       static_cast<const T *>(X), l.router, w.logits, w.fx, tokens, l.hidden,
                       l.experts, l.folds, router_wgs);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(MoeRouteKernel, dim3(static_cast<unsigned>(tokens)), dim3(256), 0, s,
                     logits ? logits : w.logits, w.pair_expert, w.pair_weight, ids, weights,
                     l.experts, l.top_k, l.normalize);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  // Column groups per pass over an expert's rows: what its share of the tokens fills.
  const bool many = static_cast<int64_t>(tokens) * l.top_k > static_cast<int64_t>(l.experts) * kTokens<ND> / 2;
  if (l.zeros)
    return many ? LaunchFolds<ND, 2, true, T>(l, w, tokens, Y, s)
                : LaunchFolds<ND, 1, true, T>(l, w, tokens, Y, s);
  return many ? LaunchFolds<ND, 2, false, T>(l, w, tokens, Y, s)
              : LaunchFolds<ND, 1, false, T>(l, w, tokens, Y, s);
}

} // namespace

hipError_t LaunchRelayout(const mnb_moe_weight &src, int64_t N, int64_t K, int block_size,
                          int experts, int r, int R, uint8_t *rec, float *scales, int8_t *zeros,
                          hipStream_t s) {
  const int64_t units = CeilDiv(K, kUnit);
  const int64_t groups = R == 2 ? CeilDiv(N, kUnit) * (kUnit / 16) : CeilDiv(N, 16);
  const int64_t nb = CeilDiv(K, block_size);
  const int64_t row_bytes = nb * (block_size / 2);
  const int folds = std::max(1, kUnit / block_size);
  // Experts at a time, so that a grid's threads stay below 2^32 (one expert's
  // are at most 2^31: hidden * intermediate <= 2^34).
  const int64_t one = groups * units * std::max(64, 16 * folds);
  const int64_t per = std::max<int64_t>(1, (int64_t{1} << 31) / one);
  for (int64_t e = 0; e < experts; e += per) {
    const int64_t n = std::min<int64_t>(per, experts - e);
    const int64_t total = n * groups * units;
    const int64_t first = e * groups * units * R;
    hipLaunchKernelGGL(MoeRecordKernel, dim3(static_cast<unsigned>(CeilDiv(total * 64, 256))),
                       dim3(256), 0, s, src.B + e * N * row_bytes, rec + first * kRec, N, K,
                       row_bytes, groups, units, r, R, total * 64);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(MoeScaleKernel, dim3(static_cast<unsigned>(CeilDiv(total * 16 * folds, 256))),
                       dim3(256), 0, s, src.scales + e * N * nb,
                       src.zero_points ? src.zero_points + e * N * ((nb + 1) / 2) : nullptr,
                       scales + first * 16 * folds, zeros ? zeros + first * 16 * folds : nullptr, N,
                       nb, groups, units, folds, block_size, r, R, total * 16 * folds);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

size_t WorkBytes(const Layer &l, int T, int32_t x_type) {
  return Split(l, T, x_type == MNB_TYPE_FLOAT ? 3 : 2, nullptr).bytes;
}

hipError_t LaunchLayer(const Layer &l, int T, int32_t x_type, const void *X, const float *logits,
                       void *Y, int32_t *ids, float *weights, void *work, hipStream_t s) {
  switch (x_type) {
  case MNB_TYPE_FLOAT16:
    return LaunchLayerT<_Float16>(l, T, X, logits, Y, ids, weights, work, s);
  case MNB_TYPE_BFLOAT16:
    return LaunchLayerT<__bf16>(l, T, X, logits, Y, ids, weights, work, s);
  default: return LaunchLayerT<float>(l, T, X, logits, Y, ids, weights, work, s);
  }
}

} // namespace moe
} // namespace mnb

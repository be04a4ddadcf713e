// The mixture-of-experts layer for few tokens on 4-bit weights.
//
// A layer of few tokens is bound by reading the weights of the experts that
// they meet, 4.25 bits a value; what a CU does per weight has to stay small.
// The products are exact integers on the int8 MFMA:
//
//   x = 2^s (256^2 d2 + 256 d1 + d0), digits in [-128, 127], one power of two for
//   each block of 128 values, 22 bits below the block's largest magnitude. A float16
//   value keeps all its bits down to 2^-11 of that magnitude, a bfloat16 one down to
//   2^-14; smaller ones, and fp32 values and experts' rows, are off by at most 2^-22 of
//   it, as much as four fp32 additions to the largest value's product. (With two digits
//   for 16-bit activations, 14 bits, the values beside an outlier of 2^12 times their
//   size kept two.)
//   w = scale (q - z), q - z in a byte by three or four operations on four
//   weights at once, without conversions.
//
// A token's digits are columns of one MFMA tile: 16 columns hold five tokens of
// three digits, so the digits of few tokens cost no extra matrix instruction,
// and the rows of a tile are 16 weight rows. A weight block's sums are exact
// integers (below 2^21); they are scaled and added up in fp32, column by column,
// and the columns of a token join after the last block.
//
// Three to five launches: logits and the fixed-point tokens; the choice (of one
// token the gate/up workgroups each make it); gate/up with the activation, whose
// rows leave in fixed point; down, with the weighted sum over the experts where
// few tokens' sums fit its workgroups, otherwise that sum on its own. Every sum of
// floating-point values has one fixed order.
#include "mnb_moe.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mnb {
namespace moe {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// Digits of a value.
constexpr int kND = 3;

// Columns of a tile per digit: the tokens of one column group. ONE: a group of
// one token, whose digits alone are kept and copied.
template <bool ONE>
constexpr int kTokens = ONE ? 1 : 16 / kND;

// ---- fixed point ---------------------------------------------------------------

// Rows in fixed point: digits [rows][kND][units * 128] and the powers of two of
// each unit's `scales` parts [rows][units][scales].
struct Fixed {
  int8_t *dig;
  float *power;
  int64_t units;
  int scales;
};

// Eight values of a unit of row `row`, k = 8 i .. 8 i + 7, by thread i (% 16) of
// 16, or of the 16 / scales that share a part. The unit's 128 bytes of a digit
// lie as the weight layout takes them, 16 for each half of the unit and lane
// group: the eight of i at 64 (i / 8) + 16 (i % 4) + 8 (i / 4 % 2).
__device__ __forceinline__ void StoreUnit(const Fixed &f, int64_t row, int64_t unit, int i,
                                          const float (&x)[8]) {
  // As integers, magnitudes order like their values, infinity above them and NaN on top.
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  const int part = 16 / f.scales;
  for (int off = part >> 1; off >= 1; off >>= 1)
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 16)));
  const bool finite = top < 0x7F800000u;
  // 2^e <= amax < 2^(e + 1), at least 2^-90: smaller values count against that.
  // The largest magnitude becomes at most 2^22, so that the top digit with its
  // carries stays in a byte.
  const int e = finite ? max(static_cast<int>(top >> 23) - 127, -90) : 0;
  constexpr int kBits = 8 * kND - 3;
  int n[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    n[j] = finite ? static_cast<int>(rintf(ldexpf(x[j], kBits - e))) : 0;
  if (i % part == 0)
    f.power[(row * f.units + unit) * f.scales + i / part] =
        finite ? ldexpf(1.0f, e - kBits) : __uint_as_float(0x7FC00000u);
#pragma unroll
  for (int d = 0; d < kND; ++d) {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int digit = d + 1 < kND ? static_cast<int>(static_cast<int8_t>(n[j])) : n[j];
      n[j] = (n[j] - digit) >> 8;
      const uint32_t b = static_cast<uint32_t>(digit) & 0xFFu;
      if (j < 4) lo |= b << (8 * j);
      else hi |= b << (8 * (j - 4));
    }
    *reinterpret_cast<uint2 *>(f.dig + ((row * kND + d) * f.units + unit) * kUnit + 64 * (i >> 3) +
                               16 * (i & 3) + 8 * ((i >> 2) & 1)) = make_uint2(lo, hi);
  }
}

// ---- first launch: the tokens in fixed point and the logits ----------------------

// Workgroups 0 .. router_wgs - 1: one expert and up to RT tokens each, sums in
// 64 bits (the choice is a comparison of sums: it shall not hang on their
// order). The others: 16 lanes per (token, unit). VEC: H a multiple of 4, rows of
// X and R aligned to four values.
template <int RT, bool VEC, typename T>
__global__ __launch_bounds__(256) void MoePrepKernel(const T *__restrict__ X,
                                                     const float *__restrict__ R, float *logits,
                                                     Fixed fx, int tokens, int64_t H, int E,
                                                     int router_wgs) {
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
    const int width = static_cast<int>(H);
    if constexpr (VEC) {
      typedef T Four __attribute__((ext_vector_type(4)));
#pragma unroll 4
      for (int k = 4 * tid; k < width; k += 1024) {
        const floatx4 w = *reinterpret_cast<const floatx4 *>(r + k);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const Four v = *reinterpret_cast<const Four *>(x[t] + k);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sum[t] = fma(static_cast<double>(w[j]),
                         static_cast<double>(static_cast<float>(v[j])), sum[t]);
        }
      }
    } else {
      for (int k = tid; k < width; k += 256) {
        const double w = static_cast<double>(r[k]);
#pragma unroll
        for (int t = 0; t < RT; ++t)
          sum[t] = fma(w, static_cast<double>(static_cast<float>(x[t][k])), sum[t]);
      }
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
  StoreUnit(fx, row, unit, tid & 15, x);
}

// ---- second launch: the choice ------------------------------------------------

// Order-preserving bits of a logit, NaN as -inf.
__device__ __forceinline__ uint32_t Key(float l) {
  const uint32_t b = __float_as_uint(l != l ? -__builtin_inff() : l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The first k experts of a token, by all THREADS of a workgroup: best[i] and who[i]
// the i-th largest logit and its expert. An expert's place is the number of experts
// before it, by key and then by index.
template <int THREADS>
__device__ __forceinline__ void Choose(const float *__restrict__ l, int E, int k, uint32_t *key,
                                       float *best, int32_t *who) {
  const int tid = threadIdx.x;
  const int padded = (E + 3) & ~3;
  // -0 and 0 are equal logits; key 0 is below every logit's.
  for (int e = tid; e < padded; e += THREADS) key[e] = e < E ? Key(l[e] + 0.0f) : 0u;
  __syncthreads();
  const uint4 *key4 = reinterpret_cast<const uint4 *>(key);
  for (int e = tid; e < E; e += THREADS) {
    const uint32_t me = key[e];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < padded / 4; ++j) {
      const uint4 v = key4[j];
      // Before e equal keys count too: they exceed me - 1 (keys are above 0).
      const int at = 4 * j;
      place += v.x > me - (at < e ? 1u : 0u) ? 1 : 0;
      place += v.y > me - (at + 1 < e ? 1u : 0u) ? 1 : 0;
      place += v.z > me - (at + 2 < e ? 1u : 0u) ? 1 : 0;
      place += v.w > me - (at + 3 < e ? 1u : 0u) ? 1 : 0;
    }
    if (place < k) {
      best[place] = __uint_as_float(me & 0x80000000u ? me & 0x7FFFFFFFu : ~me);
      who[place] = e;
    }
  }
  __syncthreads();
}

// What the weights expf(best[i] - best[0]) are divided by: the sum over the chosen,
// or over all; by all THREADS.
template <int THREADS>
__device__ __forceinline__ float WeightSum(const float *__restrict__ l, int E, int k, bool normalize,
                                           const float *best) {
  __shared__ float red[THREADS / 64];
  const int tid = threadIdx.x;
  const float top = best[0];
  float total = 0.0f;
  if (normalize) {
    for (int j = 0; j < k; ++j) total += expf(best[j] - top);
    return total;
  }
  float s = 0.0f;
  for (int e = tid; e < E; e += THREADS)
    s += expf((l[e] != l[e] ? -__builtin_inff() : l[e]) - top);
  for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  for (int w = 0; w < THREADS / 64; ++w) total += red[w];
  return total;
}

// One workgroup per token.
__global__ __launch_bounds__(256) void MoeRouteKernel(const float *__restrict__ logits,
                                                      int32_t *pair_expert, float *pair_weight,
                                                      int32_t *ids, float *weights, int E, int k,
                                                      bool normalize) {
  __shared__ uint4 key[kMaxExperts / 4];
  __shared__ float best[kMaxTopK];
  __shared__ int32_t who[kMaxTopK];
  const int tid = threadIdx.x, t = blockIdx.x;
  const float *l = logits + static_cast<int64_t>(t) * E;
  Choose<256>(l, E, k, reinterpret_cast<uint32_t *>(key), best, who);
  const float total = WeightSum<256>(l, E, k, normalize, best);
  if (tid < k) {
    const float p = expf(best[tid] - best[0]) / total;
    pair_expert[t * k + tid] = who[tid];
    pair_weight[t * k + tid] = p;
    if (ids) ids[t * k + tid] = who[tid];
    if (weights) weights[t * k + tid] = p;
  }
}

// ---- the products ---------------------------------------------------------------

// A pipe streams units through LDS: SHARE wavefronts, each with R records of its
// own per unit (both of its row group, or one of them), and one set of GC column
// groups for all of them (SHARE = 1: a pipe of one wavefront, without barriers).
// NS units are in flight by direct global -> LDS copies, so what keeps the memory
// busy needs no registers. F weight blocks per unit, XB parts of it with powers
// of two of their own.
template <bool ONE, int GC, int R, int F, int XB, bool ZP, int SHARE, int NS>
struct Pipe {
  static_assert(!ONE || GC == 1, "one token, one column group");
  static constexpr int kT = kTokens<ONE>;
  static constexpr int kCols = ONE ? 4 : 16;  // kept columns of a group
  static constexpr int kFolds = F > XB ? F : XB;
  static constexpr int kMeta = MetaBytes(F, ZP);
  static constexpr int kMetaCopies = (kMeta + kRec - 1) / kRec;
  static constexpr int kDigitCopies = ONE ? 1 : 2 * GC;
  static constexpr int kShared = kDigitCopies + 1;  // the last one the powers'
  static constexpr int kSharedPer = (kShared + SHARE - 1) / SHARE;
  static constexpr int kOps = R + kMetaCopies + kSharedPer;
  static constexpr int kPrivate = R * kRec + kMeta;
  static constexpr int kDigits = SHARE * kPrivate;  // offsets in a stage
  static constexpr int kPowers = kDigits + GC * 128 * kCols;
  static constexpr int kStage = kPowers + (ONE ? 16 : GC * 16 * XB * 4);
  static constexpr int kLds = NS * kStage;
  static_assert(kMeta % 16 == 0 && kOps * (NS - 1) < 64, "copies");
  static_assert(XB == 1 || GC == 1, "powers: one copy");

  const uint8_t *lds;  // this pipe's
  uint32_t base;       // its LDS byte
  int lane, ws;        // lane and wavefront of the pipe
  int half;            // R = 1: which record
  // Sources at unit 0 of the current segment.
  const uint8_t *w_src, *m_src;
  uint32_t s_off[kSharedPer];  // bytes from the digits or the powers (below 2^31)
  bool s_on[kSharedPer];  // this lane's column has a token

  __device__ __forceinline__ Pipe(const uint8_t *at, int lane_, int ws_, int half_ = 0)
      : lds(at), base(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at))), lane(lane_), ws(ws_),
        half(half_) {}

  // Which of the shared copies this wavefront makes; past the last it repeats that.
  __device__ __forceinline__ int SharedCopy(int i) const {
    return min(i * SHARE + ws, kShared - 1);
  }
  // A segment: row group `group` (of 32 rows) of a matrix, and n tokens (at
  // most GC * kT) whose fixed-point rows row_of(0 .. n - 1) names.
  template <typename RowOf>
  __device__ __forceinline__ void Segment(const Matrix &m, int64_t matrix, int64_t group,
                                          const Fixed &f, int n, RowOf row_of) {
    const int64_t first = (matrix * m.groups + group) * m.units;
    w_src = m.rec + (first * kRecords + half) * kRec;
    m_src = m.meta + first * kMeta;
#pragma unroll
    for (int i = 0; i < kSharedPer; ++i) {
      const int s = SharedCopy(i);
      const bool powers = s == kDigitCopies;
      // The column whose data this lane copies; of digits eight columns of 128 bytes
      // (whole lines), the 16-byte unit x of column c at place x ^ ((c / 2) % 8).
      const int column = powers ? lane : ONE ? lane >> 3 : s * 8 + (lane >> 3);
      const int c = column & 15, digit = c / kT, token = (column >> 4) * kT + c % kT;
      // Columns without a token keep what LDS holds: nothing reads their sums. One
      // lane is always on, so that every copy is issued and counted.
      // A wavefront without a copy of its own repeats one lane of the last.
      s_on[i] = (token < n && digit < kND && column < 16 * GC && (!ONE || !powers || lane == 0) &&
                 i * SHARE + ws < kShared) || lane == 0;
      const uint32_t row = row_of(token < n ? token : 0), units = static_cast<uint32_t>(f.units);
      s_off[i] = powers ? row * units * (XB * 4)
                        : (row * kND + min(digit, kND - 1)) * units * kUnit +
                              ((lane & 7) ^ ((c >> 1) & 7)) * 16;
    }
  }
  __device__ __forceinline__ void Issue(const Fixed &f, int u, int stage) const {
    const uint32_t st = base + stage * kStage;
    const uint32_t mine = st + ws * kPrivate;
    const uint32_t l16 = static_cast<uint32_t>(lane) * 16;
#pragma unroll
    for (int r = 0; r < R; ++r)
      CopyToLds16S(w_src + (static_cast<int64_t>(u) * kRecords + r) * kRec, l16, mine + r * kRec);
#pragma unroll
    for (int i = 0; i < kMetaCopies; ++i)
      if (i * 64 + lane < kMeta / 16)
        CopyToLds16S(m_src + static_cast<int64_t>(u) * kMeta + i * kRec, l16, mine + (R + i) * kRec);
#pragma unroll
    for (int i = 0; i < kSharedPer; ++i) {
      const int s = SharedCopy(i);
      if (s_on[i]) {
        if (s < kDigitCopies) CopyToLds16S(f.dig + u * kUnit, s_off[i], st + kDigits + s * kRec);
        else if constexpr (XB == 1) CopyToLds4S(f.power + u, s_off[i], st + kPowers);
        else CopyToLds16S(f.power + u * XB, s_off[i], st + kPowers);
      }
    }
  }
  // Waits until all but the newest N copies of this wavefront are in LDS (for
  // every wavefront of the pipe).
  template <int N>
  static __device__ __forceinline__ void Wait() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
    if constexpr (SHARE > 1) __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    __asm__ volatile("" ::: "memory");
  }
  static __device__ __forceinline__ long Long(int lo, int hi) {
    return static_cast<long>((static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) |
                             static_cast<uint32_t>(lo));
  }
  // Four nibbles (in the low halves of the bytes) less the zero points zz: with
  // the top bit set no byte borrows (128 + q - z is in 113 .. 143), and flipping it
  // leaves the two's complement.
  static __device__ __forceinline__ int Shift(uint32_t nibbles, uint32_t zz) {
    return static_cast<int>((((nibbles & 0x0F0F0F0Fu) | 0x80808080u) - zz) ^ 0x80808080u);
  }
  // acc[r][g][v] += row 4 q + v of record r, this lane's column of group g
  // (groups past `groups` are left out).
  __device__ __forceinline__ void Multiply(int stage, int groups, floatx4 (&acc)[R][GC]) const {
    const uint8_t *st = lds + stage * kStage, *mine = st + ws * kPrivate;
    const int c = lane & 15, q = lane >> 4;
    const bool low = q < 2;  // lane groups of the first 16 values of each 32
    int a[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint4 wv = *reinterpret_cast<const uint4 *>(mine + r * kRec + lane * 16);
      const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
      if constexpr (ZP) {
        const uint8_t *zp = mine + R * kRec + kRecords * 64 * F + ((r + half) * 16 + c) * F;
        uint32_t z[2];
        if constexpr (F == 1) z[0] = *zp;
        else if constexpr (F == 2) z[0] = *reinterpret_cast<const uint16_t *>(zp);
        else z[0] = *reinterpret_cast<const uint32_t *>(zp);
        if constexpr (F == 8) z[1] = *reinterpret_cast<const uint32_t *>(zp + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t zz;
          if constexpr (F == 8) {  // lane groups 0, 1: block 2 i, the others block 2 i + 1
            const uint32_t pair = z[i >> 1] >> (16 * (i & 1));
            zz = __builtin_amdgcn_perm(0, low ? pair : pair >> 8, 0u);
          } else {
            const int f = F == 4 ? i : F == 2 ? i / 2 : 0;
            zz = __builtin_amdgcn_perm(0, z[0], 0x01010101u * f);
          }
          a[r][2 * i] = Shift(w[i], zz);
          a[r][2 * i + 1] = Shift(w[i] >> 4, zz);
        }
      } else {
        // Nibbles are two's complement here: 16 of them in the high half of a byte.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[r][2 * i] = static_cast<int>((w[i] << 4) & 0xF0F0F0F0u);
          a[r][2 * i + 1] = static_cast<int>(w[i] & 0xF0F0F0F0u);
        }
      }
    }
    floatx4 scale[R][F];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < F; ++f)
        scale[r][f] = *reinterpret_cast<const floatx4 *>(mine + R * kRec + (r + half) * (64 * F) +
                                                         (q * F + f) * 16);
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      if (GC > 1 && g >= groups) continue;
      const int kept = min(c, kCols - 1);
      const uint8_t *dig = st + kDigits + 2 * g * kRec + kept * kUnit;
      const int flip = (kept >> 1) & 7;
      const intx4 b0 = *reinterpret_cast<const intx4 *>(dig + (q ^ flip) * 16);
      const intx4 b1 = *reinterpret_cast<const intx4 *>(dig + ((4 + q) ^ flip) * 16);
      float power[XB];
      const uint8_t *at = st + kPowers + (ONE ? 0 : (g * 16 + c) * XB * 4);
      if constexpr (XB == 1) {
        power[0] = *reinterpret_cast<const float *>(at);
      } else {
        const floatx4 p = *reinterpret_cast<const floatx4 *>(at);
#pragma unroll
        for (int j = 0; j < 4; ++j) power[j] = p[j];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const intx4 a0{a[r][0], a[r][1], a[r][2], a[r][3]}, a1{a[r][4], a[r][5], a[r][6], a[r][7]};
        floatx4 part{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < kFolds; ++f) {
          intx4 sum{0, 0, 0, 0};
          if constexpr (kFolds == 1) {
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b0, sum, 0, 0, 0);
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b1, sum, 0, 0, 0);
          } else if constexpr (kFolds == 2) {
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(f == 0 ? a0 : a1, f == 0 ? b0 : b1, sum, 0,
                                                        0, 0);
          } else {
            const int i = kFolds == 4 ? f : f / 2;
            const intx4 b = i < 2 ? b0 : b1;
            int lo = b[2 * (i & 1)], hi = b[2 * (i & 1) + 1];
            if constexpr (kFolds == 8) {  // half of the 32 values
              const bool use = low == (f % 2 == 0);
              lo = use ? lo : 0;
              hi = use ? hi : 0;
            }
            sum = __builtin_amdgcn_mfma_i32_16x16x32_i8(Long(a[r][2 * i], a[r][2 * i + 1]),
                                                        Long(lo, hi), sum, 0, 0, 0);
          }
          const floatx4 s = scale[r][f * F / kFolds];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float t = static_cast<float>(sum[v]);
            part[v] = f % (kFolds / XB) == 0 ? t * s[v] : fmaf(t, s[v], part[v]);
          }
          if ((f + 1) % (kFolds / XB) == 0) {  // the end of a part with its own power
#pragma unroll
            for (int v = 0; v < 4; ++v)
              acc[r][g][v] = fmaf(part[v], power[f / (kFolds / XB)], acc[r][g][v]);
          }
        }
        // One record's sums at a time where all at once would cost a workgroup's registers.
        if constexpr (GC > 1 && kFolds >= 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// The value `n` lanes up in the row of 16 (0 past its end).
template <int N>
__device__ __forceinline__ float LanesUp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x100 + N, 0xF, 0xF, true));
}

// The sum of a token's digit columns (kTokens apart), in the column of digit 0
// (garbage in the others): v holds this lane's column times 256^digit.
template <bool ONE>
__device__ __forceinline__ float JoinDigits(float v) {
  constexpr int kT = kTokens<ONE>;
  return (LanesUp<2 * kT>(v) + LanesUp<kT>(v)) + v;
}

// What a column's sum counts for: 256^digit, and 1/16 without zero points (the
// weights' bytes hold 16 times their value there).
template <bool ONE, bool ZP>
__device__ __forceinline__ float ColumnWeight(int lane) {
  const int digit = (lane & 15) / kTokens<ONE>;
  if (digit >= kND) return 0.0f;
  const float w = digit == 0 ? 1.0f : digit == 1 ? 256.0f : 65536.0f;
  return ZP ? w : w * 0.0625f;
}

// What the choice gives down: the pairs (token * top_k + place), those of an expert
// one after another, with their weights, cut into segments of up to GC * kTokens
// of one expert: place in that list, length and expert in 12, 8 and 12 bits.
struct Plan {
  int32_t *pair;      // [pairs], by expert and then in order
  float *weight;
  uint32_t *segment;  // [0]: their number, then the segments
};

__device__ __forceinline__ uint32_t MakeSegment(int offset, int n, int expert) {
  return static_cast<uint32_t>(offset) | static_cast<uint32_t>(n) << 12 |
         static_cast<uint32_t>(expert) << 20;
}
__device__ __forceinline__ int Offset(uint32_t segment) { return segment & 0xFFFu; }
__device__ __forceinline__ int Count(uint32_t segment) { return (segment >> 12) & 0xFFu; }
__device__ __forceinline__ int Expert(uint32_t segment) { return segment >> 20; }

// The segments of up to `most` pairs, by a whole workgroup; counts: LDS.
__device__ __forceinline__ void CutSegments(const int32_t *pair_expert, int pairs, int experts,
                                            int most, int32_t *counts, uint32_t *segment) {
  const int tid = threadIdx.x, lane = tid & 63, threads = blockDim.x;
  for (int e = tid; e < experts; e += threads) counts[e] = 0;
  __syncthreads();
  for (int p = tid; p < pairs; p += threads) atomicAdd(&counts[pair_expert[p]], 1);
  __syncthreads();
  if (tid >= 64) return;
  int at = 0, offset = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int n = e0 + lane < experts ? counts[e0 + lane] : 0;
    const int cut = (n + most - 1) / most;
    int end = cut, last = n;  // inclusive sums over the lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int a = __shfl_up(end, off, 64), b = __shfl_up(last, off, 64);
      if (lane >= off) {
        end += a;
        last += b;
      }
    }
    for (int j = 0; j < cut; ++j)
      segment[1 + at + end - cut + j] =
          MakeSegment(offset + last - n + j * most, min(n - j * most, most), e0 + lane);
    at += __shfl(end, 63, 64);
    offset += __shfl(last, 63, 64);
  }
  if (lane == 0) segment[0] = at;
}

// The pairs that chose expert e, in order, and how many chose a lower one: by
// every thread of one wavefront.
__device__ __forceinline__ int CollectPairs(const int32_t *pair_expert, int pairs, int e,
                                            int32_t *out, int *before) {
  const int lane = threadIdx.x & 63;
  int n = 0, lower = 0;
  for (int p0 = 0; p0 < pairs; p0 += 64) {
    const int p = p0 + lane;
    const int who = p < pairs ? pair_expert[p] : kMaxExperts;
    const uint64_t mask = __ballot(who == e);
    if (who == e) out[n + __popcll(mask & ((uint64_t{1} << lane) - 1))] = p;
    n += __popcll(mask);
    lower += __popcll(__ballot(who < e));
  }
  *before = lower;
  return n;
}

// CHOOSE: of one token, whose choice each workgroup makes from its logits.
struct Choice {
  const float *logits;
  int32_t *ids;
  float *weights;
  int experts;
  bool normalize;
};

// Wavefronts per SIMD that the registers are to leave room for: three workgroups of
// eight a CU for one column group, two for several, one where two would spill.
constexpr int WavesPerSimd(int gc, int folds) {
  return gc * folds >= 16 ? 2 : gc > 1 || folds == 8 ? 4 : 6;
}

// Gate/up: workgroup (b, i) the channels of block b of entry i's expert, 16
// (gate and up) for each of GROUPS wavefronts that share a pipe, or, with KS runs
// of the units, for each of GROUPS * KS wavefronts with pipes of their own. Bound by
// reading: one token of 4096 x 14336, 2 of 8 experts, 25 us (5.1 TB/s); one of 2048 x
// 1024, 6 of 64, 9 to 11 us, its launch and two round trips; 64 tokens of 4096 x 14336
// 119 us, 4.2 TB/s counting each weight once: experts of more than 20 tokens, one in
// ten of even choices, read theirs twice.
template <bool ONE, int GC, int F, bool ZP, int GROUPS, int KS, int NS, bool CHOOSE>
__global__ __launch_bounds__(64 * GROUPS *KS,
                             GROUPS == 8 ? WavesPerSimd(GC, F) : 1) void MoeGateUpKernel(
    Matrix m, Fixed fx, Fixed fh, const int32_t *__restrict__ pair_expert,
    const float *__restrict__ pair_weight, Plan plan, int pairs, int top_k, bool by_expert,
    Choice choice) {
  using P = Pipe<ONE, GC, 2, F, 1, ZP, KS == 1 ? GROUPS : 1, NS>;
  constexpr int kT = P::kT, kChannels = 16 * GROUPS, kWaves = GROUPS * KS;
  constexpr int kPipes = KS == 1 ? 1 : kWaves;
  static_assert(kPipes * P::kLds >= GC * kT * kChannels * 4 + (KS - 1) * GROUPS * GC * 2048,
                "the activations and the runs' sums reuse the pipes' LDS");
  extern __shared__ uint4 dynamic[];
  __shared__ int32_t list[kMaxTokens];
  __shared__ int32_t shared_n;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int entry = blockIdx.y;
  int e;
  if constexpr (CHOOSE) {
    __shared__ float best[kMaxTopK];
    __shared__ int32_t who[kMaxTopK];
    static_assert(kPipes * P::kLds >= kMaxExperts * 4, "the keys use the pipes' LDS");
    Choose<64 * kWaves>(choice.logits, choice.experts, top_k, reinterpret_cast<uint32_t *>(dynamic),
                        best, who);
    e = __builtin_amdgcn_readfirstlane(who[entry]);
    if (blockIdx.x == 0) {
      const float total = WeightSum<64 * kWaves>(choice.logits, choice.experts, top_k,
                                                 choice.normalize, best);
      if (tid == 0) {
        const float p = expf(best[entry] - best[0]) / total;
        plan.pair[entry] = entry;
        plan.weight[entry] = p;
        plan.segment[1 + entry] = MakeSegment(entry, 1, e);
        if (entry == 0) plan.segment[0] = top_k;
        if (choice.ids) choice.ids[entry] = e;
        if (choice.weights) choice.weights[entry] = p;
      }
    }
    if (tid == 0) {
      list[0] = entry;
      shared_n = 1;
    }
  } else {
    if (entry == static_cast<int>(gridDim.y) - 1) {  // the last row's first workgroup
      static_assert(kPipes * P::kLds >= kMaxExperts * 4, "the counts use the pipes' LDS");
      if (blockIdx.x == 0)
        CutSegments(pair_expert, pairs, choice.experts, GC * kT, reinterpret_cast<int32_t *>(dynamic),
                    plan.segment);
      return;
    }
    e = by_expert ? entry : pair_expert[entry];
    if (wave == 0) {
      int before;
      int n = CollectPairs(pair_expert, pairs, e, list, &before);
      // Of the pairs that share an expert the first one works.
      if (!by_expert && list[0] != entry) n = 0;
      if (lane == 0) shared_n = n;
      if (blockIdx.x == 0 && lane < n) {
        plan.pair[before + lane] = list[lane];
        plan.weight[before + lane] = pair_weight[list[lane]];
      }
    }
  }
  __syncthreads();
  const int n = __builtin_amdgcn_readfirstlane(shared_n);
  if (n == 0) return;
  const int c = lane & 15, q = lane >> 4;
  const float weight = ColumnWeight<ONE, ZP>(lane);
  const int cg = wave % GROUPS, ks = wave / GROUPS;
  P pipe(reinterpret_cast<const uint8_t *>(dynamic) + (KS == 1 ? 0 : wave * P::kLds), lane,
         KS == 1 ? wave : 0);
  float *hidden = reinterpret_cast<float *>(dynamic);  // [GC * kT][kChannels]
  floatx4 *sums = reinterpret_cast<floatx4 *>(hidden + GC * kT * kChannels);
  const int units = static_cast<int>(m.units);
  const int u0 = units * ks / KS, u1 = units * (ks + 1) / KS;
  // Workgroups start at different units (KS = 1): in step they would ask the same
  // memory channels (2 to 4% slower at 16 tokens of 128 experts, 64 of 8).
  const int rot = KS == 1 ? (blockIdx.x * 7 + blockIdx.y * 3) % units : 0;
  auto turn = [&](int u) __attribute__((always_inline)) {
    return u + rot >= units && KS == 1 ? u + rot - units : u + rot;
  };
  for (int t0 = 0; t0 < n; t0 += GC * kT) {
    const int left = min(n - t0, GC * kT), groups = (left + kT - 1) / kT;
    floatx4 acc[2][GC];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int g = 0; g < GC; ++g) acc[r][g] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (u0 < u1) {
      pipe.Segment(m, e, static_cast<int64_t>(blockIdx.x) * GROUPS + cg, fx, left,
                   [&](int i) { return list[t0 + i] / top_k; });
#pragma unroll
      for (int p = 0; p < NS - 1; ++p) pipe.Issue(fx, turn(min(u0 + p, u1 - 1)), p);
      int stage = 0;
      for (int u = u0; u < u1; ++u) {
        P::template Wait<P::kOps *(NS - 2)>();
        pipe.Issue(fx, turn(min(u + NS - 1, u1 - 1)), stage == 0 ? NS - 1 : stage - 1);
        pipe.Multiply(stage, groups, acc);
        stage = stage + 1 == NS ? 0 : stage + 1;
      }
      P::template Wait<0>();
    }
    if constexpr (KS > 1) {
      __syncthreads();
      if (ks > 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int g = 0; g < GC; ++g)
            sums[((wave - GROUPS) * 2 * GC + r * GC + g) * 64 + lane] = acc[r][g];
      }
      __syncthreads();
    }
    if (ks == 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int g = 0; g < GC; ++g)
#pragma unroll
          for (int s = 1; s < KS; ++s)
            acc[r][g] += sums[(((s - 1) * GROUPS + cg) * 2 * GC + r * GC + g) * 64 + lane];
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        floatx4 h;
#pragma unroll
        for (int v = 0; v < 4; ++v)
          h[v] = SiluMul(JoinDigits<ONE>(acc[0][g][v] * weight),
                         JoinDigits<ONE>(acc[1][g][v] * weight));
        if (c < kT)
          *reinterpret_cast<floatx4 *>(hidden + (g * kT + c) * kChannels + 16 * cg + 4 * q) = h;
      }
    }
    __syncthreads();
    constexpr int kPer = kChannels / 8;  // threads of a token
    for (int i = tid / kPer; i < GC * kT; i += 64 * kWaves / kPer) {
      if (i >= left) continue;
      const int k = tid % kPer;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = hidden[i * kChannels + 8 * k + j];
      const int64_t k0 = static_cast<int64_t>(blockIdx.x) * (kChannels / 8) + k;  // eights of the row
      StoreUnit(fh, list[t0 + i], k0 >> 4, static_cast<int>(k0 & 15), x);
    }
    __syncthreads();
  }
}

// Down, few tokens on few experts: a workgroup takes 16 columns of Y. The
// items (segment, unit) of the layer are cut into eight equal runs, one for each
// wavefront and its pipe, which adds each segment's rows, times the tokens'
// weights, to sums of its own; they join in order. One token of 4096 x 14336, 2 of 8:
// 20 us, 3.1 TB/s; neither copies eight deep nor sixteen wavefronts changed that.
template <bool ONE, int F, bool ZP, int NS, typename T>
__global__ __launch_bounds__(512) void MoeDownNarrowKernel(Matrix m, Fixed fh, Plan plan,
                                                           T *__restrict__ Y, int pairs,
                                                           int most_segments, int tokens, int top_k,
                                                           int64_t H) {
  using P = Pipe<ONE, 1, 1, F, 4, ZP, 1, NS>;
  constexpr int kT = P::kT;
  // The pipes' LDS, then sums [8][tokens][16], the pairs' weights, the segments and
  // the list of pairs.
  extern __shared__ uint4 dynamic[];
  uint8_t *lds = reinterpret_cast<uint8_t *>(dynamic);
  float *sums = reinterpret_cast<float *>(lds + 8 * P::kLds);
  float *weights = sums + 8 * tokens * 16;
  uint32_t *segments = reinterpret_cast<uint32_t *>(weights + pairs);
  uint16_t *list = reinterpret_cast<uint16_t *>(segments + most_segments + 1);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int i = tid; i < pairs; i += 512) {
    list[i] = static_cast<uint16_t>(plan.pair[i]);
    weights[i] = plan.weight[i];
  }
  for (int i = tid; i <= most_segments; i += 512) segments[i] = plan.segment[i];
  float *mine = sums + wave * tokens * 16;
  for (int i = lane; i < tokens * 16; i += 64) mine[i] = 0.0f;
  __syncthreads();
  const int units = static_cast<int>(m.units);
  const int items = __builtin_amdgcn_readfirstlane(segments[0]) * units;
  ++segments;
  const int i0 = items * wave / 8, i1 = items * (wave + 1) / 8;
  const int c = lane & 15, q = lane >> 4;
  const float weight = ColumnWeight<ONE, ZP>(lane);
  if (i0 < i1) {
    P pipe(lds + wave * P::kLds, lane, 0, blockIdx.x & 1);
    // The next item to copy.
    int next_seg = i0 / units, next_u = i0 % units;
    const int last_seg = (i1 - 1) / units, last_u = (i1 - 1) % units;
    auto enter = [&](int seg) __attribute__((always_inline)) {
      const uint32_t s = __builtin_amdgcn_readfirstlane(segments[seg]);
      pipe.Segment(m, Expert(s), blockIdx.x >> 1, fh, Count(s),
                   [&](int i) { return list[Offset(s) + i]; });
    };
    auto issue = [&](int stage) __attribute__((always_inline)) {
      pipe.Issue(fh, next_u, stage);
      if (next_seg == last_seg && next_u == last_u) return;  // past the end: the last again
      if (++next_u == units) {
        next_u = 0;
        enter(++next_seg);
      }
    };
    enter(next_seg);
    int seg = next_seg, u = next_u;  // the item to multiply
#pragma unroll
    for (int p = 0; p < NS - 1; ++p) issue(p);
    int stage = 0;
    floatx4 acc[1][1] = {{floatx4{0.f, 0.f, 0.f, 0.f}}};
    for (int i = i0; i < i1; ++i) {
      P::template Wait<P::kOps *(NS - 2)>();
      issue(stage == 0 ? NS - 1 : stage - 1);
      pipe.Multiply(stage, 1, acc);
      stage = stage + 1 == NS ? 0 : stage + 1;
      if (++u == units || i + 1 == i1) {
        const uint32_t now = __builtin_amdgcn_readfirstlane(segments[seg]);
        floatx4 y;
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = JoinDigits<ONE>(acc[0][0][v] * weight);
        acc[0][0] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (c < kT && c < Count(now)) {
          const float p = weights[Offset(now) + c];
          floatx4 *to = reinterpret_cast<floatx4 *>(mine + list[Offset(now) + c] / top_k * 16 + 4 * q);
          floatx4 s = *to;
#pragma unroll
          for (int v = 0; v < 4; ++v) s[v] = fmaf(p, y[v], s[v]);
          *to = s;
        }
        u = 0;
        ++seg;
      }
    }
    P::template Wait<0>();  // no copy may land after the workgroup
  }
  __syncthreads();
  for (int i = tid; i < tokens * 16; i += 512) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 16 + (i & 15);
    if (n >= H) continue;
    float y = sums[i];
    for (int w = 1; w < 8; ++w) y += sums[w * tokens * 16 + i];
    Y[(i >> 4) * H + n] = static_cast<T>(y);
  }
}

// Down otherwise: a workgroup takes 256 columns of Y and part blockIdx.y % cuts of the
// units of one segment. Every pair's row, times its weight, goes to parts
// [cuts][pairs][width]. 64 tokens of 4096 x 14336, 2 of 8: 55 us where no expert has
// more than 20 tokens (4.5 TB/s), 72 where one or two have.
template <bool ONE, int GC, int F, bool ZP, int NS>
__global__ __launch_bounds__(512, WavesPerSimd(GC, F)) void MoeDownKernel(Matrix m, Fixed fh, Plan plan,
                                                     float *__restrict__ parts, int pairs, int cuts,
                                                     int64_t width) {
  using P = Pipe<ONE, GC, 2, F, 1, ZP, 8, NS>;
  constexpr int kT = P::kT;
  extern __shared__ uint4 dynamic[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int cut = blockIdx.y % cuts, units = static_cast<int>(m.units);
  const int seg = blockIdx.y / cuts;
  if (seg >= __builtin_amdgcn_readfirstlane(static_cast<int>(plan.segment[0]))) return;
  const int u0 = units * cut / cuts, u1 = units * (cut + 1) / cuts;
  if (u0 >= u1) return;
  const int c = lane & 15, q = lane >> 4;
  const float weight = ColumnWeight<ONE, ZP>(lane);
  const int64_t group = min(static_cast<int64_t>(blockIdx.x) * 8 + wave, m.groups - 1);
  float *out = parts + static_cast<int64_t>(cut) * pairs * width +
               static_cast<int64_t>(blockIdx.x) * 256 + wave * 32 + 4 * q;
  P pipe(reinterpret_cast<const uint8_t *>(dynamic), lane, wave);
  const uint32_t now = __builtin_amdgcn_readfirstlane(plan.segment[1 + seg]);
  const int n = Count(now), groups = (n + kT - 1) / kT;
  pipe.Segment(m, Expert(now), group, fh, n, [&](int i) { return plan.pair[Offset(now) + i]; });
#pragma unroll
  for (int p = 0; p < NS - 1; ++p) pipe.Issue(fh, min(u0 + p, u1 - 1), p);
  int stage = 0;
  floatx4 acc[2][GC];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int g = 0; g < GC; ++g) acc[r][g] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int u = u0; u < u1; ++u) {
    P::template Wait<P::kOps *(NS - 2)>();
    pipe.Issue(fh, min(u + NS - 1, u1 - 1), stage == 0 ? NS - 1 : stage - 1);
    pipe.Multiply(stage, groups, acc);
    stage = stage + 1 == NS ? 0 : stage + 1;
  }
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    const int j = g * kT + c;
    const bool on = c < kT && j < n;
    const int at = Offset(now) + (on ? j : 0);
    const float p = plan.weight[at];
    float *to = out + plan.pair[at] * width;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      floatx4 y;
#pragma unroll
      for (int v = 0; v < 4; ++v) y[v] = p * JoinDigits<ONE>(acc[r][g][v] * weight);
      if (on) *reinterpret_cast<floatx4 *>(to + 16 * r) = y;
    }
  }
  P::template Wait<0>();  // no copy may land after the workgroup
}

// Y[t] = the sum of the parts of t's top_k pairs, in order; a thread's loads of
// eight of them are in flight together.
template <typename T>
__global__ __launch_bounds__(256) void MoeSumKernel(const float *__restrict__ parts,
                                                    T *__restrict__ Y, int64_t H, int64_t width,
                                                    int top_k, int pairs, int cuts) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int t = blockIdx.y;
  if (n >= H) return;
  const int terms = top_k * cuts;
  float y = 0.0f;
  for (int i = 0; i < terms; i += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = min(i + j, terms - 1);
      const int64_t row = static_cast<int64_t>(at / top_k) * pairs + t * top_k + at % top_k;
      v[j] = parts[row * width + n];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < terms) y += v[j];
  }
  Y[t * H + n] = static_cast<T>(y);
}

// ---- weight layout -----------------------------------------------------------------

// The record of 16-row group `group` (of `groups` in a matrix) and unit u.
__device__ __forceinline__ int64_t RecordOf(Half half, int64_t matrix, int64_t group, int64_t u,
                                            int64_t groups, int64_t units) {
  if (half == Half::kPair)
    return ((matrix * groups + (group & ~int64_t{1})) / 2 * units + u) * 2 + (group & 1);
  return ((matrix * groups + group) * units + u) * 2 + static_cast<int>(half);
}

// One thread per 16 bytes of a record.
__global__ __launch_bounds__(256) void MoeRecordKernel(const uint8_t *__restrict__ B,
                                                       uint8_t *__restrict__ rec, int64_t N,
                                                       int64_t K, int64_t row_bytes, int64_t groups,
                                                       int64_t units, Half half, uint32_t flip,
                                                       int64_t total) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int lane = static_cast<int>(i & 63);
  const int64_t id = i >> 6;  // (matrix, group of 16 rows, unit)
  const int64_t u = id % units, mg = id / units, matrix = mg / groups, group = mg - matrix * groups;
  const int64_t n = group * 16 + (lane & 15);
  uint32_t out[4] = {0, 0, 0, 0};
  if (n < N) {
    const uint8_t *row = B + (matrix * N + n) * row_bytes;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int64_t k = u * kUnit + 32 * w + 8 * (lane >> 4);
      if (k >= K) continue;
      // Values past K are multiplied by zero digits.
      const uint32_t v = *reinterpret_cast<const uint32_t *>(row + k / 2) ^ flip;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[w] |= ((v >> (4 * j)) & 15u) << (8 * j) | ((v >> (4 * j + 16)) & 15u) << (8 * j + 4);
    }
  }
  reinterpret_cast<uint4 *>(rec)[RecordOf(half, matrix, group, u, groups, units) * 64 + lane] =
      make_uint4(out[0], out[1], out[2], out[3]);
}

// One thread per scale (and zero point) of a record.
__global__ __launch_bounds__(256) void MoeScaleKernel(const float *__restrict__ S,
                                                      const uint8_t *__restrict__ Z,
                                                      uint8_t *__restrict__ meta, int64_t N,
                                                      int64_t nb, int64_t groups, int64_t units,
                                                      int folds, int block_size, Half half,
                                                      int64_t total) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int per = 16 * folds;
  const int row = static_cast<int>(i % per) / folds, f = static_cast<int>(i % per) % folds;
  const int64_t id = i / per;
  const int64_t u = id % units, mg = id / units, matrix = mg / groups, group = mg - matrix * groups;
  const int64_t n = group * 16 + row;
  const int64_t b = block_size >= kUnit ? u * kUnit / block_size : u * folds + f;
  float s = 0.0f;
  int z = 0;
  if (n < N && b < nb) {
    s = S[(matrix * N + n) * nb + b];
    if (Z) z = (Z[(matrix * N + n) * ((nb + 1) / 2) + b / 2] >> (4 * (b & 1))) & 15;
  }
  const int64_t record = RecordOf(half, matrix, group, u, groups, units);
  constexpr int R = kRecords;
  const int r = static_cast<int>(record % R);
  uint8_t *m = meta + record / R * MetaBytes(folds, Z != nullptr);
  reinterpret_cast<float *>(m)[r * per + ((row >> 2) * folds + f) * 4 + (row & 3)] = s;
  if (Z) m[R * per * 4 + (r * 16 + row) * folds + f] = static_cast<uint8_t>(z);
}

// ---- launches ------------------------------------------------------------------------

struct Work {
  Fixed fx, fh;
  float *logits, *pair_weight, *parts;
  int32_t *pair_expert;
  Plan plan;
  size_t bytes;
};

// Up to this many tokens the sums of down's eight wavefronts fit beside their pipes.
constexpr int kNarrowTokens = 8;

// How the experts' launches are cut.
struct Shape {
  int entries;
  bool narrow;  // gate/up: 32 channels a workgroup, powers of two per 32 channels
  bool split;   // ... and the units over four wavefronts each
  bool choose;  // one token: the gate/up kernel makes its choice
  int groups;   // column groups per pass over an expert's rows
  int segments; // at most
  int cuts;     // down: runs of 1 / cuts of a segment
};

Shape PickShape(const Layer &l, int tokens) {
  Shape s;
  s.entries = std::min(tokens * l.top_k, l.experts);
  const int64_t blocks = s.entries * CeilDiv(l.intermediate, 128);  // of 128 channels
  // Narrow workgroups, and down with the sum over the experts, where blocks of 128
  // channels leave CUs idle (us, narrow and not; one token of hidden 4096, experts of
  // 14336: 1 chosen 35 and 48, 2 chosen 52 and 61, 4 chosen 92 and 86; 2 tokens of
  // 4096 x 2048, 2 of 16: 25 and 41; 4 tokens of 2048 x 1024, 4 of 64: 33 and 30; 8
  // tokens, 6 of 64: 65 and 44).
  s.narrow = tokens <= kNarrowTokens && blocks < (tokens == 1 ? l.num_cus : 3 * l.num_cus / 8);
  // The units over four wavefronts each: one token of 2048 x 1024, 6 of 64: 19 us,
  // 23 without; one of 4096 x 14336, 2 of 8, whose workgroups fill the chip: 64, 52 without.
  s.split = s.narrow && 2 * blocks <= l.num_cus;
  // A workgroup's choice among more experts takes longer than a launch of its own (6 of
  // 64: 19 us, 21 with a launch).
  s.choose = tokens == 1 && l.experts <= 256;
  // What most experts' tokens fill: their mean share and two standard deviations
  // of even choices (us with one, two and four groups: 32 tokens of 4096 x 4096, 2 of 8:
  // 100, 79 and 77; 64 of 2048 x 1024, 8 of 64: 123, 116 and 105, 8 of 128: 149, 145 and
  // 162; 24 of 2048 x 1408, 4 of 60: 75, 85 and 90). Where two experts are chosen by half
  // of the tokens each, the same number is the best of the three, or within 1% of it:
  // 151, 123 and 108; 159, 138 and 120, 193, 165 and 169; 77, 77 and 82.
  const int group = tokens == 1 ? 1 : kTokens<false>;
  const double mean = static_cast<double>(tokens) * l.top_k / l.experts;
  const double most = std::min<double>(tokens, mean + 2.0 * std::sqrt(mean));
  // Four groups of 16-wide blocks would not fit the registers.
  s.groups = tokens <= kNarrowTokens || most <= group ? 1
             : most <= 2 * group || l.folds == 8     ? 2
                                                     : 4;
  s.segments = s.entries + tokens * l.top_k / (s.groups * group);
  // Down: about two workgroups a CU, of at least four units (32 tokens of 4096 x 4096,
  // 2 of 8: 77 us, 83 with whole rows; 4 of 4096 x 14336: 112 and 167).
  const double share = static_cast<double>(l.top_k) / l.experts;
  const double met = l.experts * (1.0 - std::pow(1.0 - share, tokens));
  const double blocks_down = std::max(1.0, met) * CeilDiv(l.hidden, 256);
  s.cuts = 1;
  while (blocks_down * s.cuts < 1.5 * l.num_cus && l.down.units >= 8 * s.cuts && s.cuts < 8)
    s.cuts *= 2;
  return s;
}

int64_t PartWidth(const Layer &l) { return CeilDiv(l.hidden, 256) * 256; }

Work Split(const Layer &l, int T, void *base) {
  Work w;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *p = static_cast<char *>(base) + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const size_t pairs = static_cast<size_t>(T) * l.top_k;
  const Shape shape = PickShape(l, T);
  auto fixed = [&](size_t rows, int64_t units, int scales) {
    Fixed f;
    f.units = units;
    f.scales = scales;
    f.dig = reinterpret_cast<int8_t *>(take(rows * kND * units * kUnit));
    f.power = reinterpret_cast<float *>(take(rows * units * scales * 4));
    return f;
  };
  w.fx = fixed(T, l.gate_up.units, 1);
  w.fh = fixed(pairs, l.down.units, shape.narrow ? 4 : 1);
  w.logits = reinterpret_cast<float *>(take(static_cast<size_t>(T) * l.experts * 4));
  w.pair_expert = reinterpret_cast<int32_t *>(take(pairs * 4));
  w.pair_weight = reinterpret_cast<float *>(take(pairs * 4));
  w.plan.pair = reinterpret_cast<int32_t *>(take(pairs * 4));
  w.plan.weight = reinterpret_cast<float *>(take(pairs * 4));
  w.plan.segment = reinterpret_cast<uint32_t *>(take((shape.segments + 1) * 4));
  w.parts = reinterpret_cast<float *>(
      take(shape.narrow ? 0 : static_cast<size_t>(shape.cuts) * pairs * PartWidth(l) * 4));
  w.bytes = at;
  return w;
}

template <bool ONE, int GC, int F, bool ZP, int GROUPS, int KS, bool CHOOSE>
hipError_t LaunchGateUp(const Layer &l, const Work &w, const Shape &shape, int pairs,
                        const Choice &choice, hipStream_t s) {
  constexpr int NS = KS > 1 && ONE ? 4 : GC == 1 && GROUPS == 8 ? 2 : 3;
  using P = Pipe<ONE, GC, 2, F, 1, ZP, KS == 1 ? GROUPS : 1, NS>;
  const dim3 grid(static_cast<unsigned>(l.gate_up.groups / GROUPS),
                  static_cast<unsigned>(shape.entries + (CHOOSE ? 0 : 1)));
  hipLaunchKernelGGL((MoeGateUpKernel<ONE, GC, F, ZP, GROUPS, KS, NS, CHOOSE>), grid,
                     dim3(64 * GROUPS * KS), (KS == 1 ? 1 : GROUPS * KS) * P::kLds, s, l.gate_up,
                     w.fx, w.fh, w.pair_expert, w.pair_weight, w.plan, pairs, l.top_k,
                     pairs >= l.experts, choice);
  return hipGetLastError();
}

template <bool ONE, int F, bool ZP, typename T>
hipError_t LaunchDownNarrow(const Layer &l, const Work &w, const Shape &shape, int tokens, T *Y,
                            hipStream_t s) {
  constexpr int NS = ONE ? 5 : 3;
  using P = Pipe<ONE, 1, 1, F, 4, ZP, 1, NS>;
  const int pairs = tokens * l.top_k;
  const size_t lds = static_cast<size_t>(8) * P::kLds + 8 * tokens * 16 * sizeof(float) + pairs * 6 +
                     (shape.segments + 1) * 4;
  hipLaunchKernelGGL((MoeDownNarrowKernel<ONE, F, ZP, NS, T>),
                     dim3(static_cast<unsigned>(2 * l.down.groups)), dim3(512), lds, s, l.down, w.fh,
                     w.plan, Y, pairs, shape.segments, tokens, l.top_k, l.hidden);
  return hipGetLastError();
}

template <bool ONE, int GC, int F, bool ZP, typename T>
hipError_t LaunchDown(const Layer &l, const Work &w, const Shape &shape, int tokens, T *Y,
                      hipStream_t s) {
  constexpr int NS = GC == 1 ? 2 : 3;
  using P = Pipe<ONE, GC, 2, F, 1, ZP, 8, NS>;
  const int pairs = tokens * l.top_k;
  const int64_t width = PartWidth(l);
  const dim3 grid(static_cast<unsigned>(width / 256),
                  static_cast<unsigned>(shape.segments * shape.cuts));
  hipLaunchKernelGGL((MoeDownKernel<ONE, GC, F, ZP, NS>), grid, dim3(512), P::kLds, s, l.down,
                     w.fh, w.plan, w.parts, pairs, shape.cuts, width);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((MoeSumKernel<T>),
                     dim3(static_cast<unsigned>(CeilDiv(l.hidden, 256)), static_cast<unsigned>(tokens)),
                     dim3(256), 0, s, w.parts, Y, l.hidden, width, l.top_k, pairs, shape.cuts);
  return hipGetLastError();
}

template <bool ONE, int GC, int F, bool ZP, int GROUPS, int KS>
hipError_t LaunchGateUpC(const Layer &l, const Work &w, const Shape &shape, int pairs,
                         const Choice &choice, hipStream_t s) {
  if constexpr (ONE) {
    if (shape.choose)
      return LaunchGateUp<ONE, GC, F, ZP, GROUPS, KS, true>(l, w, shape, pairs, choice, s);
  }
  return LaunchGateUp<ONE, GC, F, ZP, GROUPS, KS, false>(l, w, shape, pairs, choice, s);
}

template <bool ONE, int GC, int F, bool ZP, typename T>
hipError_t LaunchExperts(const Layer &l, const Work &w, const Shape &shape, int tokens, T *Y,
                         const Choice &choice, hipStream_t s) {
  const int pairs = tokens * l.top_k;
  hipError_t e = hipSuccess;
  if constexpr (GC == 1) {
    if (shape.narrow) {
      bool split = true;
      if constexpr (ONE) {  // several tokens' narrow layers are always small enough
        split = shape.split;
        if (!split) e = LaunchGateUpC<ONE, GC, F, ZP, 2, 1>(l, w, shape, pairs, choice, s);
      }
      if (split) e = LaunchGateUpC<ONE, GC, F, ZP, 2, 4>(l, w, shape, pairs, choice, s);
      return e != hipSuccess ? e : LaunchDownNarrow<ONE, F, ZP, T>(l, w, shape, tokens, Y, s);
    }
  }
  e = LaunchGateUpC<ONE, GC, F, ZP, 8, 1>(l, w, shape, pairs, choice, s);
  return e != hipSuccess ? e : LaunchDown<ONE, GC, F, ZP, T>(l, w, shape, tokens, Y, s);
}

template <bool ONE, int GC, bool ZP, typename T>
hipError_t LaunchFolds(const Layer &l, const Work &w, const Shape &shape, int tokens, T *Y,
                       const Choice &choice, hipStream_t s) {
  switch (l.folds) {
  case 1: return LaunchExperts<ONE, GC, 1, ZP, T>(l, w, shape, tokens, Y, choice, s);
  case 2: return LaunchExperts<ONE, GC, 2, ZP, T>(l, w, shape, tokens, Y, choice, s);
  case 4: return LaunchExperts<ONE, GC, 4, ZP, T>(l, w, shape, tokens, Y, choice, s);
  default: break;
  }
  if constexpr (GC < 4) return LaunchExperts<ONE, GC, 8, ZP, T>(l, w, shape, tokens, Y, choice, s);
  else return hipErrorInvalidValue;  // PickShape gives eight folds no four groups
}

template <typename T>
hipError_t LaunchLayerT(const Layer &l, int tokens, const void *X, const float *logits, void *Y,
                        int32_t *ids, float *weights, void *work, hipStream_t s) {
  const Work w = Split(l, tokens, work);
  constexpr int kRT = 4;
  const int router_wgs =
      logits ? 0 : l.experts * (tokens == 1 ? 1 : static_cast<int>(CeilDiv(tokens, kRT)));
  const unsigned prep =
      static_cast<unsigned>(router_wgs + CeilDiv(tokens * l.gate_up.units, 16));
  const bool vec = l.hidden % 4 == 0 && reinterpret_cast<uintptr_t>(X) % (4 * sizeof(T)) == 0;
  auto launch_prep = [&](auto rt, auto v) {
    hipLaunchKernelGGL((MoePrepKernel<decltype(rt)::value, decltype(v)::value, T>), dim3(prep),
                       dim3(256), 0, s, static_cast<const T *>(X), l.router, w.logits, w.fx, tokens,
                       l.hidden, l.experts, router_wgs);
  };
  using One = std::integral_constant<int, 1>;
  using Several = std::integral_constant<int, kRT>;
  if (tokens == 1) vec ? launch_prep(One{}, std::true_type{}) : launch_prep(One{}, std::false_type{});
  else vec ? launch_prep(Several{}, std::true_type{}) : launch_prep(Several{}, std::false_type{});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const Shape shape = PickShape(l, tokens);
  const Choice choice{logits ? logits : w.logits, ids, weights, l.experts, l.normalize};
  if (!shape.choose) {
    hipLaunchKernelGGL(MoeRouteKernel, dim3(static_cast<unsigned>(tokens)), dim3(256), 0, s,
                       choice.logits, w.pair_expert, w.pair_weight, ids, weights, l.experts,
                       l.top_k, l.normalize);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  T *y = static_cast<T *>(Y);
  auto experts = [&](auto groups, auto one) {
    constexpr int GC = decltype(groups)::value;
    constexpr bool kOne = decltype(one)::value;
    return l.zeros ? LaunchFolds<kOne, GC, true, T>(l, w, shape, tokens, y, choice, s)
                   : LaunchFolds<kOne, GC, false, T>(l, w, shape, tokens, y, choice, s);
  };
  if (tokens == 1) return experts(std::integral_constant<int, 1>{}, std::true_type{});
  switch (shape.groups) {
  case 1: return experts(std::integral_constant<int, 1>{}, std::false_type{});
  case 2: return experts(std::integral_constant<int, 2>{}, std::false_type{});
  default: return experts(std::integral_constant<int, 4>{}, std::false_type{});
  }
}

} // namespace

hipError_t LaunchRelayout(const mnb_moe_weight &src, int64_t N, int64_t K, int block_size,
                          int experts, Half half, const Matrix &m, uint8_t *rec, uint8_t *meta,
                          hipStream_t s) {
  const int64_t groups = half == Half::kPair ? 2 * m.groups : m.groups, units = m.units;
  const int64_t nb = CeilDiv(K, block_size);
  const int64_t row_bytes = nb * (block_size / 2);
  const int folds = std::max(1, kUnit / block_size);
  const bool zeros = src.zero_points != nullptr;
  // Experts at a time, so that a grid's threads stay below 2^32 (one expert's
  // are at most 2^31: hidden * intermediate <= 2^34).
  const int64_t one = groups * units * std::max(64, 16 * folds);
  const int64_t per = std::max<int64_t>(1, (int64_t{1} << 31) / one);
  for (int64_t e = 0; e < experts; e += per) {
    const int64_t n = std::min<int64_t>(per, experts - e);
    const int64_t total = n * groups * units;
    const int64_t first = e * m.groups * units;
    hipLaunchKernelGGL(MoeRecordKernel, dim3(static_cast<unsigned>(CeilDiv(total * 64, 256))),
                       dim3(256), 0, s, src.B + e * N * row_bytes, rec + first * kRecords * kRec, N,
                       K, row_bytes, groups, units, half, zeros ? 0u : 0x88888888u, total * 64);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(MoeScaleKernel, dim3(static_cast<unsigned>(CeilDiv(total * 16 * folds, 256))),
                       dim3(256), 0, s, src.scales + e * N * nb,
                       zeros ? src.zero_points + e * N * ((nb + 1) / 2) : nullptr,
                       meta + first * MetaBytes(folds, zeros), N, nb, groups, units, folds,
                       block_size, half, total * 16 * folds);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

size_t WorkBytes(const Layer &l, int T) { return Split(l, T, nullptr).bytes; }

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

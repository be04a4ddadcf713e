// The 8-bit product on CDNA4's e4m3 MFMA (16x16x128: one instruction per
// block of 128 values of K).
//
// A block's scales are one weight scale s_w (shared by 128 columns) and one
// row scale s_a, so each block's partial product p = a . w starts from zero
// in the MFMA and joins the fp32 sum as acc += p * (s_a s_w). The weights are
// the MFMA's row operand: a lane's four results are four columns of Y for one
// row, so s_a s_w is one value per lane and fragment.
//
// The e4m3 MFMA adds its products in groups of eight, each product cut off
// 13 bits below the group's largest (measured; between groups it adds in
// fp32): up to 7 2^-13 of the sum of the products' magnitudes, 1.4e-5 of Y where
// all are of one size, all of a small product beside a large one. A bfloat16 Y takes
// it: that is less than half of bfloat16's own rounding, 2^-9, of the same sum, and
// the codes stand for values that were rounded by up to 2^-4. float16 rounds by
// 2^-12, so for it and for an fp32 Y both operands are widened to fp16 (EXACT), where
// e4m3 values and their products are exact, for four fp16 MFMAs (16x16x32) at twice
// the matrix time.
#include "mnb_fp8.h"

#include <type_traits>
#include <utility>

namespace mnb {
namespace fp8 {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// Whether a Y of type T takes exact products.
template <typename T>
constexpr bool kExact = !std::is_same_v<T, __bf16>;

// One lane's 32 values of a fragment: as codes, or widened to fp16 (EXACT).
template <bool EXACT>
struct Fragment;

template <>
struct Fragment<false> {
  intx8 v;
  __device__ __forceinline__ Fragment(intx4 lo, intx4 hi)
      : v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]} {}
};

__device__ __forceinline__ halfx8 Widen(int lo, int hi) {
  const halfx2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const halfx2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const halfx2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const halfx2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return halfx8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <>
struct Fragment<true> {
  halfx8 v[4];
  __device__ __forceinline__ Fragment(intx4 lo, intx4 hi)
      : v{Widen(lo[0], lo[1]), Widen(lo[2], lo[3]), Widen(hi[0], hi[1]), Widen(hi[2], hi[3])} {}
};

__device__ __forceinline__ floatx4 Mfma(const Fragment<false> &w, const Fragment<false> &a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      w.v, a.v, floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ floatx4 Mfma(const Fragment<true> &w, const Fragment<true> &a) {
  floatx4 p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], p, 0, 0, 0);
  return p;
}

// Workgroup -> tile: an XCD (blockIdx % 8) takes a contiguous run of an order that
// walks groups of 4 row tiles column tile by column tile.
__device__ __forceinline__ void TileOf(int L, int tiles_m, int tiles_n, int &tm, int &tn) {
  const int tiles = tiles_m * tiles_n;
  if (tiles % 8 == 0) L = (L & 7) * (tiles / 8) + (L >> 3);
  constexpr int kGM = 4;
  const int group = L / (kGM * tiles_n);
  const int gm = min(kGM, tiles_m - group * kGM);
  const int rem = L - group * kGM * tiles_n;
  tm = group * kGM + rem % gm;
  tn = rem / gm;
}

// Rows of A in LDS: 128 bytes each, the eight 16-byte units of row r at places
// unit ^ ((r / 2) % 8). A copy takes eight whole rows (full cache lines: 55 bytes a
// clock and CU; the fragments' own order, 16 rows of 64 bytes, 16), and a
// fragment's read, 16 rows of one unit, meets every bank once.
__device__ __forceinline__ uint32_t CopyUnit(int lane, int row) {  // source byte of a copying lane
  return static_cast<uint32_t>(((lane & 7) ^ ((row >> 1) & 7)) * 16);
}
__device__ __forceinline__ uint32_t ReadUnit(int lane, int h) {  // a lane's half h of a fragment
  const int c = lane & 15, q = lane >> 4;
  return static_cast<uint32_t>(c * 128 + ((4 * h + q) ^ ((c >> 1) & 7)) * 16);
}

// n (up to C) consecutive values of a row of Y; whole: all C, at an address
// that 16 bytes (or the C values) divide.
template <typename T, int C>
__device__ __forceinline__ void StoreRow(T *p, const float *v, int64_t n, bool whole) {
  if (whole) {
    constexpr int kPer = C * sizeof(T) >= 16 ? 16 / sizeof(T) : C;
    typedef T Vec __attribute__((ext_vector_type(kPer)));
#pragma unroll
    for (int i = 0; i < C; i += kPer) {
      Vec q;
#pragma unroll
      for (int j = 0; j < kPer; ++j) q[j] = static_cast<T>(v[i + j]);
      *reinterpret_cast<Vec *>(p + i) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (i < n) p[i] = static_cast<T>(v[i]);
  }
}

// ---- few rows: the weights streamed once ------------------------------------
//
// Up to 16 rows: a workgroup takes 16 columns and all rows, one fragment each; its
// wavefronts take the blocks of K in turn, D of them in flight, and add up in LDS. One
// row of 4096 x 6144: 6.3 to 7.6 us, a launch and two round trips (3.3 TB/s); of 14336 x
// 4096 13 us (4.6 TB/s).
template <int WAVES, int D, bool EXACT, typename T>
__global__ __launch_bounds__(64 * WAVES) void Fp8StreamKernel(
    const uint8_t *__restrict__ W, const float *__restrict__ SW, const uint8_t *__restrict__ A,
    const float *__restrict__ SA, T *__restrict__ Y, int M, int64_t N, int64_t lda, int nb) {
  __shared__ floatx4 red[WAVES][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int c = lane & 15, qd = lane >> 4;
  const int64_t g = blockIdx.x >> 2;
  const int j = blockIdx.x & 3;
  const uint8_t *w = W + (g * nb * 8 + 2 * j) * kRec + lane * 16;
  const float *sw = SW + (g >> 1) * nb;
  const int64_t row = min(c, M - 1);
  const uint8_t *a = A + row * lda + 16 * qd;
  const float *sa = SA + row * nb;
  struct Block {
    intx4 w[2], a[2];
    float s;
  };
  auto load = [&](int b, Block &o) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      o.w[h] = *reinterpret_cast<const intx4 *>(w + (static_cast<int64_t>(b) * 8 + h) * kRec);
      o.a[h] = *reinterpret_cast<const intx4 *>(a + static_cast<int64_t>(b) * kBlock + 64 * h);
    }
    o.s = sa[b] * sw[b];
  };
  floatx4 acc{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Block &o) __attribute__((always_inline)) {
    const floatx4 p = Mfma(Fragment<EXACT>(o.w[0], o.w[1]), Fragment<EXACT>(o.a[0], o.a[1]));
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[v] = fmaf(p[v], o.s, acc[v]);
  };
  // This wavefront's blocks wave, wave + WAVES, ..: n of them, none loaded twice.
  Block x[D];
  const int n = (nb - wave + WAVES - 1) / WAVES;
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < n) load(wave + d * WAVES, x[d]);
  int i = 0;
  for (; i + 2 * D <= n; i += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      multiply(x[d]);
      load(wave + (i + d + D) * WAVES, x[d]);
    }
  }
#pragma unroll
  for (int d = 0; d < 2 * D - 1; ++d) {
    if (i + d < n) multiply(x[d % D]);
    if (d < D - 1 && i + d + D < n) load(wave + (i + d + D) * WAVES, x[d]);
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
  floatx4 sum = red[0][lane];
  for (int u = 1; u < WAVES; ++u) sum += red[u][lane];
  const int64_t col = 64 * g + 16 * qd + 4 * j;
  if (c < M && col < N) {
    const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    StoreRow<T, 4>(Y + c * N + col, v, N - col, N % 4 == 0);
  }
}

// 17 to 64 rows: the rows, and with them the weights and the row scales, pass
// through LDS, each wavefront's own blocks NS deep, so that the rows are copied by
// whole lines (gathered into registers they bound it: 32 us at 48 x 14336 x 4096 with the
// weights in the last cache, 16.6 so). Bound by those rows, which every 16 columns read
// again: 32 x 14336 x 4096 18 us, 3.3 TB/s of weights, 17 rows 14.5.
template <int MC, int WAVES, int NS, bool EXACT, typename T>
__global__ __launch_bounds__(64 * WAVES) void Fp8StreamLdsKernel(
    const uint8_t *__restrict__ W, const float *__restrict__ SW, const uint8_t *__restrict__ A,
    const float *__restrict__ SA, T *__restrict__ Y, int M, int64_t N, int64_t lda, int nb) {
  constexpr int kRows = 2 * kRec, kScales = kRows + 2 * MC * kRec;  // offsets in a stage
  constexpr int kStage = kScales + 256, kOps = 2 + 2 * MC + 1;
  static_assert(NS * kStage >= MC * 1024, "the sums reuse the stages");
  extern __shared__ uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int c = lane & 15, qd = lane >> 4;
  const int64_t g = blockIdx.x >> 2;
  const int j = blockIdx.x & 3;
  const uint8_t *w = W + (g * nb * 8 + 2 * j) * kRec;
  const float *sw = SW + (g >> 1) * nb;
  uint32_t a_off[2 * MC];
#pragma unroll
  for (int i = 0; i < 2 * MC; ++i) {
    const int row = 8 * i + (lane >> 3);
    a_off[i] = static_cast<uint32_t>(min(row, M - 1) * lda) + CopyUnit(lane, row);
  }
  const uint32_t s_off = static_cast<uint32_t>(min(lane, M - 1) * nb * 4), l16 = lane * 16;
  const uint8_t *mine = lds + wave * NS * kStage;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(mine));
  auto issue = [&](int b, int stage) __attribute__((always_inline)) {
    const uint32_t st = base + stage * kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      CopyToLds16S(w + (static_cast<int64_t>(b) * 8 + h) * kRec, l16, st + h * kRec);
#pragma unroll
    for (int i = 0; i < 2 * MC; ++i)
      CopyToLds16S(A + static_cast<int64_t>(b) * kBlock, a_off[i], st + kRows + i * kRec);
    CopyToLds4S(SA + b, s_off, st + kScales);
  };
  floatx4 acc[MC];
#pragma unroll
  for (int m = 0; m < MC; ++m) acc[m] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int b, int stage) __attribute__((always_inline)) {
    const uint8_t *st = mine + stage * kStage;
    const float scale = sw[b];
    const Fragment<EXACT> wf(*reinterpret_cast<const intx4 *>(st + l16),
                             *reinterpret_cast<const intx4 *>(st + kRec + l16));
#pragma unroll
    for (int m = 0; m < MC; ++m) {
      const uint8_t *at = st + kRows + 2 * m * kRec;
      const Fragment<EXACT> af(*reinterpret_cast<const intx4 *>(at + ReadUnit(lane, 0)),
                               *reinterpret_cast<const intx4 *>(at + ReadUnit(lane, 1)));
      const float f = *reinterpret_cast<const float *>(st + kScales + (16 * m + c) * 4) * scale;
      const floatx4 p = Mfma(wf, af);
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[m][v] = fmaf(p[v], f, acc[m][v]);
    }
  };
  // This wavefront's blocks wave, wave + WAVES, ..: n of them.
  const int n = (nb - wave + WAVES - 1) / WAVES;
#pragma unroll
  for (int p = 0; p < NS - 1; ++p)
    if (p < n) issue(wave + p * WAVES, p);
  int i = 0, stage = 0;
  for (; i + NS - 1 < n; ++i) {
    WaitCopies<kOps *(NS - 2)>();
    issue(wave + (i + NS - 1) * WAVES, stage == 0 ? NS - 1 : stage - 1);
    multiply(wave + i * WAVES, stage);
    stage = stage + 1 == NS ? 0 : stage + 1;
  }
  WaitCopies<0>();
  for (; i < n; ++i) {
    multiply(wave + i * WAVES, stage);
    stage = stage + 1 == NS ? 0 : stage + 1;
  }
  __syncthreads();
  floatx4 *red = reinterpret_cast<floatx4 *>(lds);  // [WAVES][MC][64]
#pragma unroll
  for (int m = 0; m < MC; ++m) red[(wave * MC + m) * 64 + lane] = acc[m];
  __syncthreads();
  for (int m = wave; m < MC; m += WAVES) {
    floatx4 sum = red[m * 64 + lane];
    for (int u = 1; u < WAVES; ++u) sum += red[(u * MC + m) * 64 + lane];
    const int row = 16 * m + c;
    const int64_t col = 64 * g + 16 * qd + 4 * j;
    if (row < M && col < N) {
      const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
      StoreRow<T, 4>(Y + row * N + col, v, N - col, N % 4 == 0);
    }
  }
}

// ---- more rows: tiles of 16 MI WM rows and 64 WN columns ------------------------
//
// WM by WN wavefronts of MI x 4 fragments, and NS blocks of K in LDS (W in the
// fragments' own order). A block is 4 MI slots, one fragment's product each;
// between them go the fold of two slots before and the LDS reads of the next
// group, in an order that sched_barrier keeps. The barrier that makes the next
// block visible stands before the last group, when this block's reads are done:
// its stage takes the copies of the block NS ahead, and the next block's weight
// fragments are read behind their last use (with the barrier between the blocks
// 47 us instead of 44 at 200 x 4096 x 28672). Four wavefronts, one per SIMD, and
// two workgroups a CU where LDS allows: one's waits are the other's work (300 x 4096
// x 4096, fp32 Y: 31 us with 128 x 128 tiles of eight wavefronts and K in two parts,
// 27 with 64 x 128 of four; 8192 x 4096 x 14336, 128 x 128: fp32 Y 903 us, fp16 Y 830,
// 1.16 PFLOP/s). What bounds it: the start and the end of a tile (10 us of
// the 20 at 333 x 2500 x 5001, fp32 Y, with one block of K), then copies, LDS reads
// and MFMAs about equally.
template <int MI, int WM, int WN, int NS, bool EXACT, typename T>
__global__ __launch_bounds__(64 * WM *WN) void Fp8TileKernel(
    const uint8_t *__restrict__ W, const float *__restrict__ SW, const uint8_t *__restrict__ A,
    const float *__restrict__ SA, T *__restrict__ Y, int64_t M, int64_t N, int64_t lda, int nb,
    int tiles_m, int tiles_n, int groups) {
  constexpr int NJ = 4, kWaves = WM * WN;
  constexpr int kARecs = 2 * MI * WM, kWRecs = 8 * WN;  // of 1 KiB
  constexpr int kAC = kARecs / kWaves, kWC = kWRecs / kWaves, kOps = kAC + kWC + 1;
  static_assert(kARecs % kWaves == 0 && kWRecs % kWaves == 0, "copies");
  static_assert(64 * kWaves >= 16 * MI * WM, "one row scale per thread");
  constexpr int kStage = (kARecs + kWRecs) * kRec + 256 * kWaves;  // bytes; row scales last
  extern __shared__ uint8_t lds[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int c = lane & 15, qd = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  int tm, tn;
  TileOf(static_cast<int>(blockIdx.x), tiles_m, tiles_n, tm, tn);
  const int splits = gridDim.y, split = blockIdx.y;
  const int b0 = static_cast<int>(static_cast<int64_t>(nb) * split / splits);
  const int last = static_cast<int>(static_cast<int64_t>(nb) * (split + 1) / splits) - 1;
  Y += static_cast<int64_t>(split) * M * N;
  const int64_t m0 = static_cast<int64_t>(tm) * 16 * MI * WM;
  const int64_t rows = min(M - m0, static_cast<int64_t>(16 * MI * WM));
  const int last_row = static_cast<int>(rows) - 1;

  uint32_t a_off[kAC];
  const uint8_t *w_src[kWC];
#pragma unroll
  for (int i = 0; i < kAC; ++i) {
    const int row = 8 * (i * kWaves + wave) + (lane >> 3);
    a_off[i] = static_cast<uint32_t>(min(row, last_row) * lda) + CopyUnit(lane, row);
  }
#pragma unroll
  for (int i = 0; i < kWC; ++i) {
    const int rec = i * kWaves + wave;  // group rec / 8 of the tile
    const int g = min(tn * WN + (rec >> 3), groups - 1);
    w_src[i] = W + (static_cast<int64_t>(g) * nb * 8 + (rec & 7)) * kRec;
  }
  const uint8_t *a_base = A + m0 * lda;
  const uint32_t s_off = static_cast<uint32_t>(min(static_cast<int>(threadIdx.x), last_row) * nb * 4);
  const float *sa_base = SA + m0 * nb;
  const uint32_t l16 = static_cast<uint32_t>(lane) * 16;
  auto issue = [&](int b, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t st = lds0 + stage;
#pragma unroll
    for (int i = 0; i < kAC; ++i)
      CopyToLds16S(a_base + static_cast<int64_t>(b) * kBlock, a_off[i],
                   st + (i * kWaves + wave) * kRec);
#pragma unroll
    for (int i = 0; i < kWC; ++i)
      CopyToLds16S(w_src[i] + static_cast<int64_t>(b) * 8 * kRec, l16,
                   st + (kARecs + i * kWaves + wave) * kRec);
    CopyToLds4S(sa_base + b, s_off, st + (kARecs + kWRecs) * kRec + wave * 256);
  };
  const uint8_t *a_at0 = lds + wm * MI * 2 * kRec + ReadUnit(lane, 0);
  const uint8_t *a_at1 = lds + wm * MI * 2 * kRec + ReadUnit(lane, 1);
  const uint8_t *w_at = lds + (kARecs + wn * 8) * kRec + lane * 16;
  const uint8_t *s_at = lds + (kARecs + kWRecs) * kRec + (wm * MI * 16 + c) * 4;
  struct Raw {
    intx4 lo, hi;
  };
  auto readA = [&](uint32_t st, int i) __attribute__((always_inline)) {
    return Raw{*reinterpret_cast<const intx4 *>(a_at0 + st + 2 * i * kRec),
               *reinterpret_cast<const intx4 *>(a_at1 + st + 2 * i * kRec)};
  };
  auto readW = [&](uint32_t st, int j) __attribute__((always_inline)) {
    const uint8_t *p = w_at + st + 2 * j * kRec;
    return Raw{*reinterpret_cast<const intx4 *>(p), *reinterpret_cast<const intx4 *>(p + kRec)};
  };
  auto readS = [&](uint32_t st, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const float *>(s_at + st + 64 * i);
  };
  using Frag = Fragment<EXACT>;

  floatx4 acc[MI][NJ], part[4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < 4; ++v) part[v] = floatx4{0.f, 0.f, 0.f, 0.f};
  const float *sw = SW + static_cast<int64_t>(min(tn * WN + wn, groups - 1) >> 1) * nb;
#pragma unroll
  for (int p = 0; p < NS; ++p) issue(min(b0 + p, last), p * kStage);
  WaitBarrier<kOps *(NS - 1)>();
  float f[2], scale = sw[b0];
  Raw raw_w[NJ], raw_a = readA(0, 0);
#pragma unroll
  for (int j = 0; j < NJ; ++j) raw_w[j] = readW(0, j);
  f[0] = readS(0, 0) * scale;
  f[1] = 0.0f;
  Frag af[2] = {Frag(raw_a.lo, raw_a.hi), Frag(raw_a.lo, raw_a.hi)};
  Frag wf[NJ] = {Frag(raw_w[0].lo, raw_w[0].hi), Frag(raw_w[1].lo, raw_w[1].hi),
                 Frag(raw_w[2].lo, raw_w[2].hi), Frag(raw_w[3].lo, raw_w[3].hi)};

  auto fold = [&](auto kc) __attribute__((always_inline)) {  // slot k of a block
    constexpr int k = decltype(kc)::value, i = k / NJ, j = k % NJ;
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(part[k % 4][v], f[i % 2], acc[i][j][v]);
  };
  constexpr int kSlots = MI * NJ, kLast = kSlots - NJ;
  static_assert(MI % 2 == 0, "the row fragments' parity");
  uint32_t st = 0;
  for (int b = b0; b <= last; ++b) {
    const uint32_t next = st + kStage == NS * kStage ? 0 : st + kStage;
    const float next_scale = sw[min(b + 1, last)];
    float s_next = 0.0f;
    auto slot = [&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value, i = k / NJ, j = k % NJ;
      // The next block is in LDS, this block's reads are done.
      if constexpr (k == kLast) WaitBarrier<kOps *(NS - 2)>();
      part[k % 4] = Mfma(wf[j], af[i % 2]);
      if constexpr (j == 0) raw_a = i + 1 < MI ? readA(st, i + 1) : readA(next, 0);
      if constexpr (j == 1) s_next = i + 1 < MI ? readS(st, i + 1) : readS(next, 0);
      if constexpr (i + 1 == MI) {
        raw_w[j] = readW(next, j);
        if constexpr (!EXACT) wf[j] = Frag(raw_w[j].lo, raw_w[j].hi);
      }
      // Two slots back; the first two of a block are the last ones of the block
      // before (of its products with f[1], still there).
      if constexpr (k >= 2) fold(std::integral_constant<int, k - 2>{});
      else fold(std::integral_constant<int, kSlots - 2 + k>{});
      if constexpr (j == 3) {
        // The factor of group i + 1 takes the place of group i - 1's after its last fold.
        f[(i + 1) % 2] = s_next * (i + 1 < MI ? scale : next_scale);
        af[(i + 1) % 2] = Frag(raw_a.lo, raw_a.hi);
      }
      if constexpr (k == kLast) issue(min(b + NS, last), st);
      __builtin_amdgcn_sched_barrier(0);
    };
    [&]<int... k>(std::integer_sequence<int, k...>) __attribute__((always_inline)) {
      (slot(std::integral_constant<int, k>{}), ...);
    }(std::make_integer_sequence<int, kSlots>{});
    if constexpr (EXACT) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) wf[j] = Frag(raw_w[j].lo, raw_w[j].hi);
    }
    scale = next_scale;
    st = next;
  }
  fold(std::integral_constant<int, kSlots - 2>{});
  fold(std::integral_constant<int, kSlots - 1>{});
  WaitBarrier<0>();  // no copy may land after this workgroup

  const int64_t n0 = static_cast<int64_t>(tn) * WN * 64, n = n0 + wn * 64 + 16 * qd;
  if ((N * static_cast<int64_t>(sizeof(T))) % 16 == 0) {
    if (n >= N) return;
    const bool whole = n + 16 <= N;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int64_t row = 16 * (wm * MI + i) + c;
      float v[16];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) v[4 * j + u] = acc[i][j][u];
      if (row < rows) StoreRow<T, 16>(Y + (m0 + row) * N + n, v, N - n, whole);
    }
    return;
  }
  // Rows that no vector store fits pass through LDS and leave by consecutive values
  // (333 x 2500 x 5001: 21 us; 35 where each lane stored its 16 one by one).
  constexpr int kPitch = 64 * WN + 4;
  static_assert(16 * MI * WM * kPitch * 4 <= NS * kStage, "the tile reuses the stages");
  float *tile = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      *reinterpret_cast<floatx4 *>(tile + (16 * (wm * MI + i) + c) * kPitch + wn * 64 + 16 * qd +
                                   4 * j) = acc[i][j];
  __syncthreads();
  for (int row = wave; row < rows; row += kWaves) {
#pragma unroll
    for (int u = 0; u < WN; ++u)
      if (n0 + 64 * u + lane < N)
        Y[(m0 + row) * N + n0 + 64 * u + lane] = static_cast<T>(tile[row * kPitch + 64 * u + lane]);
  }
}

// ---- many rows, bf16 Y: 256 x 256 tiles ---------------------------------------
//
// Eight wavefronts, two per SIMD, of 8 x 4 fragments. A block of K is 32 slots,
// one MFMA each; between them go the fold of two slots before (its products have
// left the matrix unit by then), the LDS reads of the next group and the copies
// of the block after next, in an order that sched_barrier keeps.
//  - The barrier that makes the next block visible stands before the last group,
//    when this block's reads are done: the next block's weight fragments are
//    read in place, each behind its last MFMA, so that the matrix unit does not
//    wait at the block's end.
//  - LDS holds two blocks, and the copies of one take about as long as a block's
//    MFMAs (1.8 us), so most start half a block earlier: a barrier in the
//    middle says that the weights and half of the rows have been read.
//  - A workgroup goes through its tiles without a pause: the last blocks of one
//    copy the first blocks of the next, and its stores run beside those.
// Left is the power limit: with these operands moving, the clock falls to 1.6-1.7
// GHz (1.55 with the copies switched off, 2.1 on constant operands).
// 8192 x 4096 x 14336: 604 us with barriers between the blocks, 510 with them
// inside, 460 with copies half a block earlier, 437 with rows copied by whole lines,
// 418 so (2.30 PFLOP/s).
constexpr int kWideTile = 256;

__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void Fp8WideKernel(
    const uint8_t *__restrict__ W, const float *__restrict__ SW, const uint8_t *__restrict__ A,
    const float *__restrict__ SA, __bf16 *__restrict__ Y, int64_t M, int64_t N, int64_t lda, int nb,
    int tiles_m, int tiles_n, int groups) {
  constexpr int MI = 8, NJ = 4, WM = 2, WN = 4;
  constexpr int kARecs = 32, kWRecs = 32;
  constexpr int kStage = (kARecs + kWRecs) * kRec + 2048;  // bytes; row scales last
  extern __shared__ uint8_t lds[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int c = lane & 15, qd = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  const int tiles = tiles_m * tiles_n, last = nb - 1;

  // A tile's copy sources. Copy n < 4 takes eight of rows 32 n .. 32 n + 31 and
  // 128 + 32 n .. (groups 2 n and 2 n + 1 of both halves of the tile), copies 4 .. 7
  // the weights', copy 8 the row scales.
  struct Source {
    uint32_t a_off[4], s_off;
    const uint8_t *a, *w[4];
    const float *sa;
  };
  const uint32_t l16 = static_cast<uint32_t>(lane) * 16;
  const int row0 = (wave >> 2) * 128 + (wave & 3) * 8;  // of copy 0
  auto source = [&](int tile, Source &o) __attribute__((always_inline)) {
    int tm, tn;
    TileOf(tile, tiles_m, tiles_n, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * kWideTile;
    const int last_row = static_cast<int>(min(M - m0, static_cast<int64_t>(kWideTile))) - 1;
    o.a = A + m0 * lda;
    o.sa = SA + m0 * nb;
    o.s_off = static_cast<uint32_t>(min(static_cast<int>(threadIdx.x), last_row) * nb * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 32 * i + (lane >> 3);
      o.a_off[i] = static_cast<uint32_t>(min(row, last_row) * lda) + CopyUnit(lane, row);
      const int g = min(tn * WN + i, groups - 1);
      o.w[i] = W + (static_cast<int64_t>(g) * nb * 8 + wave) * kRec;
    }
  };
  auto copy = [&](auto nc, const Source &o, int b, uint32_t st) __attribute__((always_inline)) {
    constexpr int n = decltype(nc)::value;
    if constexpr (n < 4)
      CopyToLds16S(o.a + static_cast<int64_t>(b) * kBlock, o.a_off[n],
                   lds0 + st + (row0 + 32 * n) * 128);
    else if constexpr (n < 8)
      CopyToLds16S(o.w[n - 4] + static_cast<int64_t>(b) * 8 * kRec, l16,
                   lds0 + st + (kARecs + (n - 4) * 8 + wave) * kRec);
    else
      CopyToLds4S(o.sa + b, o.s_off, lds0 + st + (kARecs + kWRecs) * kRec + wave * 256);
  };
  auto issue = [&](const Source &o, int b, uint32_t st) __attribute__((always_inline)) {
    [&]<int... n>(std::integer_sequence<int, n...>) __attribute__((always_inline)) {
      (copy(std::integral_constant<int, n>{}, o, b, st), ...);
    }(std::make_integer_sequence<int, 9>{});
  };
  const uint8_t *a_at0 = lds + wm * MI * 2 * kRec + ReadUnit(lane, 0);
  const uint8_t *a_at1 = lds + wm * MI * 2 * kRec + ReadUnit(lane, 1);
  const uint8_t *w_at = lds + (kARecs + wn * 8) * kRec + lane * 16;
  const uint8_t *s_at = lds + (kARecs + kWRecs) * kRec + (wm * MI * 16 + c) * 4;
  auto readA = [&](uint32_t st, int i) __attribute__((always_inline)) {
    return Fragment<false>(*reinterpret_cast<const intx4 *>(a_at0 + st + 2 * i * kRec),
                           *reinterpret_cast<const intx4 *>(a_at1 + st + 2 * i * kRec)).v;
  };
  auto readW = [&](uint32_t st, int j) __attribute__((always_inline)) {
    const uint8_t *p = w_at + st + 2 * j * kRec;
    return Fragment<false>(*reinterpret_cast<const intx4 *>(p),
                           *reinterpret_cast<const intx4 *>(p + kRec)).v;
  };
  auto readS = [&](uint32_t st, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const float *>(s_at + st + 64 * i);
  };
  // The weight scales of this wavefront's columns of a tile.
  auto scales_of = [&](int tile) __attribute__((always_inline)) {
    int tm, tn;
    TileOf(tile, tiles_m, tiles_n, tm, tn);
    return SW + static_cast<int64_t>(min(tn * WN + wn, groups - 1) >> 1) * nb;
  };

  floatx4 acc[MI][NJ], part[4];
  const floatx4 zero{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < 4; ++v) part[v] = zero;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = zero;
  Source now, next;
  source(static_cast<int>(blockIdx.x), now);
  issue(now, 0, 0);
  issue(now, 1, kStage);
  const float *sw = scales_of(static_cast<int>(blockIdx.x));
  WaitBarrier<9>();
  intx8 wf[NJ], af[2];
  float f[2], scale = sw[0];
#pragma unroll
  for (int j = 0; j < NJ; ++j) wf[j] = readW(0, j);
  af[0] = readA(0, 0);
  f[0] = readS(0, 0) * scale;
  f[1] = 0.0f;

  auto fold = [&](auto kc) __attribute__((always_inline)) {  // slot k of a block
    constexpr int k = decltype(kc)::value, i = k / NJ, j = k % NJ;
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(part[k % 4][v], f[i % 2], acc[i][j][v]);
  };
  constexpr int kSlots = MI * NJ, kMid = 16, kLast = kSlots - NJ;
  uint32_t st = 0;
  for (int tile = static_cast<int>(blockIdx.x); tile < tiles; tile += gridDim.x) {
    // Behind the last tile its last block is copied again.
    const bool more = tile + static_cast<int>(gridDim.x) < tiles;
    const int next_tile = more ? tile + static_cast<int>(gridDim.x) : tile;
    const float *sw_next = scales_of(next_tile);
    source(next_tile, next);
    for (int b = 0; b < nb; ++b) {
      const uint32_t other = kStage - st;
      // The block after next: of this tile or of the next one. No branch here: it
      // would cost the registers of the slots' pinned order.
      const bool ahead = b + 2 > last;
      const int cb = ahead ? (more ? b + 2 - nb : last) : b + 2;
      Source from;
      from.a = ahead ? next.a : now.a;
      from.sa = ahead ? next.sa : now.sa;
      from.s_off = ahead ? next.s_off : now.s_off;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        from.a_off[i] = ahead ? next.a_off[i] : now.a_off[i];
        from.w[i] = ahead ? next.w[i] : now.w[i];
      }
      const float next_scale = *(b < last ? sw + b + 1 : sw_next);
      float s_next = 0.0f;
      auto slot = [&](auto kc) __attribute__((always_inline)) {
        constexpr int k = decltype(kc)::value, i = k / NJ, j = k % NJ;
        if constexpr (k == kMid) WaitBarrier<63>();  // LDS reads up to group 4 are done
        // The next block is in LDS (six newer copies are on their way), this block's
        // reads are done.
        if constexpr (k == kLast) WaitBarrier<6>();
        part[k % 4] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], af[i % 2], zero, 0, 0,
                                                                      0, 0, 0, 0);
        if constexpr (i + 1 < MI) {
          if constexpr (j == 0) af[(i + 1) % 2] = readA(st, i + 1);
          if constexpr (j == 1) s_next = readS(st, i + 1);
        } else {
          if constexpr (j == 0) af[(i + 1) % 2] = readA(other, 0);
          if constexpr (j == 1) s_next = readS(other, 0);
          wf[j] = readW(other, j);
        }
        // Two slots back; the first two of a block are the last ones of the block
        // before (of its products with f[1], still there).
        if constexpr (k >= 2) fold(std::integral_constant<int, k - 2>{});
        else fold(std::integral_constant<int, kSlots - 2 + k>{});
        // The factor of group i + 1 takes the place of group i - 1's after its last fold.
        if constexpr (j == 3) f[(i + 1) % 2] = s_next * (i + 1 < MI ? scale : next_scale);
        // The block after next into this block's stage: the weights and the first four
        // groups of rows, then the others and the row scales.
        if constexpr (k >= kMid && k < kMid + 4)
          copy(std::integral_constant<int, 4 + k - kMid>{}, from, cb, st);
        if constexpr (k >= kMid + 4 && k < kMid + 6)
          copy(std::integral_constant<int, k - kMid - 4>{}, from, cb, st);
        if constexpr (k >= kLast && k < kLast + 2)
          copy(std::integral_constant<int, 2 + k - kLast>{}, from, cb, st);
        if constexpr (k == kLast + 2) copy(std::integral_constant<int, 8>{}, from, cb, st);
        __builtin_amdgcn_sched_barrier(0);
      };
      [&]<int... k>(std::integer_sequence<int, k...>) __attribute__((always_inline)) {
        (slot(std::integral_constant<int, k>{}), ...);
      }(std::make_integer_sequence<int, kSlots>{});
      scale = next_scale;
      st = other;
    }
    sw = sw_next;
    now = next;
    fold(std::integral_constant<int, kSlots - 2>{});
    fold(std::integral_constant<int, kSlots - 1>{});
    // The next tile's first block folds them again, by a factor of its own: this tile's
    // last one may be infinite or NaN, and 0 times that would stay in the next tile's sums.
    part[(kSlots - 2) % 4] = part[(kSlots - 1) % 4] = zero;
    f[1] = 0.0f;
    int tm, tn;
    TileOf(tile, tiles_m, tiles_n, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * kWideTile;
    const int64_t rows = min(M - m0, static_cast<int64_t>(kWideTile));
    const int64_t n = (static_cast<int64_t>(tn) * WN + wn) * 64 + 16 * qd;
    const bool whole = n + 16 <= N && (N * 2) % 16 == 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int64_t row = 16 * (wm * MI + i) + c;
      float v[16];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[4 * j + u] = acc[i][j][u];
        acc[i][j] = zero;
      }
      if (row < rows && n < N) StoreRow<__bf16, 16>(Y + (m0 + row) * N + n, v, N - n, whole);
    }
  }
  WaitBarrier<0>();  // no copy may land after this workgroup
}

// Y = the sum of S partial products, in order.
template <typename T>
__global__ __launch_bounds__(256) void Fp8SumKernel(const float *__restrict__ P, T *__restrict__ Y,
                                                    int64_t mn, int S) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < mn; i += step) {
    float v = P[i];
    for (int s = 1; s < S; ++s) v += P[s * mn + i];
    Y[i] = static_cast<T>(v);
  }
}

// Whether M rows take the kernels that stream the weights. Their workgroups of 16
// columns each read all rows, M K bytes, and the more of them a CU has (r, rounded up)
// the earlier the tiles' longer start is paid for: r r M K decides, up to 256 KiB of it
// where up to 16 rows are gathered into registers, up to 448 KiB where they pass through
// LDS. From r = 6, or 3, on the tiles lose 1 us at the few K and M where they lose at
// all, and gain more elsewhere.
// us, stream and tile, bf16 Y, weights not in a cache:
//   N = 4096 (r = 1): K = 14336 16 rows 16 and 17, 32 rows 18 and 18, 33 rows 19 and 19,
//     48 rows 23 and 20, 64 rows 26 and 22; K = 20480 17 rows 20 and 21, 32 rows 24 and
//     22; K = 28672 9 rows 26 and 27, 16 rows 32 and 27; K = 8192 64 rows 16 and 16
//   N = 1024: K = 16384 9 rows 11 and 13, 16 rows 15 and 14, 33 rows 15 and 14
//   r = 2: 4096 x 8192 (K x N) 32 rows 13 and 13, 64 rows 17 and 16; 8192 x 5120 8 rows 13
//     and 13, 16 rows 17 and 14
//   r = 3: 2048 x 12288 16 rows 9 and 10, 32 rows 11 and 11; 1024 x 12288 48 rows 8 and 7
//   r = 4: 4096 x 14336 1 row 15 and 16, 8 rows 16 and 15; 1024 x 14336 64 rows 13 and 7
//   r = 5: 2048 x 20480 1 row 10 and 13, 16 rows 12 and 12
//   r = 6: 4096 x 24576 1 row 23 and 22; 2048 x 24576 1 row 12 and 13, 4 rows 13 and 12
bool Streams(const Weight &w, int64_t M) {
  if (M > 64) return false;
  const int64_t r = CeilDiv(w.groups * 4, w.num_cus), bytes = r * r * M * w.nb * kBlock;
  return M <= 16 ? r <= 5 && bytes <= 256 << 10 : r <= 2 && bytes <= 448 << 10;
}

struct TileShape {
  int rows, cols, splits;
};

// exact: an fp32 or fp16 Y.
TileShape PickTile(const Weight &w, int64_t M, bool exact) {
  // bf16 results: large tiles where they fill the chip (rows of whole vectors), of
  // rows that fill half a tile at least (K = 4096, N = 65536, us, in these tiles and in
  // those below: 1 row 62 and 52, 40 rows 65 and 60, 128 rows 67 and 63, 129 rows 67 and
  // 87; N = 128256: 1 row 123 and 93, 128 rows 136 and 124, 129 rows 133 and 167).
  if (!exact && M > 128 && w.nb >= 2 && w.N % 8 == 0 &&
      CeilDiv(M, 256) * CeilDiv(w.N, 256) >= w.num_cus)
    return TileShape{256, 256, 1};
  // 64 x 128, two workgroups a CU. Larger ones take fewer reads of LDS and the
  // caches: 128 rows where they still fill the chip (512 x 4096 x 14336, bf16: 48 us
  // instead of 58), and all of 129 to 256 rows for bf16 results where half the chip
  // has one (250 x 4096 x 20480: 40 us instead of 49; with fewer the other half
  // counts: 200 x 4096 x 14336: 39 instead of 30).
  TileShape t{64, 128, 1};
  if (!exact && M > 128 && M <= 256 && 2 * CeilDiv(w.N, 128) > w.num_cus) t.rows = 256;
  else if (M > 64 && CeilDiv(M, 128) * CeilDiv(w.N, 128) >= w.num_cus) t.rows = 128;
  // K is split so that every CU has work, of at least eight blocks each, ten for bf16
  // results: the second launch takes as long (333 x 2048 x 2560, bf16: 13 us in two
  // parts of eight, 10 whole; 65 x 2048 x 1024, fp32: 12 and 15).
  const int64_t tiles = CeilDiv(M, t.rows) * CeilDiv(w.N, t.cols);
  const int64_t s = std::min<int64_t>({w.num_cus / tiles, w.nb / (exact ? 8 : 10), 8});
  t.splits = static_cast<int>(std::max<int64_t>(1, s));
  return t;
}

template <typename T>
hipError_t StreamT(const Weight &w, int M, const uint8_t *A, int64_t lda, const float *sa, void *Y,
                   hipStream_t s) {
  constexpr int kWaves = 8, kDepth = 4;
  hipLaunchKernelGGL((Fp8StreamKernel<kWaves, kDepth, kExact<T>, T>),
                     dim3(static_cast<unsigned>(w.groups * 4)), dim3(64 * kWaves), 0, s, w.W,
                     w.scales, A, sa, static_cast<T *>(Y), M, w.N, lda, static_cast<int>(w.nb));
  return hipGetLastError();
}

template <int MC, typename T>
hipError_t StreamLdsT(const Weight &w, int M, const uint8_t *A, int64_t lda, const float *sa,
                      void *Y, hipStream_t s) {
  constexpr int kWaves = MC == 2 ? 8 : MC == 3 ? 6 : 4, NS = 3;
  const size_t lds = static_cast<size_t>(kWaves) * NS * ((2 + 2 * MC) * kRec + 256);
  hipLaunchKernelGGL((Fp8StreamLdsKernel<MC, kWaves, NS, kExact<T>, T>),
                     dim3(static_cast<unsigned>(w.groups * 4)), dim3(64 * kWaves), lds, s, w.W,
                     w.scales, A, sa, static_cast<T *>(Y), M, w.N, lda, static_cast<int>(w.nb));
  return hipGetLastError();
}

template <int MI, int WM, int WN, int NS, bool EXACT, typename T>
hipError_t TileLaunch(const Weight &w, const TileShape &t, int64_t M, const uint8_t *A, int64_t lda,
                      const float *sa, T *Y, hipStream_t s) {
  const int64_t tiles_m = CeilDiv(M, 16 * MI * WM), tiles_n = CeilDiv(w.N, 64 * WN);
  const size_t lds = static_cast<size_t>(NS) * ((2 * MI * WM + 8 * WN) * kRec + 256 * WM * WN);
  hipLaunchKernelGGL((Fp8TileKernel<MI, WM, WN, NS, EXACT, T>),
                     dim3(static_cast<unsigned>(tiles_m * tiles_n), t.splits), dim3(64 * WM * WN),
                     lds, s, w.W, w.scales, A, sa, Y, M, w.N, lda, static_cast<int>(w.nb),
                     static_cast<int>(tiles_m), static_cast<int>(tiles_n),
                     static_cast<int>(w.groups));
  return hipGetLastError();
}

template <typename T>
hipError_t TileT(const Weight &w, const TileShape &t, int64_t M, const uint8_t *A, int64_t lda,
                 const float *sa, T *Y, hipStream_t s) {
  if constexpr (!kExact<T>) {
    if (t.cols == 256) {
      const int64_t tiles_m = CeilDiv(M, 256), tiles_n = CeilDiv(w.N, 256);
      const int64_t wgs = std::min<int64_t>(tiles_m * tiles_n, w.num_cus);
      hipLaunchKernelGGL(Fp8WideKernel, dim3(static_cast<unsigned>(wgs)), dim3(512),
                         2 * (64 * kRec + 2048), s, w.W, w.scales, A, sa, Y, M, w.N, lda,
                         static_cast<int>(w.nb), static_cast<int>(tiles_m),
                         static_cast<int>(tiles_n), static_cast<int>(w.groups));
      return hipGetLastError();
    }
    if (t.rows == 256) return TileLaunch<8, 2, 2, 3, kExact<T>, T>(w, t, M, A, lda, sa, Y, s);
  }
  if (t.rows == 128) return TileLaunch<4, 2, 2, 2, kExact<T>, T>(w, t, M, A, lda, sa, Y, s);
  return TileLaunch<2, 2, 2, 3, kExact<T>, T>(w, t, M, A, lda, sa, Y, s);
}

template <typename T>
hipError_t ProductT(const Weight &w, int64_t M, const uint8_t *A, int64_t lda, const float *sa,
                    void *Y, void *work, hipStream_t s) {
  if (Streams(w, M)) {
    const int m = static_cast<int>(M);
    switch ((M + 15) / 16) {
    case 1: return StreamT<T>(w, m, A, lda, sa, Y, s);
    case 2: return StreamLdsT<2, T>(w, m, A, lda, sa, Y, s);
    case 3: return StreamLdsT<3, T>(w, m, A, lda, sa, Y, s);
    default: return StreamLdsT<4, T>(w, m, A, lda, sa, Y, s);
    }
  }
  const TileShape t = PickTile(w, M, kExact<T>);
  if (t.splits == 1) return TileT<T>(w, t, M, A, lda, sa, static_cast<T *>(Y), s);
  float *parts = static_cast<float *>(work);
  // Larger tiles are never split: they fill half the chip.
  hipError_t e = TileLaunch<2, 2, 2, 3, kExact<T>, float>(w, t, M, A, lda, sa, parts, s);
  if (e != hipSuccess) return e;
  const int64_t mn = M * w.N;
  hipLaunchKernelGGL((Fp8SumKernel<T>),
                     dim3(static_cast<unsigned>(std::min<int64_t>(CeilDiv(mn, 256), 1 << 16))),
                     dim3(256), 0, s, parts, static_cast<T *>(Y), mn, t.splits);
  return hipGetLastError();
}

} // namespace

size_t WorkBytes(const Weight &w, int64_t M) {
  if (Streams(w, M)) return 0;
  const int splits = std::max(PickTile(w, M, false).splits, PickTile(w, M, true).splits);
  return splits == 1 ? 0 : static_cast<size_t>(splits) * M * w.N * sizeof(float);
}

const char *ProductKernelName(const Weight &w, int64_t M) {
  if (Streams(w, M)) return M <= 16 ? "Fp8StreamKernel" : "Fp8StreamLdsKernel";
  return PickTile(w, M, false).cols == 256 ? "Fp8WideKernel" : "Fp8TileKernel";
}

hipError_t LaunchProduct(const Weight &w, int64_t M, const uint8_t *A, int64_t lda,
                         const float *sa, int32_t y_type, void *Y, void *work, hipStream_t s) {
  switch (y_type) {
  case MNB_TYPE_FLOAT16: return ProductT<_Float16>(w, M, A, lda, sa, Y, work, s);
  case MNB_TYPE_BFLOAT16: return ProductT<__bf16>(w, M, A, lda, sa, Y, work, s);
  default: return ProductT<float>(w, M, A, lda, sa, Y, work, s);
  }
}

} // namespace fp8
} // namespace mnb

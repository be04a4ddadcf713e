// Rows to e4m3 with a scale for each block of 128, the weight layout of the
// 8-bit product, and the padding of ragged code rows.
#include "mnb_fp8.h"

namespace mnb {
namespace fp8 {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float ToFloat(T v) {
  return static_cast<float>(v);
}

// Eight values at p (n of them exist), zeros behind them.
template <typename T, bool VEC>
__device__ __forceinline__ void Load8(const T *p, int n, float (&x)[8]) {
  if constexpr (VEC) {
    if (n <= 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.0f;
      return;
    }
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int v = 0; v < static_cast<int>(sizeof(T)) / 2; ++v) {
      const Vec q = reinterpret_cast<const Vec *>(p)[v];
#pragma unroll
      for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i)
        x[v * static_cast<int>(16 / sizeof(T)) + i] = ToFloat(q[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? ToFloat(p[i]) : 0.0f;
  }
}

// One (row, block) item per 16 lanes, eight values a lane. The quotient
// 448 x / amax is correctly rounded to fp32 (for fp32 x up to rare double
// roundings of a 2^-47 residue), since half-way codes are common among 16-bit rows
// and a reciprocal's rounding would push them to either side: with
// a = amax 2^-e in [1, 2) and r the rounded 1 / a, q0 = t r is off by at most
// two units, its remainder t - q0 a is exact in one fma, and q0 + remainder r
// rounds to the nearest (Markstein). t = 448 x 2^-e carries its own rounding
// error along for fp32 rows. Four to six operations a value instead of a
// division's eleven; bound by memory.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void QuantizeKernel(const T *__restrict__ X,
                                                           uint8_t *__restrict__ Q,
                                                           float *__restrict__ S, int64_t M,
                                                           int64_t K, int64_t ldx, int64_t ldq,
                                                           int64_t nb) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 16) + threadIdx.x / 16;
  if (item >= M * nb) return;
  const int64_t row = item / nb, b = item - row * nb;
  const int64_t k0 = b * kBlock + 8 * (threadIdx.x & 15);
  const int n = static_cast<int>(min(int64_t{8}, K - k0));  // <= 0 past the row
  float x[8];
  Load8<T, VEC>(X + row * ldx + k0, n, x);
  // As integers, magnitudes order like their values, infinity above them and NaN on top.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1)
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 16)));
  const uint32_t least = static_cast<uint32_t>(127 - 100) << 23;  // 2^-100
  const float amax = __uint_as_float(max(top, least));
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
  float q[8];
  if (top < 0x7F800000u) {
    const float a = ldexpf(amax, -e);
    const float r = 1.0f / a;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float xs = ldexpf(x[i], -e);
      const float t = xs * 448.0f;
      const float q0 = t * r;
      float rem = fmaf(-q0, a, t);
      if constexpr (sizeof(T) == 4) rem += fmaf(xs, 448.0f, -t);
      q[i] = fmaf(rem, r, q0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = x[i] / amax;  // 0 where x is finite (448 x may not be)
  }
  if ((threadIdx.x & 15) == 0) S[item] = amax / 448.0f;
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
  uint8_t *out = Q + row * ldq + k0;
  if constexpr (VEC) {
    if (k0 < ldq) *reinterpret_cast<int2 *>(out) = make_int2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < ldq) out[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

__global__ __launch_bounds__(kThreads) void PadKernel(const uint8_t *__restrict__ A,
                                                      uint8_t *__restrict__ P, int64_t M,
                                                      int64_t K, int64_t ldp) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 4;
  if (i >= M * ldp) return;
  const int64_t row = i / ldp, k = i - row * ldp;
  const uint8_t *a = A + row * K + k;
  uint32_t v = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (k + j < K) v |= static_cast<uint32_t>(a[j]) << (8 * j);
  *reinterpret_cast<uint32_t *>(P + i) = v;
}

// One thread per 16 bytes of the records.
__global__ __launch_bounds__(kThreads) void RelayoutKernel(const uint8_t *__restrict__ W,
                                                           uint8_t *__restrict__ R, int64_t K,
                                                           int64_t N, int64_t nb, int64_t units) {
  const int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (u >= units) return;
  const int lane = static_cast<int>(u & 63), h = static_cast<int>(u >> 6) & 1,
            j = static_cast<int>(u >> 7) & 3;
  const int64_t gb = u >> 9, g = gb / nb, b = gb - g * nb;
  const int r = lane & 15;
  const int64_t n = 64 * g + 16 * (r >> 2) + 4 * j + (r & 3);
  const int64_t k = b * kBlock + 64 * h + 16 * (lane >> 4);
  uint32_t v[4] = {0, 0, 0, 0};
  if (n < N) {
    const uint8_t *src = W + n * K + k;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) v[i / 4] |= static_cast<uint32_t>(src[i]) << (8 * (i % 4));
  }
  reinterpret_cast<uint4 *>(R)[u] = make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T>
hipError_t QuantizeT(int64_t M, int64_t K, const void *X, int64_t ldx, uint8_t *Q, int64_t ldq,
                     float *scales, hipStream_t s) {
  const int64_t nb = CeilDiv(K, kBlock);
  const T *x = static_cast<const T *>(X);
  const bool vec = K % 8 == 0 && (ldx * sizeof(T)) % 16 == 0 && ldq % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(X) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(Q) % 8 == 0;
  // Launches of at most 2^27 items, 16 lanes each: a grid's threads stay below 2^32.
  const int64_t rows = std::max<int64_t>(1, (int64_t{1} << 27) / nb);
  for (int64_t m = 0; m < M; m += rows) {
    const int64_t n = std::min(rows, M - m);
    const dim3 grid(static_cast<unsigned>(CeilDiv(n * nb, kThreads / 16)));
    if (vec)
      hipLaunchKernelGGL((QuantizeKernel<T, true>), grid, dim3(kThreads), 0, s, x + m * ldx,
                         Q + m * ldq, scales + m * nb, n, K, ldx, ldq, nb);
    else
      hipLaunchKernelGGL((QuantizeKernel<T, false>), grid, dim3(kThreads), 0, s, x + m * ldx,
                         Q + m * ldq, scales + m * nb, n, K, ldx, ldq, nb);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

} // namespace

hipError_t LaunchQuantize(int64_t M, int64_t K, int32_t x_type, const void *X, int64_t ldx,
                          uint8_t *Q, int64_t ldq, float *scales, hipStream_t s) {
  switch (x_type) {
  case MNB_TYPE_FLOAT16: return QuantizeT<_Float16>(M, K, X, ldx, Q, ldq, scales, s);
  case MNB_TYPE_BFLOAT16: return QuantizeT<__bf16>(M, K, X, ldx, Q, ldq, scales, s);
  default: return QuantizeT<float>(M, K, X, ldx, Q, ldq, scales, s);
  }
}

hipError_t LaunchPad(int64_t M, int64_t K, const uint8_t *A, uint8_t *P, hipStream_t s) {
  const int64_t ldp = CeilDiv(K, kBlock) * kBlock;
  const int64_t rows = std::max<int64_t>(1, (int64_t{1} << 32) / ldp);
  for (int64_t m = 0; m < M; m += rows) {
    const int64_t n = std::min(rows, M - m);
    hipLaunchKernelGGL(PadKernel, dim3(static_cast<unsigned>(CeilDiv(n * ldp / 4, kThreads))),
                       dim3(kThreads), 0, s, A + m * K, P + m * ldp, n, K, ldp);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t LaunchRelayout(const uint8_t *dW, const Weight &w, uint8_t *records, hipStream_t s) {
  // Groups at a time, so that a grid's threads stay below 2^32.
  const int64_t per = std::max<int64_t>(1, (int64_t{1} << 30) / (w.nb * 512));
  for (int64_t g = 0; g < w.groups; g += per) {
    const int64_t n = std::min(per, w.groups - g), units = n * w.nb * 512;
    hipLaunchKernelGGL(RelayoutKernel, dim3(static_cast<unsigned>(CeilDiv(units, kThreads))),
                       dim3(kThreads), 0, s, dW + 64 * g * w.K, records + g * w.nb * 8 * kRec, w.K,
                       w.N - 64 * g, w.nb, units);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

} // namespace fp8
} // namespace mnb

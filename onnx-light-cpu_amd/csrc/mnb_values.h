// Loads, stores and 8-bit codes of rows in fp32, fp16 or bf16, shared by the
// kernels that take them.
#pragma once

#include "mnb_kernels.h"

#include <type_traits>

namespace mnb {

typedef float floatx4v __attribute__((ext_vector_type(4)));

// 16 bytes of values, at an address that is aligned to 16 bytes or to a value only:
// global memory takes wide accesses at any such address, and the compiler makes them of this.
template <typename T, bool ALIGNED>
struct Wide {
  typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef T Loose __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  typedef std::conditional_t<ALIGNED, Vec, Loose> Type;
  static constexpr int kValues = 16 / sizeof(T);
};

// Eight values at p (n of them exist), zeros behind them. VEC: p is aligned to 16
// bytes, and all eight exist or none.
template <typename T, bool VEC>
__device__ __forceinline__ void Load8(const T *p, int n, float (&x)[8]) {
  typedef Wide<T, VEC> W;
  if (n >= 8) {
#pragma unroll
    for (int v = 0; v < 8 / W::kValues; ++v) {
      const typename W::Type q = reinterpret_cast<const typename W::Type *>(p)[v];
#pragma unroll
      for (int i = 0; i < W::kValues; ++i) x[v * W::kValues + i] = static_cast<float>(q[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = !VEC && i < n ? static_cast<float>(p[i]) : 0.0f;
}

// Eight values to p, each rounded to T, n of them.
template <typename T, bool VEC>
__device__ __forceinline__ void Store8(T *p, int n, const float (&x)[8]) {
  typedef Wide<T, VEC> W;
  if (n >= 8) {
#pragma unroll
    for (int v = 0; v < 8 / W::kValues; ++v) {
      typename W::Type q;
#pragma unroll
      for (int i = 0; i < W::kValues; ++i) q[i] = static_cast<T>(x[v * W::kValues + i]);
      reinterpret_cast<typename W::Type *>(p)[v] = q;
    }
    return;
  }
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<T>(x[i]);
  }
}

// Eight codes to p, n of them.
template <bool VEC>
__device__ __forceinline__ void StoreCodes8(uint8_t *p, int n, int2 code) {
  typedef int Pair __attribute__((ext_vector_type(2)));
  typedef int Loose __attribute__((ext_vector_type(2), aligned(1)));
  typedef std::conditional_t<VEC, Pair, Loose> Type;
  if (n >= 8) {
    *reinterpret_cast<Type *>(p) = Type{code.x, code.y};
    return;
  }
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? code.x : code.y) >> (8 * (i & 3)));
  }
}

// The bits of the largest magnitude: as integers, magnitudes order like their
// values, infinity above them and NaN on top.
__device__ __forceinline__ uint32_t TopBits(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  return top;
}

// Four e4m3 codes of four values, ties to even.
__device__ __forceinline__ int Codes4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// What the codes of eight values of a row's block of 128 are rounded from, the block's largest
// magnitude having the bits `top`: 448 x / amax, amax at least 2^-100. FP32: the values are fp32, not
// widened 16-bit ones. The quotient is correctly rounded to fp32 (for fp32 x up to
// rare double roundings of a 2^-47 residue), since half-way codes are common among
// 16-bit rows and a reciprocal's rounding would push them to either side: with
// a = amax 2^-e in [1, 2) and r the rounded 1 / a, q0 = t r is off by at most
// two units, its remainder t - q0 a is exact in one fma, and q0 + remainder r
// rounds to the nearest (Markstein). t = 448 x 2^-e carries its own rounding
// error along for fp32 rows. Four to six operations a value instead of a
// division's eleven.
constexpr uint32_t kLeastAmax = static_cast<uint32_t>(127 - 100) << 23;  // 2^-100

template <bool FP32>
__device__ __forceinline__ void BlockQuotients(const float (&x)[8], uint32_t top, float (&q)[8],
                                               float *amax_out) {
  const float amax = __uint_as_float(max(top, kLeastAmax));
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
  if (top < 0x7F800000u) {
    const float a = ldexpf(amax, -e);
    const float r = 1.0f / a;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float xs = ldexpf(x[i], -e);
      const float t = xs * 448.0f;
      const float q0 = t * r;
      float rem = fmaf(-q0, a, t);
      if constexpr (FP32) rem += fmaf(xs, 448.0f, -t);
      q[i] = fmaf(rem, r, q0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = x[i] / amax;  // 0 where x is finite (448 x may not be)
  }
  *amax_out = amax;
}

__device__ __forceinline__ int2 Codes8(const float (&q)[8]) {
  return make_int2(Codes4(q[0], q[1], q[2], q[3]), Codes4(q[4], q[5], q[6], q[7]));
}

} // namespace mnb

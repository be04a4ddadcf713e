// RMS norm with the residual's addition, to 8-bit codes with block scales or to
// the rows' own type: kernel and C ABI.
#include "mnb_values.h"
#include "../../include/mnb_norm.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace mnb;

constexpr int kMaxThreads = 1024;
constexpr int kBlock = MNB_FP8_BLOCK;

struct Args {
  const void *X, *R;
  const float *gamma;
  void *Y, *H;
  float *scales;
  int64_t K, ldx, ldr;
  float epsilon;
};

// v rounded to fp32 such that a second rounding, to a code, is that of v itself: to the neighbour
// with an odd last bit, if it is none.
__device__ __forceinline__ float RoundToOdd(double v) {
  const float f = static_cast<float>(v);
  const double rest = v - static_cast<double>(f);
  const uint32_t u = __float_as_uint(f);
  if (rest == 0.0 || f == 0.0f || (u & 1) != 0) return f;
  return __uint_as_float((rest > 0.0) == (f > 0.0f) ? u + 1 : u - 1);
}

// Codes of eight values h g of a block of 128 that 16 lanes hold, the nearest to 448 h g /
// amax. The row's factor norm is in y = h g norm as in amax, which has the bits `top`, and drops
// out. In fp32 the quotient is off by seven half units, 2^-24, at most: two each of y and amax, the
// reciprocal's two and its product's. `less` and `more` hold it between them: 8 half units below
// what was computed and 10 above it. Only where their codes differ, in one of 2^16, can it matter: a
// wavefront that has such a code computes them again in 64 bits, where products and the middle
// between two codes are exact. 8192 rows of 4096 take what they took with fp32 codes alone (44 us
// over and over), rows of 16384, whose registers it raises from 69 to 90, 50 us for 46 (2000).
__device__ __forceinline__ int2 NearestCodes(const float (&y)[8], const float (&h)[8],
                                             const float (&g)[8], uint32_t top, float *amax) {
  *amax = __uint_as_float(max(top, kLeastAmax));
  const float by = 448.0f / *amax * (1.0f - 0x1p-21f);
  float less[8], more[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    less[i] = y[i] * by;
    more[i] = less[i] * (1.0f + 0x1.2p-20f);
  }
  int2 code = Codes8(less);
  const int2 other = Codes8(more);
  if (__any(code.x != other.x || code.y != other.y)) {
    double most = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmax(most, fabs(static_cast<double>(h[i]) * g[i]));
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) most = fmax(most, __shfl_xor(most, off, 16));
    float q[8];
    if (top > kLeastAmax && top < 0x7F800000u) {
      const double over = 1.0 / most;
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // the nearest quotient, as in BlockQuotients
        const double t = static_cast<double>(h[i]) * g[i] * 448.0, q0 = t * over;
        q[i] = RoundToOdd(fma(fma(-q0, most, t), over, q0));
      }
    } else {
      BlockQuotients<true>(y, top, q, amax);
    }
    code = Codes8(q);
  }
  return code;
}

// One workgroup per row; thread t holds the units of eight values t, t + T, ...,
// so that a block of 128 is 16 neighbouring lanes. NV > 0: a row of at most NV T
// units stays in registers between the sum of its squares and its second use, one
// read of X and R and one write of each result; NV == 0: longer rows are read
// again (h from where it was stored). Many rows are bound by memory: 8192 rows of 4096,
// bf16, with residual and codes take 48 us (236 MB, 4.9 TB/s; 43 over and over, where the
// last cache holds most of them), 333 fp32 rows of 2500 4.4. Few are one round trip to memory
// and the sum's: one row of 4096 3.1 us.
template <typename T, bool VEC, bool CODES, int NV>
__global__ __launch_bounds__(kMaxThreads) void RmsNormKernel(Args a) {
  constexpr int kUnits = NV > 0 ? NV : 1;
  const int threads = blockDim.x, t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(a.X) + row * a.ldx;
  const T *r = a.R ? static_cast<const T *>(a.R) + row * a.ldr : nullptr;
  T *h = a.R ? static_cast<T *>(a.H) + row * a.K : nullptr;
  const int units = static_cast<int>((a.K + 7) / 8);
  const int rounds = NV > 0 ? NV : (units + threads - 1) / threads;
  float v[kUnits][8];
  float sum = 0.0f;
  const auto load = [&](int j, float(&out)[8]) {
    const int64_t k0 = 8 * (static_cast<int64_t>(j) * threads + t);
    const int n = static_cast<int>(min(int64_t{8}, a.K - k0));  // <= 0 past the row
    Load8<T, VEC>(x + k0, n, out);
    if (r) {
      float add[8];
      Load8<T, VEC>(r + k0, n, add);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = static_cast<float>(static_cast<T>(out[i] + add[i]));
      Store8<T, VEC>(h + k0, n, out);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(out[i], out[i], sum);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) load(j, v[j]);
  } else {
    for (int j = 0; j < rounds; ++j) load(j, v[0]);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
  double total = sum;
  if (threads > 64) {
    __shared__ float part[kMaxThreads / 64];
    if ((t & 63) == 0) part[t >> 6] = sum;
    __syncthreads();
    total = 0.0;
    for (int w = 0; w < threads / 64; ++w) total += part[w];
  }
  // One rounding for the factor that all values of the row share.
  const float norm = static_cast<float>(
      rsqrt(total / static_cast<double>(a.K) + static_cast<double>(a.epsilon)));
  const int64_t nb = (a.K + kBlock - 1) / kBlock;
  const auto finish = [&](int j, float(&y)[8]) {
    const int64_t k0 = 8 * (static_cast<int64_t>(j) * threads + t);
    const int n = static_cast<int>(min(int64_t{8}, a.K - k0));
    float g[8], h[8];
    Load8<float, VEC>(a.gamma + k0, n, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] = y[i];
      y[i] = n > i ? y[i] * norm * g[i] : 0.0f;
    }
    if constexpr (CODES) {
      uint32_t top = TopBits(y);
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1)
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 16)));
      float amax;
      const int2 code = NearestCodes(y, h, g, top, &amax);
      if (n <= 0) return;
      if ((t & 15) == 0) a.scales[row * nb + k0 / kBlock] = amax / 448.0f;
      StoreCodes8<VEC>(static_cast<uint8_t *>(a.Y) + row * a.K + k0, n, code);
    } else {
      Store8<T, VEC>(static_cast<T *>(a.Y) + row * a.K + k0, n, y);
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) finish(j, v[j]);
  } else {
    for (int j = 0; j < rounds; ++j) {
      const int64_t k0 = 8 * (static_cast<int64_t>(j) * threads + t);
      Load8<T, VEC>((r ? h : x) + k0, static_cast<int>(min(int64_t{8}, a.K - k0)), v[0]);
      finish(j, v[0]);
    }
  }
}

template <typename T, bool VEC, bool CODES>
hipError_t Launch(Args a, int64_t M, hipStream_t s) {
  const int64_t units = (a.K + 7) / 8;
  const int waves = static_cast<int>(std::min<int64_t>(kMaxThreads / 64, (units + 63) / 64));
  int threads = 64 * waves;
  // Many rows: fewer threads with more units each, so that a CU holds several rows (8192 rows
  // of 4096, over and over: 43.3 us, 46.4 with a unit a thread; 600 rows 6.5 and 6.7). Few rows are done
  // sooner with a unit a thread (256 rows of 8192: 5.7 us, 8.6 with four).
  if (M > 512)
    while (threads > 256 && (threads / 2) % 64 == 0 && units <= 4 * (threads / 2)) threads /= 2;
  const int64_t nv = (units + threads - 1) / threads;
  const int64_t size = sizeof(T), ysize = CODES ? 1 : size;
  const int64_t nb = (a.K + kBlock - 1) / kBlock;
  // Rows at a time, so that a grid's threads stay below 2^32.
  const int64_t rows = int64_t{1} << 21;
  for (int64_t m = 0; m < M; m += rows) {
    const dim3 grid(static_cast<unsigned>(std::min(rows, M - m))), block(threads);
    Args b = a;
    b.X = static_cast<const char *>(a.X) + m * a.ldx * size;
    if (a.R) {
      b.R = static_cast<const char *>(a.R) + m * a.ldr * size;
      b.H = static_cast<char *>(a.H) + m * a.K * size;
    }
    b.Y = static_cast<char *>(a.Y) + m * a.K * ysize;
    if (CODES) b.scales = a.scales + m * nb;
    if (nv == 1)
      hipLaunchKernelGGL((RmsNormKernel<T, VEC, CODES, 1>), grid, block, 0, s, b);
    else if (nv == 2)
      hipLaunchKernelGGL((RmsNormKernel<T, VEC, CODES, 2>), grid, block, 0, s, b);
    else if (nv <= 4)
      hipLaunchKernelGGL((RmsNormKernel<T, VEC, CODES, 4>), grid, block, 0, s, b);
    else
      hipLaunchKernelGGL((RmsNormKernel<T, VEC, CODES, 0>), grid, block, 0, s, b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

bool Aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
hipError_t Choose(const Args &a, int64_t M, bool codes, hipStream_t s) {
  const int64_t size = sizeof(T);
  const bool vec = a.K % 8 == 0 && a.ldx * size % 16 == 0 && a.ldr * size % 16 == 0 &&
                   Aligned(a.X, 16) && Aligned(a.R, 16) && Aligned(a.H, 16) &&
                   Aligned(a.gamma, 16) && Aligned(a.Y, codes ? 8 : 16);
  if (vec) return codes ? Launch<T, true, true>(a, M, s) : Launch<T, true, false>(a, M, s);
  return codes ? Launch<T, false, true>(a, M, s) : Launch<T, false, false>(a, M, s);
}

} // namespace

extern "C" int mnb_rms_norm(int64_t M, int64_t K, int32_t x_type, const void *dX, int64_t ldx,
                            const void *dResidual, int64_t ldr, const float *dGamma, float epsilon,
                            int32_t y_type, void *dY, float *dScales, void *dSum, void *stream) {
  const bool codes = y_type == MNB_TYPE_FLOAT8E4M3FN;
  if (x_type != MNB_TYPE_FLOAT && x_type != MNB_TYPE_FLOAT16 && x_type != MNB_TYPE_BFLOAT16)
    return MNB_ERR_BAD_ATTRIBUTE;
  if (!codes && y_type != x_type) return MNB_ERR_BAD_ATTRIBUTE;
  if (!(epsilon >= 0.0f) || std::isinf(epsilon)) return MNB_ERR_BAD_ATTRIBUTE;
  const int64_t far = int64_t{1} << 40;
  if (M < 0 || M > (int64_t{1} << 30) || K <= 0 || K > (int64_t{1} << 22) || ldx < K || ldx > far)
    return MNB_ERR_BAD_SHAPE;
  if (dResidual != nullptr && (ldr < K || ldr > far)) return MNB_ERR_BAD_SHAPE;
  if (M == 0) return MNB_OK;
  if (dX == nullptr || dGamma == nullptr || dY == nullptr) return MNB_ERR_NULL_POINTER;
  if (codes != (dScales != nullptr)) return codes ? MNB_ERR_NULL_POINTER : MNB_ERR_UNSUPPORTED;
  if ((dResidual != nullptr) != (dSum != nullptr))
    return dSum == nullptr ? MNB_ERR_NULL_POINTER : MNB_ERR_UNSUPPORTED;
  const uintptr_t size = x_type == MNB_TYPE_FLOAT ? 4 : 2;
  if (!Aligned(dX, size) || !Aligned(dResidual, size) || !Aligned(dSum, size) ||
      !Aligned(dGamma, 4) || !Aligned(dScales, 4) || !Aligned(dY, codes ? 1 : size))
    return MNB_ERR_BAD_SHAPE;
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) {
    SetLastHipError("hipGetDevice", e);
    return MNB_ERR_NO_DEVICE;
  }
  const Args a{dX, dResidual, dGamma, dY, dSum, dScales, K, ldx, dResidual ? ldr : 0, epsilon};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (x_type) {
  case MNB_TYPE_FLOAT16: e = Choose<_Float16>(a, M, codes, s); break;
  case MNB_TYPE_BFLOAT16: e = Choose<__bf16>(a, M, codes, s); break;
  default: e = Choose<float>(a, M, codes, s);
  }
  if (e == hipSuccess) return MNB_OK;
  SetLastHipError("RMS norm", e);
  return MNB_ERR_HIP;
}

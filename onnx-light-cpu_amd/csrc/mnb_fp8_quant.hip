// Rows to e4m3 with a scale for each block of 128, the weight layout of the
// 8-bit product, and the padding of ragged code rows.
#include "mnb_fp8.h"
#include "mnb_values.h"

namespace mnb {
namespace fp8 {
namespace {

constexpr int kThreads = 256;

// One (row, block) item per 16 lanes, eight values a lane; bound by memory.
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
  uint32_t top = TopBits(x);
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1)
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 16)));
  float amax, q[8];
  BlockQuotients<sizeof(T) == 4>(x, top, q, &amax);
  const int2 code = Codes8(q);
  if ((threadIdx.x & 15) == 0) S[item] = amax / 448.0f;
  StoreCodes8<VEC>(Q + row * ldq + k0, static_cast<int>(min(int64_t{8}, ldq - k0)), code);
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

// Rotary positions with several axes: kernel and C ABI.
#include "mnb_values.h"
#include "../../include/mnb_rotary.h"

#include <algorithm>

namespace {

using namespace mnb;

constexpr int kThreads = 256;
constexpr int kMaxPairs = MNB_ROTARY_MAX_PAIRS;

struct Part {
  const void *x;
  void *y;
  int64_t xt, xh, yt, yh;  // token and head strides
};

struct Args {
  Part part[2];
  const void *pos;
  int64_t axis_stride, T;
  int32_t heads0, heads;  // query heads, all heads
  int32_t head_dim, pairs;
  int32_t tokens;         // a workgroup's
  bool pos64, interleaved;
};

// Frequencies travel with the launch, so that a call depends on no memory but its tensors;
// a launch with 64 of them is 1.7 KiB shorter than one with 256.
template <int PAIRS>
struct Frequencies {
  uint64_t turns[PAIRS];
  uint8_t axis[PAIRS];
};

// cos and sin of `turn` 2^-64 turns. The nearest quarter turn goes off in
// integers; what is left is at most an eighth, x = 2 pi r with |x| <= pi / 4,
// where the Taylor series to x^9 and x^10 are off by 2e-9 and 3e-10.
__device__ __forceinline__ float2 CosSin(uint64_t turn) {
  const uint64_t quarter = (turn + (uint64_t{1} << 61)) >> 62;
  const int32_t rest = static_cast<int32_t>((turn - (quarter << 62)) >> 32);
  const float x = static_cast<float>(rest) * 0x1.921fb6p-30f;  // 2 pi 2^-32
  const float z = x * x;
  float s = fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = fmaf(z, s, 1.0f / 120.0f);
  s = fmaf(z, s, -1.0f / 6.0f);
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(z, c, -1.0f / 720.0f);
  c = fmaf(z, c, 1.0f / 24.0f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const bool swap = quarter & 1;
  const float u = swap ? s : c, v = swap ? c : s;
  return make_float2((quarter + 1) & 2 ? -u : u, quarter & 2 ? -v : v);
}

// A workgroup first makes the cos and sin of its tokens in LDS, once for all
// heads (one 64-bit product, 30 operations a pair), then turns the heads: an
// item is one head's eight pairs, two loads and two stores of 16 bytes for 16-bit
// types. Memory bounds it: 6144 tokens of 40 heads of 128, bf16, take 24 us (126 MB,
// 5.1 TB/s; 21 over and over, from the last cache in part); 64 tokens 4.3, which is the launch
// and three trips to memory one after another.
template <typename T, bool VEC, int PAIRS>
__global__ __launch_bounds__(kThreads) void RotaryKernel(Args a, Frequencies<PAIRS> f) {
  extern __shared__ float2 table[];  // [tokens][pairs]
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(a.tokens), a.T - t0));
  for (int i = threadIdx.x; i < tokens * a.pairs; i += kThreads) {
    const int t = i / a.pairs, j = i - t * a.pairs;
    const int64_t at = f.axis[j] * a.axis_stride + t0 + t;
    const int64_t p = a.pos64 ? static_cast<const int64_t *>(a.pos)[at]
                              : static_cast<const int32_t *>(a.pos)[at];
    table[i] = CosSin(static_cast<uint64_t>(p) * f.turns[j]);
  }
  __syncthreads();
  const int rot = (a.pairs + 7) / 8;                       // items of a head that turn,
  const int kept = (a.head_dim - 2 * a.pairs + 15) / 16;   // and that are copied
  const int each = rot + kept, total = tokens * a.heads * each;
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < total; i += gridDim.y * kThreads) {
    const int th = i / each, item = i - th * each;
    const int t = th / a.heads, all = th - t * a.heads;
    const Part &p = all < a.heads0 ? a.part[0] : a.part[1];
    const int h = all < a.heads0 ? all : all - a.heads0;
    const T *x = static_cast<const T *>(p.x) + (t0 + t) * p.xt + h * p.xh;
    T *y = static_cast<T *>(p.y) + (t0 + t) * p.yt + h * p.yh;
    float lo[8], hi[8];
    if (item >= rot) {
      if (x == y) continue;
      const int d = 2 * a.pairs + 16 * (item - rot), n = a.head_dim - d;
      Load8<T, VEC>(x + d, n, lo);
      Load8<T, VEC>(x + d + 8, n - 8, hi);
      Store8<T, VEC>(y + d, n, lo);
      Store8<T, VEC>(y + d + 8, n - 8, hi);
      continue;
    }
    const int j = 8 * item, n = a.pairs - j;
    const float2 *cs = table + t * a.pairs + j;
    float2 w[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) w[q] = VEC || q < n ? cs[q] : make_float2(0.0f, 0.0f);
    if (a.interleaved) {
      Load8<T, VEC>(x + 2 * j, 2 * n, lo);
      Load8<T, VEC>(x + 2 * j + 8, 2 * n - 8, hi);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float *pair = q < 4 ? lo + 2 * q : hi + 2 * (q - 4);
        const float u = pair[0], v = pair[1];
        pair[0] = fmaf(u, w[q].x, -(v * w[q].y));
        pair[1] = fmaf(v, w[q].x, u * w[q].y);
      }
      Store8<T, VEC>(y + 2 * j, 2 * n, lo);
      Store8<T, VEC>(y + 2 * j + 8, 2 * n - 8, hi);
    } else {
      Load8<T, VEC>(x + j, n, lo);
      Load8<T, VEC>(x + a.pairs + j, n, hi);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float u = lo[q], v = hi[q];
        lo[q] = fmaf(u, w[q].x, -(v * w[q].y));
        hi[q] = fmaf(v, w[q].x, u * w[q].y);
      }
      Store8<T, VEC>(y + j, n, lo);
      Store8<T, VEC>(y + a.pairs + j, n, hi);
    }
  }
}

bool Aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

bool VecPart(const Part &p, int64_t size) {
  return Aligned(p.x, 16) && Aligned(p.y, 16) && p.xt * size % 16 == 0 && p.xh * size % 16 == 0 &&
         p.yt * size % 16 == 0 && p.yh * size % 16 == 0;
}

template <typename T, int PAIRS>
hipError_t LaunchFor(Args &a, const mnb_rotary_desc &d, hipStream_t s) {
  Frequencies<PAIRS> f;
  std::copy_n(d.turns, a.pairs, f.turns);
  std::copy_n(d.axis, a.pairs, f.axis);
  const int items = a.heads * ((a.pairs + 7) / 8 + (a.head_dim - 2 * a.pairs + 15) / 16);
  // About two items a thread; the table of cos and sin has one entry a thread or
  // little more. Few tokens are shared by several workgroups. (6144 tokens and 64, 40 heads,
  // over and over: 23.0 and 4.3 us; four times as many items 23.5 and 5.2, a quarter 23.3 and 4.6.)
  a.tokens = std::max(1, std::min(2 * kThreads / items, 2 * kThreads / a.pairs));
  const int split = std::min(64, std::max(1, a.tokens * items / (2 * kThreads)));
  const bool vec = a.pairs % 8 == 0 && a.head_dim % 8 == 0 &&
                   VecPart(a.part[0], sizeof(T)) && VecPart(a.part[1], sizeof(T));
  const size_t lds = sizeof(float2) * a.tokens * a.pairs;
  // Tokens at a time, so that a grid's threads stay below 2^32.
  const int64_t most = (int64_t{1} << 23) * a.tokens;
  for (int64_t t = 0; t < a.T; t += most) {
    Args b = a;
    b.T = std::min(most, a.T - t);
    b.pos = static_cast<const char *>(a.pos) + t * (a.pos64 ? 8 : 4);
    for (Part &p : b.part) {
      p.x = static_cast<const T *>(p.x) + t * p.xt;
      p.y = static_cast<T *>(p.y) + t * p.yt;
    }
    const dim3 grid(static_cast<unsigned>((b.T + b.tokens - 1) / b.tokens), split);
    if (vec)
      hipLaunchKernelGGL((RotaryKernel<T, true, PAIRS>), grid, dim3(kThreads), lds, s, b, f);
    else
      hipLaunchKernelGGL((RotaryKernel<T, false, PAIRS>), grid, dim3(kThreads), lds, s, b, f);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t Launch(Args &a, const mnb_rotary_desc &d, hipStream_t s) {
  return a.pairs <= 64 ? LaunchFor<T, 64>(a, d, s) : LaunchFor<T, kMaxPairs>(a, d, s);
}

int CheckHeads(const mnb_rotary_heads *h, int64_t head_dim, uintptr_t size) {
  if (h->heads < 0 || h->heads > (1 << 16)) return MNB_ERR_BAD_SHAPE;
  if (h->heads == 0) return MNB_OK;
  if (h->x == nullptr || h->y == nullptr) return MNB_ERR_NULL_POINTER;
  const int64_t far = int64_t{1} << 36;
  for (const int64_t v : {h->x_token_stride, h->x_head_stride, h->y_token_stride, h->y_head_stride})
    if (v < head_dim || v > far) return MNB_ERR_BAD_SHAPE;
  if (!Aligned(h->x, size) || !Aligned(h->y, size)) return MNB_ERR_BAD_SHAPE;
  if (h->x == h->y &&
      (h->x_token_stride != h->y_token_stride || h->x_head_stride != h->y_head_stride))
    return MNB_ERR_UNSUPPORTED;
  return MNB_OK;
}

} // namespace

extern "C" int mnb_rotary(const mnb_rotary_desc *desc, int64_t T, int32_t pos_type,
                          const void *positions, int64_t axis_stride, int32_t x_type,
                          const mnb_rotary_heads *query, const mnb_rotary_heads *key,
                          void *stream) {
  if (desc == nullptr || query == nullptr) return MNB_ERR_NULL_POINTER;
  if (x_type != MNB_TYPE_FLOAT && x_type != MNB_TYPE_FLOAT16 && x_type != MNB_TYPE_BFLOAT16)
    return MNB_ERR_BAD_ATTRIBUTE;
  if (pos_type != MNB_TYPE_INT32 && pos_type != MNB_TYPE_INT64) return MNB_ERR_BAD_ATTRIBUTE;
  const int D = desc->head_dim, R = desc->rotary_dim;
  if (D <= 0 || D > 4096 || R < 2 || R > D || R % 2 != 0 || R > 2 * kMaxPairs)
    return MNB_ERR_BAD_SHAPE;
  if (desc->axes < 1 || desc->axes > MNB_ROTARY_MAX_AXES) return MNB_ERR_BAD_ATTRIBUTE;
  if (desc->interleaved != 0 && desc->interleaved != 1) return MNB_ERR_BAD_ATTRIBUTE;
  if (desc->turns == nullptr || desc->axis == nullptr) return MNB_ERR_NULL_POINTER;
  if (T < 0 || T > (int64_t{1} << 24)) return MNB_ERR_BAD_SHAPE;
  if (axis_stride < (desc->axes > 1 ? T : 0) || axis_stride > (int64_t{1} << 36))
    return MNB_ERR_BAD_SHAPE;
  Args a;
  a.pairs = R / 2;
  for (int j = 0; j < a.pairs; ++j)
    if (desc->axis[j] >= desc->axes) return MNB_ERR_BAD_ATTRIBUTE;
  const uintptr_t size = x_type == MNB_TYPE_FLOAT ? 4 : 2;
  if (T == 0) return MNB_OK;
  a.heads0 = query->heads;
  a.heads = query->heads;
  a.part[0] = a.part[1] = Part{};
  int st = CheckHeads(query, D, size);
  if (st != MNB_OK) return st;
  if (query->heads > 0)
    a.part[0] = {query->x, query->y, query->x_token_stride, query->x_head_stride,
                 query->y_token_stride, query->y_head_stride};
  if (key != nullptr) {
    st = CheckHeads(key, D, size);
    if (st != MNB_OK) return st;
    a.heads += key->heads;
    if (key->heads > 0)
      a.part[1] = {key->x, key->y, key->x_token_stride, key->x_head_stride,
                   key->y_token_stride, key->y_head_stride};
  }
  if (a.heads == 0) return MNB_OK;
  if (positions == nullptr) return MNB_ERR_NULL_POINTER;
  a.pos64 = pos_type == MNB_TYPE_INT64;
  if (!Aligned(positions, a.pos64 ? 8 : 4)) return MNB_ERR_BAD_SHAPE;
  a.pos = positions;
  a.axis_stride = axis_stride;
  a.T = T;
  a.head_dim = D;
  a.interleaved = desc->interleaved != 0;
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) {
    SetLastHipError("hipGetDevice", e);
    return MNB_ERR_NO_DEVICE;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (x_type) {
  case MNB_TYPE_FLOAT16: e = Launch<_Float16>(a, *desc, s); break;
  case MNB_TYPE_BFLOAT16: e = Launch<__bf16>(a, *desc, s); break;
  default: e = Launch<float>(a, *desc, s);
  }
  if (e == hipSuccess) return MNB_OK;
  SetLastHipError("rotary positions", e);
  return MNB_ERR_HIP;
}

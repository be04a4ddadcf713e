// New keys and values into the 8-bit cache.
#include "mnb_kv.h"
#include "mnb_values.h"

namespace mnb {
namespace kv {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void Load16(const T *p, float (&x)[16]) {
  float lo[8], hi[8];
  Load8<T, true>(p, 8, lo);
  Load8<T, true>(p + 8, 8, hi);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = lo[i];
    x[8 + i] = hi[i];
  }
}

__device__ __forceinline__ bool Finite(float x) {
  return (__float_as_uint(x) & 0x7FFFFFFFu) < 0x7F800000u;
}

// Sixteen codes of x / scale, NaN where x is not finite; by is 1 / scale. A scale that a page had
// may be no power of two, and its reciprocal's rounding would move halves of a code's last
// place to either side: the quotient's remainder, exact in one fma, corrects it.
__device__ __forceinline__ uint4 Codes16(const float (&x)[16], float scale, float by) {
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = Finite(x[i]) ? x[i] * by : __builtin_nanf("");
  if ((__float_as_uint(scale) & 0x7FFFFFu) != 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = fmaf(fmaf(-y[i], scale, x[i]), by, y[i]);
  }
  uint4 r;
  r.x = Codes4(y[0], y[1], y[2], y[3]);
  r.y = Codes4(y[4], y[5], y[6], y[7]);
  r.z = Codes4(y[8], y[9], y[10], y[11]);
  r.w = Codes4(y[12], y[13], y[14], y[15]);
  return r;
}

__device__ __forceinline__ uint32_t Scaled4(uint32_t code, float by) {
  typedef float floatx2 __attribute__((ext_vector_type(2)));
  const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), false);
  const floatx2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), true);
  return static_cast<uint32_t>(Codes4(a.x * by, a.y * by, b.x * by, b.y * by));
}

// The least power of two, 2^-64 at least, that brings a magnitude with these bits to 448
// = 1.75 2^8 or below.
__device__ __forceinline__ float PageScale(uint32_t top) {
  const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, -64) + 127) << 23);
}

__host__ __device__ inline Units PageUnits(const Cache &c) { return {1, c.page_shift, 2}; }

// One workgroup per page that a sequence's new rows reach, head, and keys or
// values: it alone writes that page, so nothing is atomic. An item is sixteen
// values of a row; the rows are read for their largest magnitude and again, from
// the caches, for their codes. Memory bounds prompts: 2 x 4001 tokens of 8 heads of
// 128, bf16, take 12.6 us (33 MB read, 16 written: 3.9 TB/s). A token of each of 64 sequences takes
// 4.6: table, old scale and rows are three trips to memory, a page that grows a fourth.
template <typename T>
__global__ __launch_bounds__(kThreads) void AppendKernel(Cache c, Batch b, Rows k, Rows v) {
  int s = blockIdx.z, nth = blockIdx.x;  // of the pages that this sequence's rows reach
  const int h = blockIdx.y >> 1, which = blockIdx.y & 1;
  if (b.starts != nullptr) {
    int64_t unit;
    s = SequenceOf(b, PageUnits(c), blockIdx.x, &unit);
    nth = blockIdx.x - static_cast<int>(unit);
    if (nth < 0) return;
  }
  const Span span = SpanOf(b, s, c.page_shift);
  const int page = 1 << c.page_shift;
  const int first = max(span.first, 0);
  if (first >= span.end) return;
  const int p = (first >> c.page_shift) + nth;
  const int64_t begin = static_cast<int64_t>(p) << c.page_shift;
  if (begin >= span.end) return;
  const int lo = max(first - static_cast<int>(begin), 0);  // the new tokens' slots
  const int hi = min(span.end - static_cast<int>(begin), page);
  const uint32_t id = PageOf(b, s, p);
  if (id >= c.pages) return;
  const Rows &rows = which ? v : k;
  const T *x = static_cast<const T *>(rows.x) + h * rows.head_stride +
               (span.row + static_cast<int>(begin) + lo - span.first) * rows.token_stride;
  const int64_t at = static_cast<int64_t>(id) * c.heads + h;
  uint8_t *codes = c.codes[which] + ((at * c.dim) << c.page_shift);
  const int per = c.dim / 16, total = (hi - lo) * per;

  uint32_t top = 0;
  for (int u = threadIdx.x; u < total; u += kThreads) {
    const int t = u / per, d = 16 * (u - t * per);
    float f[16];
    Load16(x + t * rows.token_stride + d, f);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (Finite(f[i])) top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off)));
  __shared__ uint32_t tops[kThreads / 64];
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  const float old = lo > 0 ? c.scales[which][at] : 0.0f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = max(top, tops[w]);
  const float scale = fmaxf(old, PageScale(top));
  if (lo > 0 && old != scale) {
    const float by = old / scale;
    for (int u = threadIdx.x; u < page * per; u += kThreads) {
      const int t = u / per;
      if (t >= lo && t < hi) continue;
      uint4 *q = reinterpret_cast<uint4 *>(codes) + u;
      const uint4 w = *q;
      *q = make_uint4(Scaled4(w.x, by), Scaled4(w.y, by), Scaled4(w.z, by), Scaled4(w.w, by));
    }
  }
  const float by = 1.0f / scale;
  for (int u = threadIdx.x; u < total; u += kThreads) {
    const int t = u / per, d = 16 * (u - t * per);
    float f[16];
    Load16(x + t * rows.token_stride + d, f);
    reinterpret_cast<uint4 *>(codes)[lo * per + u] = Codes16(f, scale, by);
  }
  if (threadIdx.x == 0) c.scales[which][at] = scale;
}

template <typename T>
hipError_t Launch(const Cache &c, const Batch &b, const Rows &k, const Rows &v, hipStream_t s) {
  const int64_t page = int64_t{1} << c.page_shift;
  // Pages that max_tokens neighbouring positions reach at most; the table has no more.
  const int64_t reach = std::min<int64_t>((b.max_tokens + page - 2) / page + 1, b.width);
  const dim3 grid(
      static_cast<unsigned>(b.starts == nullptr ? reach : UnitsOf(b, PageUnits(c))), 2u * c.heads,
      b.starts == nullptr ? b.sequences : 1);
  hipLaunchKernelGGL((AppendKernel<T>), grid, dim3(kThreads), 0, s, c, b, k, v);
  return hipGetLastError();
}

} // namespace

hipError_t LaunchAppend(const Cache &c, const Batch &b, int32_t x_type, const Rows &k,
                        const Rows &v, hipStream_t s) {
  switch (x_type) {
  case MNB_TYPE_FLOAT16: return Launch<_Float16>(c, b, k, v, s);
  case MNB_TYPE_BFLOAT16: return Launch<__bf16>(c, b, k, v, s);
  default: return Launch<float>(c, b, k, v, s);
  }
}

} // namespace kv
} // namespace mnb

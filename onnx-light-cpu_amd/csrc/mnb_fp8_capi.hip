// C ABI of the 8-bit product: validation, plan lifetime, workspace layout.
#include "mnb_fp8.h"

#include <new>

struct mnb_fp8_plan {
  mnb::fp8::Weight w;
  int device;
  uint8_t *records;
  float *scales;
  size_t bytes;
};

namespace {

using mnb::fp8::CeilDiv;
using mnb::fp8::kBlock;

bool FloatType(int32_t t) {
  return t == MNB_TYPE_FLOAT || t == MNB_TYPE_FLOAT16 || t == MNB_TYPE_BFLOAT16;
}

bool Aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

size_t Round256(size_t v) { return (v + 255) / 256 * 256; }

constexpr int64_t kMaxRows = int64_t{1} << 30;
constexpr int64_t kMaxK = int64_t{1} << 22;
constexpr int64_t kMaxN = int64_t{1} << 26;
constexpr int64_t kMaxY = int64_t{1} << 36;  // M * N: grids stay below 2^32 threads

int Fail(const char *what, hipError_t e, int status) {
  mnb::SetLastHipError(what, e);
  return status;
}

void FreePlan(mnb_fp8_plan *p) {
  if (p->records) (void)hipFree(p->records);
  if (p->scales) (void)hipFree(p->scales);
  delete p;
}

int CheckPlanInputs(int64_t K, int64_t N, const void *W, const void *scales,
                    mnb_fp8_plan **out_plan) {
  if (out_plan == nullptr) return MNB_ERR_NULL_POINTER;
  *out_plan = nullptr;
  if (K <= 0 || N <= 0 || K > kMaxK || N > kMaxN) return MNB_ERR_BAD_SHAPE;
  if (W == nullptr || scales == nullptr) return MNB_ERR_NULL_POINTER;
  return MNB_OK;
}

// W and scales: device pointers (device) or host pointers.
int Create(int64_t K, int64_t N, const uint8_t *W, const float *scales, bool device,
           mnb_fp8_plan **out_plan) {
  int dev = -1;
  const int st = mnb::CurrentGfx950(&dev);
  if (st != MNB_OK) return st;
  mnb_fp8_plan *p = new (std::nothrow) mnb_fp8_plan();
  if (p == nullptr) return MNB_ERR_ALLOC;
  p->device = dev;
  mnb::fp8::Weight &w = p->w;
  w.K = K;
  w.N = N;
  w.nb = CeilDiv(K, kBlock);
  w.groups = CeilDiv(N, 64);
  w.num_cus = mnb::DeviceComputeUnits(dev);
  const size_t rec_bytes = static_cast<size_t>(w.groups) * w.nb * 64 * kBlock;
  const size_t s_bytes = static_cast<size_t>(CeilDiv(N, kBlock)) * w.nb * sizeof(float);
  p->bytes = rec_bytes + s_bytes;
  uint8_t *staged = nullptr;
  hipError_t e = hipMalloc(reinterpret_cast<void **>(&p->records), rec_bytes);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->scales), s_bytes);
  if (e == hipSuccess && !device)
    e = hipMalloc(reinterpret_cast<void **>(&staged), static_cast<size_t>(N) * K);
  if (e != hipSuccess) {
    (void)hipGetLastError();  // the failed allocation's, reported here
    FreePlan(p);
    return Fail("hipMalloc", e, MNB_ERR_ALLOC);
  }
  // The copies run on the null stream, which does not wait for non-blocking
  // streams: every write to the sources must have landed first.
  if (device) e = hipDeviceSynchronize();
  else e = hipMemcpy(staged, W, static_cast<size_t>(N) * K, hipMemcpyHostToDevice);
  if (e == hipSuccess)
    e = hipMemcpy(p->scales, scales, s_bytes,
                  device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
  w.W = p->records;
  w.scales = p->scales;
  if (e == hipSuccess) e = mnb::fp8::LaunchRelayout(device ? W : staged, w, p->records, nullptr);
  if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
  if (staged) (void)hipFree(staged);
  if (e != hipSuccess) {
    FreePlan(p);
    return Fail("8-bit weight layout", e, MNB_ERR_HIP);
  }
  *out_plan = p;
  return MNB_OK;
}

bool RowsOk(const mnb_fp8_plan *p, int64_t M) {
  return M >= 0 && M <= kMaxRows && M * p->w.N <= kMaxY;
}

// Where a run's parts of the workspace lie.
struct Parts {
  size_t codes = 0, scales = 0, work = 0, total = 0;
  bool quantize = false, pad = false;
};

Parts WorkParts(const mnb_fp8_plan *p, int64_t M, int32_t a_type) {
  Parts r;
  r.quantize = a_type != MNB_TYPE_FLOAT8E4M3FN;
  r.pad = !r.quantize && p->w.K % kBlock != 0;
  size_t at = 0;
  if (r.quantize || r.pad) at += Round256(static_cast<size_t>(M) * p->w.nb * kBlock);
  r.scales = at;
  if (r.quantize) at += Round256(static_cast<size_t>(M) * p->w.nb * sizeof(float));
  r.work = at;
  r.total = at + mnb::fp8::WorkBytes(p->w, M);
  return r;
}

} // namespace

extern "C" {

int mnb_fp8_quantize(int64_t M, int64_t K, int32_t x_type, const void *dX, int64_t ldx,
                     uint8_t *dQ, float *dScales, void *stream) {
  if (!FloatType(x_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if (M < 0 || M > kMaxRows || K <= 0 || K > kMaxK || ldx < K || ldx > (int64_t{1} << 40))
    return MNB_ERR_BAD_SHAPE;
  if (M == 0) return MNB_OK;
  if (dX == nullptr || dQ == nullptr || dScales == nullptr) return MNB_ERR_NULL_POINTER;
  if (!Aligned(dX, x_type == MNB_TYPE_FLOAT ? 4 : 2) || !Aligned(dScales, 4))
    return MNB_ERR_BAD_SHAPE;
  int dev = -1;
  const hipError_t g = hipGetDevice(&dev);
  if (g != hipSuccess) return Fail("hipGetDevice", g, MNB_ERR_NO_DEVICE);
  const hipError_t e = mnb::fp8::LaunchQuantize(M, K, x_type, dX, ldx, dQ, K, dScales,
                                                static_cast<hipStream_t>(stream));
  return e == hipSuccess ? MNB_OK : Fail("quantize", e, MNB_ERR_HIP);
}

int mnb_fp8_plan_create(int64_t K, int64_t N, const uint8_t *W, const float *scales,
                        mnb_fp8_plan **out_plan) {
  const int st = CheckPlanInputs(K, N, W, scales, out_plan);
  return st != MNB_OK ? st : Create(K, N, W, scales, false, out_plan);
}

int mnb_fp8_plan_create_device(int64_t K, int64_t N, const uint8_t *dW, const float *dScales,
                               mnb_fp8_plan **out_plan) {
  const int st = CheckPlanInputs(K, N, dW, dScales, out_plan);
  if (st != MNB_OK) return st;
  if (!Aligned(dScales, 4)) return MNB_ERR_BAD_SHAPE;
  return Create(K, N, dW, dScales, true, out_plan);
}

int mnb_fp8_plan_destroy(mnb_fp8_plan *plan) {
  if (plan != nullptr) FreePlan(plan);
  return MNB_OK;
}

int mnb_fp8_plan_device_bytes(const mnb_fp8_plan *plan, size_t *bytes) {
  if (plan == nullptr || bytes == nullptr) return MNB_ERR_NULL_POINTER;
  *bytes = plan->bytes;
  return MNB_OK;
}

int mnb_fp8_workspace_bytes(const mnb_fp8_plan *plan, int64_t M, int32_t a_type, size_t *bytes) {
  if (plan == nullptr || bytes == nullptr) return MNB_ERR_NULL_POINTER;
  if (a_type != MNB_TYPE_FLOAT8E4M3FN && !FloatType(a_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if (!RowsOk(plan, M)) return MNB_ERR_BAD_SHAPE;
  *bytes = M == 0 ? 0 : WorkParts(plan, M, a_type).total;
  return MNB_OK;
}

int mnb_fp8_run(const mnb_fp8_plan *plan, int64_t M, int32_t a_type, const void *dA,
                const float *dAScales, int32_t y_type, void *dY, void *dWorkspace,
                size_t workspace_bytes, void *stream) {
  if (plan == nullptr) return MNB_ERR_NULL_POINTER;
  const bool codes = a_type == MNB_TYPE_FLOAT8E4M3FN;
  if ((!codes && !FloatType(a_type)) || !FloatType(y_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if (!RowsOk(plan, M)) return MNB_ERR_BAD_SHAPE;
  if (M == 0) return MNB_OK;
  if (dA == nullptr || dY == nullptr) return MNB_ERR_NULL_POINTER;
  if (codes && dAScales == nullptr) return MNB_ERR_NULL_POINTER;
  if (!codes && dAScales != nullptr) return MNB_ERR_UNSUPPORTED;
  if (!Aligned(dA, 16) || !Aligned(dY, 16) || !Aligned(dWorkspace, 16) || !Aligned(dAScales, 4))
    return MNB_ERR_BAD_SHAPE;
  const Parts parts = WorkParts(plan, M, a_type);
  if (workspace_bytes < parts.total || (dWorkspace == nullptr && parts.total > 0))
    return MNB_ERR_WORKSPACE;
  int cur = -1;
  if (hipGetDevice(&cur) != hipSuccess || cur != plan->device) return MNB_ERR_NO_DEVICE;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const mnb::fp8::Weight &w = plan->w;
  uint8_t *const base = static_cast<uint8_t *>(dWorkspace);
  const uint8_t *a = static_cast<const uint8_t *>(dA);
  const float *sa = dAScales;
  int64_t lda = w.K;
  hipError_t e = hipSuccess;
  if (parts.quantize) {
    lda = w.nb * kBlock;
    float *scales = reinterpret_cast<float *>(base + parts.scales);
    e = mnb::fp8::LaunchQuantize(M, w.K, a_type, dA, w.K, base, lda, scales, s);
    a = base;
    sa = scales;
  } else if (parts.pad) {
    lda = w.nb * kBlock;
    e = mnb::fp8::LaunchPad(M, w.K, a, base, s);
    a = base;
  }
  if (e == hipSuccess)
    e = mnb::fp8::LaunchProduct(w, M, a, lda, sa, y_type, dY, base + parts.work, s);
  return e == hipSuccess ? MNB_OK : Fail("8-bit product", e, MNB_ERR_HIP);
}

const char *mnb_fp8_kernel_name(const mnb_fp8_plan *plan, int64_t M) {
  if (plan == nullptr || M == 0 || !RowsOk(plan, M)) return "";
  return mnb::fp8::ProductKernelName(plan->w, M);
}

} // extern "C"

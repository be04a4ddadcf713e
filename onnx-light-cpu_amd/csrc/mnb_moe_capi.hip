// C ABI of the mixture-of-experts layer: validation, plan lifetime.
#include "mnb_moe.h"

#include <algorithm>
#include <new>

struct mnb_moe_plan {
  mnb::moe::Layer layer;
  int device;
  void *mem[5];  // gate/up records and meta; down's; router
  size_t bytes;
  // Workspace of up to t + 1 tokens a launch. A launch of fewer tokens can need more
  // (down is cut into more parts), and the last launch of a long run may have any number.
  size_t work[mnb::moe::kMaxTokens];
};

namespace {

using mnb::moe::CeilDiv;
using mnb::moe::Half;
using mnb::moe::kMaxTokens;
using mnb::moe::kRec;
using mnb::moe::kRecords;
using mnb::moe::kUnit;

bool FloatType(int32_t t) {
  return t == MNB_TYPE_FLOAT || t == MNB_TYPE_FLOAT16 || t == MNB_TYPE_BFLOAT16;
}

bool Aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int Fail(const char *what, hipError_t e, int status) {
  mnb::SetLastHipError(what, e);
  return status;
}

size_t RunBytes(const mnb_moe_plan *p, int64_t T) {
  return p->work[std::min<int64_t>(T, kMaxTokens) - 1];
}

void FreePlan(mnb_moe_plan *p) {
  for (void *m : p->mem)
    if (m) (void)hipFree(m);
  delete p;
}

constexpr int64_t kMaxWidth = int64_t{1} << 18;  // fixed-point offsets stay below 2^31
constexpr int64_t kMaxMatrix = int64_t{1} << 34;
constexpr int64_t kMaxRun = int64_t{1} << 24;

int CheckPlanInputs(const mnb_moe_desc *d, const mnb_moe_weight *gate, const mnb_moe_weight *up,
                    const mnb_moe_weight *down, mnb_moe_plan **out_plan) {
  if (out_plan == nullptr) return MNB_ERR_NULL_POINTER;
  *out_plan = nullptr;
  if (d == nullptr) return MNB_ERR_NULL_POINTER;
  if (d->bits != 4) return MNB_ERR_UNSUPPORTED;
  if (d->block_size < 16 || (d->block_size & (d->block_size - 1)) != 0)
    return MNB_ERR_BAD_ATTRIBUTE;
  if ((d->normalize != 0 && d->normalize != 1) ||
      (d->has_zero_points != 0 && d->has_zero_points != 1))
    return MNB_ERR_BAD_ATTRIBUTE;
  if (d->hidden <= 0 || d->intermediate <= 0 || d->hidden > kMaxWidth ||
      d->intermediate > kMaxWidth || d->hidden * d->intermediate > kMaxMatrix || d->experts < 1 ||
      d->experts > mnb::moe::kMaxExperts)
    return MNB_ERR_BAD_SHAPE;
  if (d->top_k < 1 || d->top_k > mnb::moe::kMaxTopK || d->top_k > d->experts)
    return MNB_ERR_BAD_ATTRIBUTE;
  for (const mnb_moe_weight *w : {gate, up, down}) {
    if (w == nullptr || w->B == nullptr || w->scales == nullptr) return MNB_ERR_NULL_POINTER;
    if (d->has_zero_points && w->zero_points == nullptr) return MNB_ERR_NULL_POINTER;
    if (!d->has_zero_points && w->zero_points != nullptr) return MNB_ERR_UNSUPPORTED;
  }
  return MNB_OK;
}

int Create(const mnb_moe_desc *d, const float *router, const mnb_moe_weight *gate,
           const mnb_moe_weight *up_w, const mnb_moe_weight *down, bool device,
           mnb_moe_plan **out_plan) {
  int dev = -1;
  const int st = mnb::CurrentGfx950(&dev);
  if (st != MNB_OK) return st;
  mnb_moe_plan *p = new (std::nothrow) mnb_moe_plan();
  if (p == nullptr) return MNB_ERR_ALLOC;
  p->device = dev;
  mnb::moe::Layer &l = p->layer;
  l.hidden = d->hidden;
  l.intermediate = d->intermediate;
  l.experts = d->experts;
  l.top_k = d->top_k;
  l.block_size = d->block_size;
  l.folds = std::max(1, kUnit / d->block_size);
  l.normalize = d->normalize != 0;
  l.zeros = d->has_zero_points != 0;
  l.num_cus = mnb::DeviceComputeUnits(dev);
  // 16 channels of gate and up are a group; the last unit of the experts' rows is
  // whole (the gate/up kernel works by blocks of 128 channels).
  l.gate_up.groups = CeilDiv(d->intermediate, kUnit) * (kUnit / 16);
  l.gate_up.units = CeilDiv(d->hidden, kUnit);
  l.down.groups = CeilDiv(d->hidden, 32);
  l.down.units = CeilDiv(d->intermediate, kUnit);
  for (int t = 0; t < kMaxTokens; ++t)
    p->work[t] = std::max(mnb::moe::WorkBytes(l, t + 1), t > 0 ? p->work[t - 1] : 0);
  const size_t up = static_cast<size_t>(d->experts) * l.gate_up.groups * l.gate_up.units;
  const size_t dn = static_cast<size_t>(d->experts) * l.down.groups * l.down.units;
  const size_t rec = kRecords * kRec, meta = mnb::moe::MetaBytes(l.folds, l.zeros);
  const size_t sizes[5] = {up * rec, up * meta, dn * rec, dn * meta,
                           router ? static_cast<size_t>(d->experts) * d->hidden * sizeof(float) : 0};
  hipError_t e = hipSuccess;
  for (int i = 0; i < 5 && e == hipSuccess; ++i) {
    p->bytes += sizes[i];
    if (sizes[i] > 0) e = hipMalloc(&p->mem[i], sizes[i]);
  }
  // Host sources pass through a buffer that the largest weight fills.
  const size_t nb_h = CeilDiv(d->hidden, d->block_size), nb_i = CeilDiv(d->intermediate, d->block_size);
  const size_t rows_h = static_cast<size_t>(d->experts) * d->hidden,
               rows_i = static_cast<size_t>(d->experts) * d->intermediate;
  void *staged[3] = {nullptr, nullptr, nullptr};
  if (!device && e == hipSuccess) {
    const size_t blocks = std::max(rows_i * nb_h, rows_h * nb_i);
    e = hipMalloc(&staged[0], blocks * (d->block_size / 2));
    if (e == hipSuccess) e = hipMalloc(&staged[1], blocks * sizeof(float));
    if (e == hipSuccess && l.zeros) e = hipMalloc(&staged[2], blocks);
  }
  auto done = [&](const char *what, int status) -> int {
    for (void *m : staged)
      if (m) (void)hipFree(m);
    if (status != MNB_OK) {
      if (status == MNB_ERR_ALLOC) (void)hipGetLastError();  // the failed allocation's
      FreePlan(p);
      return Fail(what, e, status);
    }
    *out_plan = p;
    return MNB_OK;
  };
  if (e != hipSuccess) return done("hipMalloc", MNB_ERR_ALLOC);
  // The copies run on the null stream, which does not wait for non-blocking
  // streams: every write to the sources must have landed first.
  if (device) e = hipDeviceSynchronize();
  struct Part {
    const mnb_moe_weight *w;
    int64_t N, K;
    Half half;
    const mnb::moe::Matrix *m;
    int mem;
  };
  const Part parts[3] = {{gate, d->intermediate, d->hidden, Half::kGate, &l.gate_up, 0},
                         {up_w, d->intermediate, d->hidden, Half::kUp, &l.gate_up, 0},
                         {down, d->hidden, d->intermediate, Half::kPair, &l.down, 2}};
  for (const Part &part : parts) {
    mnb_moe_weight w = *part.w;
    const size_t rows = static_cast<size_t>(d->experts) * part.N;
    const size_t nb = CeilDiv(part.K, d->block_size);
    if (!device && e == hipSuccess) {
      e = hipMemcpy(staged[0], w.B, rows * nb * (d->block_size / 2), hipMemcpyHostToDevice);
      if (e == hipSuccess)
        e = hipMemcpy(staged[1], w.scales, rows * nb * sizeof(float), hipMemcpyHostToDevice);
      if (e == hipSuccess && l.zeros)
        e = hipMemcpy(staged[2], w.zero_points, rows * ((nb + 1) / 2), hipMemcpyHostToDevice);
      w.B = static_cast<const uint8_t *>(staged[0]);
      w.scales = static_cast<const float *>(staged[1]);
      w.zero_points = static_cast<const uint8_t *>(staged[2]);
    }
    if (e == hipSuccess)
      e = mnb::moe::LaunchRelayout(w, part.N, part.K, d->block_size, d->experts, part.half, *part.m,
                                   static_cast<uint8_t *>(p->mem[part.mem]),
                                   static_cast<uint8_t *>(p->mem[part.mem + 1]), nullptr);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
  }
  if (e == hipSuccess && router) {
    e = hipMemcpy(p->mem[4], router, sizes[4],
                  device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
  }
  if (e != hipSuccess) return done("expert weight layout", MNB_ERR_HIP);
  l.gate_up.rec = static_cast<const uint8_t *>(p->mem[0]);
  l.gate_up.meta = static_cast<const uint8_t *>(p->mem[1]);
  l.down.rec = static_cast<const uint8_t *>(p->mem[2]);
  l.down.meta = static_cast<const uint8_t *>(p->mem[3]);
  l.router = static_cast<const float *>(p->mem[4]);
  return done("", MNB_OK);
}

} // namespace

extern "C" {

int mnb_moe_plan_create(const mnb_moe_desc *desc, const float *router, const mnb_moe_weight *gate,
                        const mnb_moe_weight *up, const mnb_moe_weight *down,
                        mnb_moe_plan **out_plan) {
  const int st = CheckPlanInputs(desc, gate, up, down, out_plan);
  return st != MNB_OK ? st : Create(desc, router, gate, up, down, false, out_plan);
}

int mnb_moe_plan_create_device(const mnb_moe_desc *desc, const float *dRouter,
                               const mnb_moe_weight *dGate, const mnb_moe_weight *dUp,
                               const mnb_moe_weight *dDown, mnb_moe_plan **out_plan) {
  const int st = CheckPlanInputs(desc, dGate, dUp, dDown, out_plan);
  if (st != MNB_OK) return st;
  for (const mnb_moe_weight *w : {dGate, dUp, dDown})
    if (!Aligned(w->B, 4) || !Aligned(w->scales, 4)) return MNB_ERR_BAD_SHAPE;
  if (!Aligned(dRouter, 4)) return MNB_ERR_BAD_SHAPE;
  return Create(desc, dRouter, dGate, dUp, dDown, true, out_plan);
}

int mnb_moe_plan_destroy(mnb_moe_plan *plan) {
  if (plan != nullptr) FreePlan(plan);
  return MNB_OK;
}

int mnb_moe_plan_device_bytes(const mnb_moe_plan *plan, size_t *bytes) {
  if (plan == nullptr || bytes == nullptr) return MNB_ERR_NULL_POINTER;
  *bytes = plan->bytes;
  return MNB_OK;
}

int mnb_moe_workspace_bytes(const mnb_moe_plan *plan, int64_t T, int32_t x_type, size_t *bytes) {
  if (plan == nullptr || bytes == nullptr) return MNB_ERR_NULL_POINTER;
  if (!FloatType(x_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if (T < 0 || T > kMaxRun) return MNB_ERR_BAD_SHAPE;
  *bytes = T == 0 ? 0 : RunBytes(plan, T);
  return MNB_OK;
}

int mnb_moe_run(const mnb_moe_plan *plan, int64_t T, int32_t x_type, const void *dX,
                const float *dLogits, void *dY, int32_t *dIds, float *dWeights, void *dWorkspace,
                size_t workspace_bytes, void *stream) {
  if (plan == nullptr) return MNB_ERR_NULL_POINTER;
  if (!FloatType(x_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if (T < 0 || T > kMaxRun) return MNB_ERR_BAD_SHAPE;
  if (T == 0) return MNB_OK;
  const mnb::moe::Layer &l = plan->layer;
  if (dX == nullptr || dY == nullptr || (dLogits == nullptr && l.router == nullptr))
    return MNB_ERR_NULL_POINTER;
  const size_t size = x_type == MNB_TYPE_FLOAT ? 4 : 2;
  if (!Aligned(dX, size) || !Aligned(dY, size) || !Aligned(dLogits, 4) || !Aligned(dIds, 4) ||
      !Aligned(dWeights, 4) || !Aligned(dWorkspace, 16))
    return MNB_ERR_BAD_SHAPE;
  if (dWorkspace == nullptr || workspace_bytes < RunBytes(plan, T))
    return MNB_ERR_WORKSPACE;
  int cur = -1;
  if (hipGetDevice(&cur) != hipSuccess || cur != plan->device) return MNB_ERR_NO_DEVICE;
  for (int64_t t = 0; t < T; t += kMaxTokens) {
    const int n = static_cast<int>(std::min<int64_t>(kMaxTokens, T - t));
    const hipError_t e = mnb::moe::LaunchLayer(
        l, n, x_type, static_cast<const char *>(dX) + t * l.hidden * size,
        dLogits ? dLogits + t * l.experts : nullptr, static_cast<char *>(dY) + t * l.hidden * size,
        dIds ? dIds + t * l.top_k : nullptr, dWeights ? dWeights + t * l.top_k : nullptr,
        dWorkspace, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return Fail("expert layer", e, MNB_ERR_HIP);
  }
  return MNB_OK;
}

} // extern "C"

// C ABI of the 8-bit key/value cache: validation and workspace.
#include "mnb_kv.h"

namespace {

using namespace mnb::kv;

bool FloatType(int32_t t) {
  return t == MNB_TYPE_FLOAT || t == MNB_TYPE_FLOAT16 || t == MNB_TYPE_BFLOAT16;
}

bool Aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// What a call is described by, without its pointers' targets.
int CheckShape(const mnb_kv_cache *c, const mnb_kv_batch *b, Cache *cache, Batch *batch) {
  if (c == nullptr || b == nullptr) return MNB_ERR_NULL_POINTER;
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page_size) ++shift;
  if ((1 << shift) != c->page_size) return MNB_ERR_BAD_ATTRIBUTE;
  if (c->pages < 1 || c->pages > INT32_MAX || c->kv_heads < 1 || c->kv_heads > 1024 ||
      c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16 != 0)
    return MNB_ERR_BAD_SHAPE;
  if (b->sequences < 0 || b->sequences > 65535 || b->tokens < 0 ||
      b->tokens > (int64_t{1} << 24) || b->max_tokens < 0 || b->table_width < 0 ||
      b->table_width > (int64_t{1} << 30) / c->page_size)
    return MNB_ERR_BAD_SHAPE;
  if (b->starts == nullptr && b->sequences > 0 && b->tokens % b->sequences != 0)
    return MNB_ERR_BAD_SHAPE;
  *cache = Cache{{c->k, c->v},
                 {c->k_scales, c->v_scales},
                 static_cast<uint32_t>(c->pages),
                 c->kv_heads,
                 shift,
                 c->head_dim};
  const int64_t each = b->sequences > 0 ? b->tokens / b->sequences : 0;
  const int64_t most = b->starts == nullptr ? each
                       : b->max_tokens == 0 ? b->tokens
                                            : std::min(b->max_tokens, b->tokens);
  *batch = Batch{b->table,
                 b->lengths,
                 b->starts,
                 static_cast<int32_t>(b->sequences),
                 static_cast<int32_t>(b->table_width),
                 static_cast<int32_t>(b->tokens),
                 static_cast<int32_t>(each),
                 static_cast<int32_t>(most)};
  return MNB_OK;
}

int CheckPointers(const mnb_kv_cache *c, const mnb_kv_batch *b) {
  if (c->k == nullptr || c->v == nullptr || c->k_scales == nullptr || c->v_scales == nullptr ||
      b->lengths == nullptr || (b->table == nullptr && b->table_width > 0))
    return MNB_ERR_NULL_POINTER;
  if (!Aligned(c->k, 16) || !Aligned(c->v, 16) || !Aligned(c->k_scales, 4) ||
      !Aligned(c->v_scales, 4) || !Aligned(b->lengths, 4) || !Aligned(b->table, 4) ||
      !Aligned(b->starts, 4))
    return MNB_ERR_BAD_SHAPE;
  return MNB_OK;
}

int CheckRows(const mnb_kv_rows *r, int64_t dim, int32_t x_type, Rows *rows) {
  if (r == nullptr || r->x == nullptr) return MNB_ERR_NULL_POINTER;
  const int64_t each = x_type == MNB_TYPE_FLOAT ? 4 : 8, far = int64_t{1} << 36;
  if (!Aligned(r->x, 16) || r->token_stride % each != 0 || r->head_stride % each != 0 ||
      r->token_stride < dim || r->head_stride < dim || r->token_stride > far ||
      r->head_stride > far)
    return MNB_ERR_BAD_SHAPE;
  *rows = Rows{r->x, r->token_stride, r->head_stride};
  return MNB_OK;
}

int CheckHeads(const mnb_kv_cache *c, const mnb_kv_batch *b, int32_t heads) {
  if (heads < 1 || heads > (1 << 16) || heads % c->kv_heads != 0) return MNB_ERR_BAD_SHAPE;
  if (b->tokens * heads > int64_t{1} << 27) return MNB_ERR_BAD_SHAPE;  // a grid's threads
  return MNB_OK;
}

int OnDevice() {
  int dev = -1;
  const hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess) return MNB_OK;
  mnb::SetLastHipError("hipGetDevice", e);
  return MNB_ERR_NO_DEVICE;
}

int Report(const char *what, hipError_t e) {
  if (e == hipSuccess) return MNB_OK;
  mnb::SetLastHipError(what, e);
  return MNB_ERR_HIP;
}

} // namespace

extern "C" {

int mnb_kv_append(const mnb_kv_cache *cache, const mnb_kv_batch *batch, int32_t x_type,
                  const mnb_kv_rows *k, const mnb_kv_rows *v, void *stream) {
  Cache c;
  Batch b;
  Rows rows[2];
  int st = CheckShape(cache, batch, &c, &b);
  if (st != MNB_OK) return st;
  if (!FloatType(x_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if (b.sequences == 0 || b.tokens == 0 || b.width == 0) return MNB_OK;
  if ((st = CheckPointers(cache, batch)) != MNB_OK ||
      (st = CheckRows(k, c.dim, x_type, &rows[0])) != MNB_OK ||
      (st = CheckRows(v, c.dim, x_type, &rows[1])) != MNB_OK || (st = OnDevice()) != MNB_OK)
    return st;
  return Report("cache append",
                LaunchAppend(c, b, x_type, rows[0], rows[1], static_cast<hipStream_t>(stream)));
}

int mnb_kv_workspace_bytes(const mnb_kv_cache *cache, const mnb_kv_batch *batch, int32_t heads,
                           int32_t x_type, size_t *bytes) {
  Cache c;
  Batch b;
  if (bytes == nullptr) return MNB_ERR_NULL_POINTER;
  int st = CheckShape(cache, batch, &c, &b);
  if (st != MNB_OK) return st;
  if (!FloatType(x_type)) return MNB_ERR_BAD_ATTRIBUTE;
  if ((st = CheckHeads(cache, batch, heads)) != MNB_OK) return st;
  *bytes = b.sequences == 0 || b.tokens == 0 ? 0 : AttendWorkBytes(c, b, heads, x_type);
  return MNB_OK;
}

int mnb_kv_attend(const mnb_kv_cache *cache, const mnb_kv_batch *batch, int32_t heads,
                  int32_t x_type, const mnb_kv_rows *q, float scale, int64_t window, void *dY,
                  void *dWorkspace, size_t workspace_bytes, void *stream) {
  Attend a;
  int st = CheckShape(cache, batch, &a.cache, &a.batch);
  if (st != MNB_OK) return st;
  if (!FloatType(x_type) || !(scale == scale) || scale - scale != 0.0f || window < 0)
    return MNB_ERR_BAD_ATTRIBUTE;
  if ((st = CheckHeads(cache, batch, heads)) != MNB_OK) return st;
  if (a.batch.sequences == 0 || a.batch.tokens == 0) return MNB_OK;
  if ((st = CheckPointers(cache, batch)) != MNB_OK ||
      (st = CheckRows(q, a.cache.dim, x_type, &a.q)) != MNB_OK)
    return st;
  if (dY == nullptr) return MNB_ERR_NULL_POINTER;
  if (!Aligned(dY, 16) || !Aligned(dWorkspace, 16)) return MNB_ERR_BAD_SHAPE;
  const size_t need = AttendWorkBytes(a.cache, a.batch, heads, x_type);
  if (workspace_bytes < need || (dWorkspace == nullptr && need > 0)) return MNB_ERR_WORKSPACE;
  if ((st = OnDevice()) != MNB_OK) return st;
  a.q_heads = heads;
  a.scale = scale;
  a.window = window > (int64_t{1} << 30) ? 0 : static_cast<int32_t>(window);
  a.y = dY;
  return Report("cache attention",
                LaunchAttend(a, x_type, dWorkspace, static_cast<hipStream_t>(stream)));
}

} // extern "C"

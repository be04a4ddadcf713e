/*
 * mnb_kv.h -- C ABI of a paged key/value cache in 8 bits and of the attention over it.
 *
 * Keys and values are OCP e4m3 codes with one scale for each page and head: a
 * page is a block of page_size tokens of one sequence, value = code * scale.
 * A table names each sequence's pages, so that a cache is shared by sequences
 * of any length. The scales that mnb_kv_append makes are powers of two (e4m3's
 * precision does not depend on where in its range a value lies, so they lose
 * nothing, and a page whose scale grows is re-rounded exactly, but for values that become
 * subnormal); mnb_kv_attend takes any from 2^-100 to 2^100, powers of two to 2^120, and
 * 0 for a page whose codes are 0.
 *
 * It stands between the QKV projection (mnb.h, mnb_fp8.h), whose rows
 * mnb_rotary turns in place, and the output projection. ONNX's Attention-24 is
 * the unfused graph's operator, over caches in the activations' type. The
 * reference has no counterpart.
 *
 * Conventions of mnb.h hold (device pointers, void* streams, status codes,
 * checks before any HIP call).
 */
#ifndef MNB_KV_H
#define MNB_KV_H

#include "mnb.h"
#include "mnb_fp8.h" /* MNB_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

/* The cache: codes [pages, kv_heads, page_size, head_dim] and scales [pages,
 * kv_heads], of keys and of values. The codes are aligned to 16 bytes. */
typedef struct mnb_kv_cache {
  int64_t pages;      /* 1 .. 2^31 - 1 */
  int32_t kv_heads;   /* 1 .. 1024 */
  int32_t page_size;  /* 16, 32, 64, 128 or 256 */
  int32_t head_dim;   /* a multiple of 16, at most 256 */
  uint8_t *k, *v;
  float *k_scales, *v_scales;
} mnb_kv_cache;

/* The sequences of a call. The tokens of sequence b are rows starts[b] ..
 * starts[b + 1] - 1 of the call's tensors (starts NULL: tokens / sequences rows
 * each), and the last of its lengths[b] tokens: row i has position lengths[b] -
 * rows + i. A row before position 0 is no token. Page table[b][p] holds
 * positions p page_size .. (p + 1) page_size - 1.
 *
 * What the device memory holds is not checked on the host; the kernels bound it:
 * starts beyond `tokens` count as `tokens`; positions that the table does
 * not reach and pages outside the cache are neither written nor seen. Rows of no
 * sequence are left as they are. A page that two sequences append to in one call
 * has codes and a scale of either, as has one that one sequence reaches twice; any
 * number may read one. */
typedef struct mnb_kv_batch {
  int64_t sequences;    /* 0 .. 65535 */
  int64_t tokens;       /* rows of the call's tensors, at most 2^24 */
  int64_t max_tokens;   /* no sequence has more rows; 0: tokens, or tokens / sequences */
  int64_t table_width;  /* pages of a table row; times page_size at most 2^30 */
  const int32_t *table;   /* [sequences, table_width] */
  const int32_t *lengths; /* [sequences]: tokens with this call's; below 0 counts as 0 */
  const int32_t *starts;  /* [sequences + 1], not falling, or NULL */
} mnb_kv_batch;

/* Rows of heads: value (t, h, d) at t * token_stride + h * head_stride + d of
 * MNB_TYPE_FLOAT, _FLOAT16 or _BFLOAT16, aligned to 16 bytes as both strides are. */
typedef struct mnb_kv_rows {
  const void *x;
  int64_t token_stride, head_stride;
} mnb_kv_rows;

/* Writes the call's keys and values [tokens, kv_heads, head_dim], both of x_type.
 * A page's scale is the least power of two, 2^-64 at least, that brings the
 * largest magnitude of its tokens to 448 or below, with s the scale that it had: a page
 * that begins with a new token starts anew, one that is continued takes no less
 * than s, power of two or not, and if it takes more its codes are re-rounded, code * s /
 * scale. Codes are x / scale in fp32 (exact for powers of two) rounded to nearest, ties to
 * even. Infinities and NaN become NaN codes and do not count for the scale. Runs on the
 * current device, asynchronous on `stream`. */
int mnb_kv_append(const mnb_kv_cache *cache, const mnb_kv_batch *batch, int32_t x_type,
                  const mnb_kv_rows *k, const mnb_kv_rows *v, void *stream);

/* Workspace (16-byte aligned) of a call of mnb_kv_attend: the parts of rows whose
 * keys are shared out over workgroups. */
int mnb_kv_workspace_bytes(const mnb_kv_cache *cache, const mnb_kv_batch *batch, int32_t heads,
                           int32_t x_type, size_t *bytes);

/* Y [tokens, heads, head_dim], dense, of Q's type, aligned to 16 bytes, overlapping
 * nothing else: for row i of sequence b at position p and query head h (tokens *
 * heads at most 2^27), the softmax over the keys t <= p (and t > p - window, where
 * window > 0; beyond 2^30 it counts as 0) of scale * q . k_t, times v; heads is a
 * multiple of kv_heads, and query heads h use cache head h / (heads / kv_heads). A row
 * that sees no key, or only scores of -inf, is 0; unseen keys and values leave no trace,
 * NaN and infinities among them, in their scales too. Products are exact for fp16 q, up to
 * 2^-31 of q's largest magnitude for bf16 and up to 2^-22 for fp32; the weights have 22 bits
 * for an fp32 or fp16 Y and 11 for a bf16 one; sums are fp32. The value scales of one head and
 * sequence lie within 2^100 of each other. Runs on the current device, asynchronous on `stream`. */
int mnb_kv_attend(const mnb_kv_cache *cache, const mnb_kv_batch *batch, int32_t heads,
                  int32_t x_type, const mnb_kv_rows *q, float scale, int64_t window, void *dY,
                  void *dWorkspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MNB_KV_H */

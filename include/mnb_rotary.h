/*
 * mnb_rotary.h -- C ABI of rotary positions with several axes.
 *
 *   pair j of a head (j < rotary_dim / 2), (a, b), becomes
 *   (a cos t - b sin t, b cos t + a sin t),   t = positions[axis[j]][token] * f_j
 *
 * The pairs are (x[j], x[j + rotary_dim / 2]) or, interleaved, (x[2j], x[2j + 1]);
 * values of a head from rotary_dim on are kept. One axis is the usual position
 * in a text; images and videos have a time, a row and a column. Queries and
 * keys are rotated by one launch, from and to rows of any stride, as the views
 * of a QKV projection's result are. With the key cache of mnb_kv.h behind it, it
 * stands between MatMulNBits or the 8-bit product and the attention. The ONNX
 * operator of one axis is RotaryEmbedding-23, which takes cos and sin as inputs.
 * The reference has no counterpart.
 *
 * A frequency is given in turns: f_j / (2 pi) modulo 1, in units of 2^-64. A
 * position times it is the angle modulo a turn with no rounding, for any 64-bit
 * position. What is rounded is the frequency, by 2^-65 of a turn at most, which moves the
 * angle of position p by 2^-65 |p| turns: less than fp32 results show up to |p| = 2^38,
 * where fp32 angles lose a bit with each doubling from 1 on. cos and sin are off by less
 * than 2^-23.
 *
 * Conventions of mnb.h hold (device pointers, void* streams, status codes,
 * checks before any HIP call).
 */
#ifndef MNB_ROTARY_H
#define MNB_ROTARY_H

#include "mnb.h"
#include "mnb_fp8.h" /* MNB_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

/* Position types, by their ONNX TensorProto codes. */
#define MNB_TYPE_INT32 6
#define MNB_TYPE_INT64 7

#define MNB_ROTARY_MAX_PAIRS 256
#define MNB_ROTARY_MAX_AXES 8

typedef struct mnb_rotary_desc {
  int32_t head_dim;     /* values of a head, at most 4096 */
  int32_t rotary_dim;   /* even, 2 .. min(head_dim, 2 MNB_ROTARY_MAX_PAIRS) */
  int32_t axes;         /* 1 .. MNB_ROTARY_MAX_AXES */
  int32_t interleaved;  /* 0 or 1 */
  const uint64_t *turns; /* host memory: rotary_dim / 2 frequencies */
  const uint8_t *axis;   /* host memory: each frequency's axis, below axes */
} mnb_rotary_desc;

/* Heads of one input and its result, all of one type: value (t, h, d) lies at
 * t * token_stride + h * head_stride + d; strides in values, head_dim at least. */
typedef struct mnb_rotary_heads {
  int32_t heads;       /* 0 .. 2^16: 0 leaves this part out */
  const void *x;
  int64_t x_token_stride, x_head_stride;
  void *y;             /* may be x, with x's strides */
  int64_t y_token_stride, y_head_stride;
} mnb_rotary_heads;

/* T tokens; positions: [axes][T] of pos_type, axis_stride positions between
 * axes. query and key: the two parts, key NULL for none. A result overlaps
 * nothing but, if it is that exactly, its own input. T == 0 is a no-op; T <= 2^24.
 * Runs on the current device, asynchronous on `stream`. */
int mnb_rotary(const mnb_rotary_desc *desc, int64_t T, int32_t pos_type, const void *positions,
               int64_t axis_stride, int32_t x_type, const mnb_rotary_heads *query,
               const mnb_rotary_heads *key, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MNB_ROTARY_H */

/*
 * mnb_norm.h -- C ABI of the RMS norm with the residual's addition, to 8 bits or not.
 *
 *   h = X + R, rounded to X's type     (h = X without a residual)
 *   y = h / sqrt(mean(h^2) + epsilon) * gamma        (over a row)
 *   Y = y rounded to X's type, or e4m3 codes with a scale for each row's block
 *       of 128: with amax the block's largest |y|, at least 2^-100, amax / 448
 *       and the code nearest to 448 y / amax, y not rounded before
 *
 * The unfused graph is an Add and an ONNX RMSNormalization-23 over the last
 * axis; mnb_run_rmsnorm (mnb.h) fuses the norm into a 4-bit projection, this
 * makes the input of an 8-bit one (mnb_fp8_run) or of a layer of experts
 * (mnb_moe_run). The reference has no counterpart.
 *
 * Conventions of mnb.h hold (device pointers, void* streams, status codes,
 * checks before any HIP call).
 */
#ifndef MNB_NORM_H
#define MNB_NORM_H

#include "mnb.h"
#include "mnb_fp8.h" /* MNB_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

/* dX: M rows of K values of x_type (MNB_TYPE_FLOAT, _FLOAT16 or _BFLOAT16), ldx
 * values apart; dResidual: the same, ldr apart, or NULL; dGamma: fp32 [K].
 * y_type x_type: dY [M, K] of it, dScales NULL. y_type MNB_TYPE_FLOAT8E4M3FN: dY
 * uint8 [M, K], dScales fp32 [M, ceil(K / 128)]. dSum: [M, K] of x_type, receives
 * h where there is a residual (it may be dX or dResidual, if that is dense),
 * NULL without one; dY and dScales overlap nothing else.
 * The squares are added up in fp32, wavefronts' sums and the root in fp64: magnitudes beyond
 * 2^63 give 0, as they do in the unfused graph. A row with an infinity or a NaN has NaN
 * there and spoils no other. epsilon >= 0; K <= 2^22, M <= 2^30. Runs on the current
 * device; M == 0 is a no-op. Asynchronous on `stream`. */
int mnb_rms_norm(int64_t M, int64_t K, int32_t x_type, const void *dX, int64_t ldx,
                 const void *dResidual, int64_t ldr, const float *dGamma, float epsilon,
                 int32_t y_type, void *dY, float *dScales, void *dSum, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MNB_NORM_H */

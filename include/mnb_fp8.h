/*
 * mnb_fp8.h -- C ABI of the 8-bit floating-point product with block scales.
 *
 *   Y[m][n] = sum_b a_scale[m][b] * w_scale[n / 128][b]
 *             * sum_{k in block b} a[m][k] * w[n][k],   b = k / 128
 *
 * a and w are OCP e4m3 codes (no infinities, 0x7F and 0xFF are NaN, largest
 * 448), a with one fp32 scale for each row's block of 128 values along K, w
 * with one for each block of 128 x 128. The last block of K and of N may be
 * shorter. It stands beside the 4-bit MatMulNBits of mnb.h (the same weight
 * layout [N, K], prepared plan, status codes and rules on streams and
 * workspaces); no ONNX operator has this contract, so it is not in the node
 * registration table. The reference has no counterpart. A block's two scales are
 * multiplied in fp32 first, so their product has to be in fp32's range.
 *
 * Conventions of mnb.h hold: device pointers on the plan's device, streams as
 * void* (NULL = the default stream), every entry point returns an mnb_status,
 * arguments are checked before any HIP call. A plan is immutable after its
 * creation; runs on distinct outputs and workspaces may overlap.
 */
#ifndef MNB_FP8_H
#define MNB_FP8_H

#include "mnb.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Value types, by their ONNX TensorProto codes. */
#define MNB_TYPE_FLOAT 1
#define MNB_TYPE_FLOAT16 10
#define MNB_TYPE_BFLOAT16 16
#define MNB_TYPE_FLOAT8E4M3FN 17

/* Values of K covered by one scale. */
#define MNB_FP8_BLOCK 128

typedef struct mnb_fp8_plan mnb_fp8_plan;

/* Rows to e4m3, one scale for each row's block of 128: with amax the block's
 * largest magnitude, at least 2^-100,
 *   scale = amax / 448,   code = 448 * x / amax rounded to e4m3, ties to even
 * (the quotient correctly rounded to fp32 first). An infinity in a block gives
 * it the scale inf, its infinities NaN and its finite values 0; a NaN gives
 * scale and codes NaN: either way the block stands for NaN.
 * dX: M rows of K values of x_type (MNB_TYPE_FLOAT, _FLOAT16 or _BFLOAT16), ldx
 * values apart (ldx >= K); dQ: uint8 [M, K]; dScales: fp32 [M, ceil(K / 128)].
 * Runs on the current device; M == 0 is a no-op. */
int mnb_fp8_quantize(int64_t M, int64_t K, int32_t x_type, const void *dX, int64_t ldx,
                     uint8_t *dQ, float *dScales, void *stream);

/* Prepared weight: W uint8 (e4m3) [N, K] and scales fp32 [ceil(N / 128),
 * ceil(K / 128)], from host memory or from the current device's. The plan
 * keeps re-laid copies of its own (N rounded up to 64, K to 128), so the
 * sources may go afterwards. mnb_fp8_plan_create_device first waits for all
 * work already issued on the device. Not during the capture of a stream.
 * K <= 2^22, N <= 2^26. */
int mnb_fp8_plan_create(int64_t K, int64_t N, const uint8_t *W, const float *scales,
                        mnb_fp8_plan **out_plan);
int mnb_fp8_plan_create_device(int64_t K, int64_t N, const uint8_t *dW, const float *dScales,
                               mnb_fp8_plan **out_plan);
int mnb_fp8_plan_destroy(mnb_fp8_plan *plan);
int mnb_fp8_plan_device_bytes(const mnb_fp8_plan *plan, size_t *bytes);

/* Device workspace (16-byte aligned) that mnb_fp8_run needs for M rows of
 * a_type: the rows' codes and scales where the run makes them (a_type not
 * MNB_TYPE_FLOAT8E4M3FN), a copy of the codes whose rows are multiples of 128
 * bytes where K is not, and the partial sums where K is split over workgroups. */
int mnb_fp8_workspace_bytes(const mnb_fp8_plan *plan, int64_t M, int32_t a_type, size_t *bytes);

/* Y[M, N] of y_type (MNB_TYPE_FLOAT, _FLOAT16 or _BFLOAT16; sums in fp32,
 * rounded once; for _FLOAT and _FLOAT16 of exact products; for _BFLOAT16 a product
 * is cut off 2^-13 below the largest of its group of eight along K, so that Y loses
 * up to 7 2^-13 of the sum of the products' magnitudes: about 1.4e-5 of Y where they
 * are of one size, all of a small product beside a large one) from dense rows dA [M, K]
 * of a_type: MNB_TYPE_FLOAT8E4M3FN codes with dAScales [M, ceil(K / 128)], or
 * values of another type with dAScales NULL, quantized as by mnb_fp8_quantize.
 * dA, dY and the workspace are aligned to 16 bytes (MNB_ERR_BAD_SHAPE otherwise);
 * dY and the workspace overlap nothing else. M == 0 is a no-op; M <= 2^30 and
 * M * N <= 2^36. Asynchronous on `stream`. */
int mnb_fp8_run(const mnb_fp8_plan *plan, int64_t M, int32_t a_type, const void *dA,
                const float *dAScales, int32_t y_type, void *dY, void *dWorkspace,
                size_t workspace_bytes, void *stream);

/* Name of the kernel that multiplies M rows into a bfloat16 Y ("" for a bad plan or
 * M == 0). */
const char *mnb_fp8_kernel_name(const mnb_fp8_plan *plan, int64_t M);

#ifdef __cplusplus
}
#endif

#endif /* MNB_FP8_H */

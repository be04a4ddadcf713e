/*
 * mnb_moe.h -- C ABI of a whole mixture-of-experts layer on 4-bit weights.
 *
 *   logits[t] = X[t] R^T                              (sums in 64 bits)
 *   chosen    = the top_k largest logits of t, ties to the lowest expert
 *   p         = softmax over the chosen logits (normalize), else over all
 *   Y[t]      = sum over the chosen e of
 *               p_e * (silu(X[t] Wg_e^T) (*) (X[t] Wu_e^T)) Wd_e^T
 *
 * Each expert's gate, up and down weights are MatMulNBits weights (mnb.h: B,
 * scales, optional zero points) with the experts as their first axis. The
 * unfused graph is a MatMul, a TopK, a Softmax and, for each token and chosen
 * expert, three MatMulNBits nodes and the activation between them. It stands
 * beside mnb_plan_create_gate_up's fusion of a dense layer; the contract is no
 * ONNX operator's, so it is not in the node registration table. The reference
 * has no counterpart.
 *
 * Meant for few tokens (a decode batch): the weights of the experts that are
 * met are read once for every 64 tokens. More tokens are taken 64 at a time.
 *
 * Activations enter the products in fixed point: each token's (or expert
 * row's) block of 128 values is scaled by a power of two and rounded to 22 bits
 * below its largest magnitude (at most 2^-22 of that, or of 2^-90 where that is
 * larger), the 4-bit weights are exact integers, and each weight block's sum is exact
 * before it is scaled and added up in fp32. A block that holds an infinity or a NaN
 * makes the token's products NaN.
 *
 * Conventions of mnb.h hold (device pointers, void* streams, status codes,
 * checks before any HIP call, immutable plans, runs on distinct outputs and
 * workspaces may overlap).
 */
#ifndef MNB_MOE_H
#define MNB_MOE_H

#include "mnb.h"
#include "mnb_fp8.h" /* MNB_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mnb_moe_desc {
  int64_t hidden;           /* width of X and Y, at most 2^18 */
  int64_t intermediate;     /* an expert's width, at most 2^18; the two multiplied at most 2^34 */
  int32_t experts;          /* 1 .. 1024 */
  int32_t top_k;            /* 1 .. min(experts, 32) */
  int32_t bits;             /* 4 only */
  int32_t block_size;       /* power of two >= 16, of all three weights */
  int32_t normalize;        /* 1: p over the chosen experts, 0: over all */
  int32_t has_zero_points;  /* all three weights have zero points, or none */
} mnb_moe_desc;

/* One weight of all experts: B uint8 [experts, N, nb, block_size / 2], scales
 * fp32 [experts, N, nb], zero_points uint8 [experts, N, ceil(nb / 2)] or NULL;
 * gate and up: N = intermediate, K = hidden; down the other way round. */
typedef struct mnb_moe_weight {
  const uint8_t *B;
  const float *scales;
  const uint8_t *zero_points;
} mnb_moe_weight;

typedef struct mnb_moe_plan mnb_moe_plan;

/* Prepared layer from host memory, or from the current device's (after
 * waiting for all work already issued on it). The plan keeps re-laid copies
 * of its own, so the sources may go afterwards. router: fp32 [experts,
 * hidden], or NULL for a plan whose runs are given the logits. Not during the
 * capture of a stream. */
int mnb_moe_plan_create(const mnb_moe_desc *desc, const float *router, const mnb_moe_weight *gate,
                        const mnb_moe_weight *up, const mnb_moe_weight *down,
                        mnb_moe_plan **out_plan);
int mnb_moe_plan_create_device(const mnb_moe_desc *desc, const float *dRouter,
                               const mnb_moe_weight *dGate, const mnb_moe_weight *dUp,
                               const mnb_moe_weight *dDown, mnb_moe_plan **out_plan);
int mnb_moe_plan_destroy(mnb_moe_plan *plan);
int mnb_moe_plan_device_bytes(const mnb_moe_plan *plan, size_t *bytes);

/* Device workspace (16-byte aligned) of a run of T tokens: their values in
 * fixed point, the logits and the choice, the chosen experts' rows. It is
 * enough for any smaller T too. */
int mnb_moe_workspace_bytes(const mnb_moe_plan *plan, int64_t T, int32_t x_type, size_t *bytes);

/* Y [T, hidden] of X [T, hidden], both of x_type (MNB_TYPE_FLOAT, _FLOAT16 or
 * _BFLOAT16; Y is rounded once). dLogits: fp32 [T, experts] to choose by in the
 * router's place, NULL to take the router's (MNB_ERR_NULL_POINTER where the
 * plan has none). A NaN logit counts as -inf. dIds (int32 [T, top_k]) and
 * dWeights (fp32 [T, top_k]) receive the choice, largest logit first, and p;
 * either may be NULL. What a run writes overlaps nothing else. T == 0 is a no-op;
 * T <= 2^24. Asynchronous on `stream`. */
int mnb_moe_run(const mnb_moe_plan *plan, int64_t T, int32_t x_type, const void *dX,
                const float *dLogits, void *dY, int32_t *dIds, float *dWeights, void *dWorkspace,
                size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MNB_MOE_H */

// Internal launch interface of the mixture-of-experts layer (mnb_moe*.hip).
#pragma once

#include "mnb_kernels.h"
#include "../../include/mnb_moe.h"

namespace mnb {
namespace moe {

// Values of K in one unit of the weight layout and of the fixed-point
// activations, and the tokens of one launch.
constexpr int kUnit = 128;
constexpr int kMaxTokens = 64;
constexpr int kMaxTopK = 32;
constexpr int kMaxExperts = 1024;
constexpr int kRec = 1024;

// Weight layout: groups of 16 rows x units of 128 values of K; R records of
// 1 KiB each (R = 2: gate and up rows of the same 16 channels, R = 1: down). A
// record holds 16 bytes per lane: lane l is row l % 16 and, with q = l / 16,
// its word w the eight nibbles k = 32 w + 8 q + 0..7: the first four in the low
// halves of the word's bytes, the others in the high ones, each the two's
// complement of (nibble - 8), so that a mask leaves 16 (nibble - 8) in a byte.
// Scales: fp32 [4 q][folds][4] per record, the rows 4 q .. 4 q + 3 that the MFMA
// leaves in lane group q; zero points likewise as int8 (zp - 8). folds =
// max(1, 128 / block_size) weight blocks of a unit. Rows and values past the
// ends are zero with zero scales.
struct Matrix {
  const uint8_t *rec;
  const float *scales;
  const int8_t *zeros;  // nullptr without zero points
  int64_t groups;       // of 16 rows
  int64_t units;
};

struct Layer {
  Matrix gate_up, down;
  const float *router;  // [experts][hidden] or nullptr
  int64_t hidden, intermediate;
  int experts, top_k, block_size, folds;
  bool normalize, zeros;
  int num_cus;
};

// Fills record r of R of every row group from MatMulNBits weights of `experts`
// matrices [N, K] (device pointers).
hipError_t LaunchRelayout(const mnb_moe_weight &src, int64_t N, int64_t K, int block_size,
                          int experts, int r, int R, uint8_t *rec, float *scales, int8_t *zeros,
                          hipStream_t s);

// Bytes of the workspace of one launch of T <= kMaxTokens tokens.
size_t WorkBytes(const Layer &l, int T, int32_t x_type);
hipError_t LaunchLayer(const Layer &l, int T, int32_t x_type, const void *X, const float *logits,
                       void *Y, int32_t *ids, float *weights, void *work, hipStream_t s);

constexpr int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

} // namespace moe
} // namespace mnb

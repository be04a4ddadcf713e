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

// Weight layout: groups of 32 rows x units of 128 values of K, two records of 1 KiB
// each (16 gate and 16 up rows of the same channels, or 32 rows of down). A
// record holds 16 bytes per lane: lane l is row l % 16 and, with q = l / 16, its
// word w the eight nibbles k = 32 w + 8 q + 0..7, the first four in the low
// halves of the word's bytes, the others in the high ones. With zero points the
// nibbles are as they come, without they are the two's complement of nibble - 8.
// A unit's meta bytes: its records' scales, fp32 [2][4 q][folds][4] (rows 4 q ..
// 4 q + 3 are what the MFMA leaves in lane group q), then the zero points, uint8
// [2][16][folds]; folds = max(1, 128 / block_size) weight blocks of a unit. Rows
// past the end have zero scales; values past K meet zero activations.
constexpr int kRecords = 2;
constexpr int MetaBytes(int folds, bool zeros) { return kRecords * 16 * folds * (zeros ? 5 : 4); }

struct Matrix {
  const uint8_t *rec, *meta;
  int64_t groups;  // of 32 rows
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

// Which record of its unit a group of 16 rows fills: the first or second half of
// a pair of groups (down), or always the same one (0: gate, 1: up).
enum class Half { kPair = -1, kGate = 0, kUp = 1 };

// Fills those records of m from MatMulNBits weights of `experts` matrices [N, K]
// (device pointers).
hipError_t LaunchRelayout(const mnb_moe_weight &src, int64_t N, int64_t K, int block_size,
                          int experts, Half half, const Matrix &m, uint8_t *rec, uint8_t *meta,
                          hipStream_t s);

// Bytes of the workspace of one launch of T <= kMaxTokens tokens.
size_t WorkBytes(const Layer &l, int T);
hipError_t LaunchLayer(const Layer &l, int T, int32_t x_type, const void *X, const float *logits,
                       void *Y, int32_t *ids, float *weights, void *work, hipStream_t s);

constexpr int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

} // namespace moe
} // namespace mnb

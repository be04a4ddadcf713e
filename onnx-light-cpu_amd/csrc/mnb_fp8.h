// Internal launch interface of the 8-bit product (mnb_fp8*.hip).
#pragma once

#include "mnb_kernels.h"
#include "../../include/mnb_fp8.h"

#include <algorithm>

namespace mnb {
namespace fp8 {

// Weight layout: groups of 64 rows x blocks of 128 values of K, each eight
// records of 1 KiB: fragment j (0..3) of 16 rows, half h (0..1) of 64 values.
// A record holds 16 bytes per lane: lane l row 64 G + 16 (r / 4) + 4 j + r % 4
// with r = l % 16, bytes 128 b + 64 h + 16 (l / 16) .. + 15. A lane's four
// results of fragment j are rows 4 (l / 16) .. + 3 of it (MFMA's result
// layout), so that the four fragments leave it 16 consecutive columns of Y.
// Rows past N and values past K are zero.
constexpr int kBlock = MNB_FP8_BLOCK;
constexpr int kRec = 1024;

struct Weight {
  const uint8_t *W;      // records [groups][nb][4][2][kRec]
  const float *scales;   // [ceil(N / 128)][nb]
  int64_t K, N, nb, groups;
  int num_cus;
};

// s_waitcnt vmcnt(N) lgkmcnt(0), nothing moved across: all but the newest N of this
// wavefront's copies are in LDS.
template <int N>
__device__ __forceinline__ void WaitCopies() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  __builtin_amdgcn_sched_barrier(0);
  __asm__ volatile("" ::: "memory");
}

// The same and a workgroup barrier.
template <int N>
__device__ __forceinline__ void WaitBarrier() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  __asm__ volatile("" ::: "memory");
}

inline int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Re-lays dW [N, K] into the records of w.
hipError_t LaunchRelayout(const uint8_t *dW, const Weight &w, uint8_t *records, hipStream_t s);

// x_type rows (ldx apart) -> codes in rows of ldq bytes, zero from K to ldq
// (ldq == K, or nb * 128), and scales [M, nb].
hipError_t LaunchQuantize(int64_t M, int64_t K, int32_t x_type, const void *X, int64_t ldx,
                          uint8_t *Q, int64_t ldq, float *scales, hipStream_t s);

// Code rows [M, K] into rows of nb * 128 bytes, zero past K.
hipError_t LaunchPad(int64_t M, int64_t K, const uint8_t *A, uint8_t *P, hipStream_t s);

// Y = product; A: code rows lda bytes apart, lda a multiple of 128, 16-byte
// aligned; sa [M, nb]. M >= 1. work: WorkBytes(w, M).
hipError_t LaunchProduct(const Weight &w, int64_t M, const uint8_t *A, int64_t lda,
                         const float *sa, int32_t y_type, void *Y, void *work, hipStream_t s);
size_t WorkBytes(const Weight &w, int64_t M);
const char *ProductKernelName(const Weight &w, int64_t M);

} // namespace fp8
} // namespace mnb

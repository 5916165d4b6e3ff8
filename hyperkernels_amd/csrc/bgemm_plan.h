// bgemm_plan.h - how a BF16 product runs, for the entry points with an epilogue of their own (bgemm.hip,
// bgemm_act.hip).
#pragma once

#include "hk_host.h"

namespace hk {

// What the rows of a product's matrices are, as the kernels see them.
enum class GemmRows {
  kAligned,  // whole 16-byte vectors: 8-element multiples for every contiguous extent, leading
             // dimension and batch stride, 16-byte aligned bases
  kRaggedC,  // A and B like that, C at any 2-byte address and any N
  kRagged,   // any 2-byte address, any extent
  kNone      // no MFMA path: no k, a leading dimension whose per-lane 32-bit byte offsets do not
             // fit, or one under 8 (a vector could leave the matrix); more batches of unaligned
             // rows than the tiles' grid takes
};
// a16, b16, c16: 16-byte aligned bases.
GemmRows bgemm_rows(bool ta, bool tb, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                    int64_t sA, int64_t sB, int64_t sC, int batch, bool a16, bool b16, bool c16);
// The library's choice for rows that are not kNone; one k split where may_split is false.
GemmPlan bgemm_rows_plan(bool ta, bool tb, int M, int N, int K, int batch, GemmRows rows,
                         bool may_split);
// Splits of a plan with several: fp32 partials [split][batch][M][part_pitch(N)].
size_t bgemm_partial_bytes(int used, int M, int N, int batch);
hipError_t bgemm_write_partials(bool ta, bool tb, int M, int N, int K, const hk_bf16* A, int64_t lda,
                                int64_t sA, const hk_bf16* B, int64_t ldb, int64_t sB, int batch,
                                const GemmPlan& plan, float* part, hipStream_t stream);

}  // namespace hk

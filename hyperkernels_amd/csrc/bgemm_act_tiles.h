// bgemm_act_tiles.h - the GEMM tiles with the epilogue of bgemm_act.h, each family compiled in a file of its own
// (bgemm_act_flex.hip, bgemm_act_ragged.hip, bgemm_act_wide.hip).
#pragma once

#include "bgemm_act.h"
#include "bgemm_flex_kernel.h"

namespace hk {
namespace gemm {

// The small and any-alignment tiles: tile shape `tile` of bgemm_flex_plan.
hipError_t act_flex_run(int tile, bool ta, bool tb, const FlexArgs<ActEpi>& g, int batch,
                        hipStream_t stream);
// The rows of C that a wave of such a tile writes: as many share a row of column sums.
int act_flex_wave_rows(int tile);
typedef hipError_t (*ActFlexRun)(bool, bool, const FlexArgs<ActEpi>&, int, hipStream_t);
ActFlexRun act_ragged(int tile);  // the shapes for rows of any alignment, NULL for another

// The 256-wide tiles, one k split.
hipError_t act_wide_run(bool ta, bool tb, int batch, hipStream_t stream, int M, int N, int K,
                        const ActEpi& ep, const uint16_t* A, int64_t lda, int64_t sA,
                        const uint16_t* B, int64_t ldb, int64_t sB, uint16_t* C, int64_t ldc,
                        int64_t sC);

}  // namespace gemm
}  // namespace hk

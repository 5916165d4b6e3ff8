// bgemm_act_wide.hip - the 256-wide BF16 GEMM tiles with the epilogue of bgemm_act.h.
#include "bgemm_act_tiles.h"
#include "bgemm_wide.h"

namespace hk {
namespace gemm {

hipError_t act_wide_run(bool ta, bool tb, int batch, hipStream_t stream, int M, int N, int K,
                        const ActEpi& ep, const uint16_t* A, int64_t lda, int64_t sA,
                        const uint16_t* B, int64_t ldb, int64_t sB, uint16_t* C, int64_t ldc,
                        int64_t sC) {
  return run_regions<false>(ta, tb, batch, stream, M, N, K, ep, A, lda, sA, B, ldb, sB, C, ldc, sC, 1,
                            K, nullptr, F32Out{});
}

}  // namespace gemm
}  // namespace hk

// bgemm_act_ragged.hip - the BF16 GEMM tiles for rows of any alignment with the epilogue of bgemm_act.h.
#include "bgemm_act_tiles.h"

namespace hk {
namespace gemm {

namespace {
template <class T, bool RAGGED>
constexpr ActFlexRun shape() {
  if constexpr (RAGGED == true) return &flex_layouts<T, RAGGED, ActEpi>;
  else return nullptr;
}
const ActFlexRun kShapes[] = {
#define HK_SHAPE(bm, bn, ragged, alone, shared, per_cu, fixed, tile) shape<tile, ragged>(),
    HK_FLEX_SHAPES(HK_SHAPE)
#undef HK_SHAPE
};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);
}  // namespace

ActFlexRun act_ragged(int tile) { return tile >= 1 && tile <= kNumShapes ? kShapes[tile - 1] : nullptr; }

}  // namespace gemm
}  // namespace hk

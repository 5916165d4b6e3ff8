// bgemm_act_flex.hip - the small BF16 GEMM tiles for aligned rows with the epilogue of bgemm_act.h.
#include "bgemm_act_tiles.h"

namespace hk {
namespace gemm {

namespace {
template <class T, bool RAGGED>
constexpr ActFlexRun shape() {
  if constexpr (RAGGED == false) return &flex_layouts<T, RAGGED, ActEpi>;
  else return nullptr;
}
const ActFlexRun kShapes[] = {
#define HK_SHAPE(bm, bn, ragged, alone, shared, per_cu, fixed, tile) shape<tile, ragged>(),
    HK_FLEX_SHAPES(HK_SHAPE)
#undef HK_SHAPE
};
const int kWaveRows[] = {
#define HK_SHAPE(bm, bn, ragged, alone, shared, per_cu, fixed, tile) tile::kShareM,
    HK_FLEX_SHAPES(HK_SHAPE)
#undef HK_SHAPE
};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);
}  // namespace

int act_flex_wave_rows(int tile) {
  return tile >= 1 && tile <= kNumShapes ? kWaveRows[tile - 1] : 0;
}

hipError_t act_flex_run(int tile, bool ta, bool tb, const FlexArgs<ActEpi>& g, int batch,
                        hipStream_t stream) {
  HK_CHECK_ARG(tile >= 1 && tile <= kNumShapes);
  const ActFlexRun run = kShapes[tile - 1] ? kShapes[tile - 1] : act_ragged(tile);
  HK_CHECK_ARG(run != nullptr);
  return run(ta, tb, g, batch, stream);
}

}  // namespace gemm
}  // namespace hk

// bgemm_flex.hip - the BF16 GEMM on small tiles and on operands of any alignment: the products that
// the 256-wide tiles of bgemm.hip leave most CUs idle on, and those whose rows are not whole
// 16-byte vectors (an odd vocabulary, an odd sequence length). Same contract: C = alpha * op(A)
// op(B) + beta * C (or + beta * bias), bf16 operands, fp32 accumulation, one rounding to bf16, all
// four transpose layouts, the k order of the sums fixed (deterministic).
//
// Design (gfx950): the LDS layout, MFMA operand order and epilogue of bgemm_tile.h on output tiles
// of BMT x BNT. Each wave owns kWaveM x kWaveN of the tile in 32 x 32 MFMA blocks. KG groups of
// waves share one output tile and take alternate k-tiles, each with an LDS ring of its own; their
// sums are added in group order through LDS before the epilogue. KG > 1 shortens the serial chain
// of k-tiles (copy, barrier, multiply), which bounds a product of few output tiles.
// Two ways for the operands to reach LDS:
//   - direct (16-byte aligned rows): global -> LDS copies that bypass registers, a ring of S
//     k-tiles, tile kt + S copied while tile kt + 1 .. kt + S - 1 wait or land;
//   - staged (RAGGED): 16-byte loads at any 2-byte address into registers (gfx950 serves
//     unaligned vector loads at 80% of the aligned rate when the rows sit in cache and 92% from
//     HBM: 6.7 against 8.4 TB/s and 5.8 against 6.3 TB/s), written to a ring of two LDS slots one
//     k-tile after they were issued.
// The last k-tile of a staged operand reads element by element where a vector would cross the end
// of K or of the matrix, and fills zeros past K.
#include "bgemm_flex_kernel.h"

namespace {

using namespace hk::gemm;

// The tile shapes, with what each costs: us per k-tile of one workgroup on a mostly idle device
// (alone), of each of those that share a CU of a busy one (shared), how many a CU holds, and the
// fixed time of a launch (fill, epilogue). A product of few tiles is bound by the serial chain of
// its k-tiles, which k groups shorten; one of many by the CU's copies and LDS reads per multiply,
// which fall with the tile's area. Fitted to back-to-back launches of random shapes on MI355X,
// where the plan's time came within 2% (aligned rows) and 4% (ragged) of the best shape and split
// of each. Times (us) on the 256-wide tiles, finalize included, and here:
//   512 x 2304 x 768 NN   22.0   8.2        2048^3 NN              39.9  21.8
//   512 x 768 x 2304 NT   22.0   9.9        1024 x 4096 x 4096 TN  54.0  37.8
//   768 x 2304 x 512 TN   10.3   6.9        64 x 256 x 192 NT       7.2   4.1
// Rows of odd length ran at about 2 TFLOP/s on the fallback kernel; here 50257 x 768 x 2048 TN takes
// 187 us (845 TFLOP/s) and 2048 x 768 x 50257 NN in 10 splits 190 us (833).
struct Shape {
  int bm, bn;
  bool ragged;
  double alone, shared;
  int per_cu;
  double fixed;
  hipError_t (*run)(bool, bool, const FlexArgs<Epi>&, int, hipStream_t);
};
const Shape kShapes[] = {
#define HK_SHAPE(bm, bn, ragged, alone, shared, per_cu, fixed, tile) \
  {bm, bn, ragged, alone, shared, per_cu, fixed, &flex_layouts<tile, ragged, Epi>},
    HK_FLEX_SHAPES(HK_SHAPE)
#undef HK_SHAPE
};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);

}  // namespace

namespace hk {

FlexPlan bgemm_flex_plan(int M, int N, int K, int batch, int split_k, bool ragged) {
  const int64_t cus = device_cu_count(), ktiles = ceil_div(K, BK);
  FlexPlan best{0, 1, K, 0.0};
  // A further round of workgroups on the CUs: its fill and the stores of its outputs. At 1.5 us the
  // aligned shapes were taken over the 256-wide tiles for large outputs of few k, up to twice as slow
  // (5208 x 6880 x 80: 43.4 us against 28.3); at 3.0 us, over 333 random products of 64 to 13,000
  // rows and columns and 8 to 6,000 k, 5 are more than 5% slower than those tiles (at most 16%)
  // where 33 were.
  const double round = ragged ? 1.5 : 3.0;
  for (int i = 0; i < kNumShapes; ++i) {
    const Shape& s = kShapes[i];
    if (s.ragged != ragged) continue;
    const int64_t tiles = ceil_div(M, s.bm) * ceil_div(N, s.bn) * batch;
    // what each further split costs at least: the partials' finalize, a launch and an HBM pass
    auto finalize = [&](int64_t used) {
      return 4.5 + 0.35 * static_cast<double>(used) +
             static_cast<double>(4 * used + 2) * M * static_cast<double>(N) * batch / 6.0e6;
    };
    for (int want = split_k > 0 ? split_k : 1; want <= (split_k > 0 ? split_k : 32); ++want) {
      // the k range of a split is a whole number of k-tiles; `used` splits are not empty
      const int64_t kt = ceil_div(ktiles, want), used = ceil_div(ktiles, kt);
      if (split_k == 0 && want > 1) {
        // no later `want` can be better: its ranges are no longer, its finalize no cheaper
        if (kt < 4 || batch * used > 65535) break;
        if (best.tile && s.fixed + finalize(want) >= best.cost) break;
        if (used != want) continue;
      }
      const int64_t wgs = tiles * used, held = cus * s.per_cu;
      const int64_t full = wgs / held, last = wgs % held;
      // `share` workgroups on each CU: the slower of one's serial chain and the CU's throughput;
      // a launch that fills under half of the CUs meets less contention
      auto per_ktile = [&](int64_t wg) {
        const double share = static_cast<double>(ceil_div(wg, cus));
        const double busy = 2 * wg < cus ? s.alone : s.shared * share;
        return busy > s.alone ? busy : s.alone;
      };
      double cost = s.fixed + round * static_cast<double>(full + (last > 0) - 1);
      if (full > 0) cost += static_cast<double>(kt * full) * per_ktile(held);
      if (last > 0) cost += static_cast<double>(kt) * per_ktile(last);
      if (used > 1) cost += finalize(used);
      if (best.tile == 0 || cost < best.cost)
        best = FlexPlan{i + 1, static_cast<int>(used), static_cast<int>(kt * BK), cost};
    }
  }
  return best;
}

int bgemm_flex_tile_rows(int tile) { return tile ? kShapes[tile - 1].bm : 0; }

hipError_t bgemm_flex_run(int tile, const FlexCall& c, hipStream_t stream) {
  HK_CHECK_ARG(tile >= 1 && tile <= kNumShapes && c.used >= 1 && (c.used == 1 || c.part));
  FlexArgs<Epi> g{};
  g.M = c.M, g.N = c.N, g.K = c.K;
  if (c.ep) g.ep = *c.ep;
  g.a = Operand{c.A, c.lda, c.sA};
  g.b = Operand{c.B, c.ldb, c.sB};
  g.C = c.C, g.ldc = c.ldc, g.sC = c.sC;
  g.split_k = c.used, g.k_per_split = c.used > 1 ? c.kps : c.K;
  g.part = c.used > 1 ? c.part : nullptr;
  if (c.used == 1 && c.out) g.fo = *c.out;
  return kShapes[tile - 1].run(c.ta, c.tb, g, c.batch, stream);
}

}  // namespace hk

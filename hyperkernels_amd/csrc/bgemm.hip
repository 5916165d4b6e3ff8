// bgemm.hip - batched BF16 GEMM on gfx950 MFMA: C = alpha * op(A) op(B) + beta * C,
// bf16 operands, fp32 accumulation, bf16 output, row-major, all four transpose layouts.
//
// Reference behaviour:
//   bgemm_NN_kernel<transA, transB>          blas/bf16/bgemm_nn_128x128_sm89_kernel.cu:23-216
//   bgemm_NN_128x128_64x3_kernel             blas/bf16/bgemm_nn_128x128_64x3_sm89_kernel.cu:23
//   bgemm_backward_template_kernel<...>      blas/bf16/bgemm_core_template.cu:61-268 (NN/NT/TN,
//                                            split-K accumulated with bf16 atomics)
//   bgemm_nt_backward_kernel (dA)            blas/bf16/bgemm_backward_nt_sm89_kernel.cu:23-180
//   bgemm_tn_backward_kernel (dB)            blas/bf16/bgemm_backward_tn_sm89_kernel.cu:25-182
// Layouts (row-major): op(A) = A [M,K] (lda >= K) or A^T with A stored [K,M] (lda >= M);
// op(B) = B [K,N] (ldb >= N) or B^T with B stored [N,K] (ldb >= K).
//
// Design (gfx950, CDNA4):
//   - Workgroup tile 256 x 256, k-tile 64, 8 waves (2 x 4, two per SIMD); each wave owns a
//     128 x 64 block of C as 4 x 2 tiles of v_mfma_f32_32x32x16_bf16 (128 fp32 accumulators
//     per lane). Per 16-deep k step a wave issues 8 MFMAs against 6 operand reads from LDS.
//     Two waves per SIMD let one issue MFMAs while the other waits on LDS or the barrier: 4-9%
//     faster than 4 waves of 128 x 128 at the BASELINE shapes and at 8192^3.
//   - HBM/L2 -> LDS copies bypass registers (global_load_lds_dwordx4, 16 bytes per lane) into
//     a 2-stage LDS ring: tile kt + 2 is copied while tile kt is multiplied, with one barrier
//     per k-tile. K-major operands are stored [row][k] and read with ds_read_b128; M/N-major
//     operands are stored as they lie in HBM, [k][row], and read with the gfx950 transposing
//     LDS read (ds_read_b64_tr_b16), so no layout needs a register transpose. The bank
//     placement of both is chosen through the per-lane source addresses of the copies.
//   - Operand reads of the next k step are interleaved with the current step's MFMAs
//     (sched_group_barrier), and the copies of the next tiles with the MFMAs of the last
//     step and of the first two.
//   - Epilogue through LDS: with the MFMA inputs swapped, each lane holds 4 consecutive
//     columns of one output row per accumulator quad; each wave stages its rows in LDS and
//     reads them back as 8 consecutive columns per lane. alpha / beta are applied in fp32 with
//     one rounding to bf16 (v_cvt_pk_bf16_f32, round to nearest even) and 16 bytes are stored
//     per lane, non-temporal (the reference rounds alpha * acc to bf16 and then blends beta * C
//     in bf16 arithmetic).
//   - Columns that would leave a last round of 256-wide tiles partly empty run as 128-wide
//     tiles in the same launch (column_split, bgemm_mixed).
//   - Edges: rows past M (N) are read clamped to the last row and their outputs are not
//     stored; k past the end of the (split's) range is zero-filled in LDS on the last k-tile.
//   - Workgroup order: consecutive tiles go to one XCD (the hardware deals workgroups to the 8
//     XCDs round-robin) in groups of 8 tile-rows, so each XCD's L2 sees a compact C region.
//   - Split-K (the core-template entry point with splitK > 1): each split writes fp32 partials
//     to the library workspace; a second kernel sums them in split order and applies
//     alpha/beta (deterministic; the reference accumulates with lossy bf16 atomics).
// Products of few such tiles and operands whose rows are no whole 16-byte vectors run on the tiles of
// bgemm_flex.hip (make_plan); leading dimensions those do not take either, and K == 0, on a simple
// fp32-accumulating kernel.
#include "bgemm_flex.h"
#include "bgemm_plan.h"
#include "bgemm_wide.h"

namespace {

using namespace hk::gemm;

// C = alpha * sum_s part[s] + beta * C or + beta * bias (split order), fp32 -> bf16, four
// consecutive outputs per thread. I: the index type, uint32_t when every index of the launch fits
// in 31 bits (a 64-bit division costs several times a 32-bit one).
template <typename I>
__global__ __launch_bounds__(256) void bgemm_splitk_finalize(const float* __restrict__ part,
                                                             int split_k, int batch, int M, int N,
                                                             Epi ep, uint16_t* __restrict__ C,
                                                             int64_t ldc, int64_t sC) {
  const I idx = (static_cast<I>(blockIdx.x) * 256 + threadIdx.x) * 4;
  const I pitch = part_pitch(N), mn = static_cast<I>(M) * pitch;
  if (idx >= mn * batch) return;
  const I b = idx / mn;
  const I e = idx - b * mn;
  const int row = static_cast<int>(e / pitch);
  const int col = static_cast<int>(e - static_cast<I>(row) * pitch);
  if (col >= N) return;
  f32x2_t lo = f32x2_t{0.f, 0.f}, hi = f32x2_t{0.f, 0.f};
  for (int k = 0; k < split_k; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(part + (static_cast<int64_t>(k) * batch + b) * mn + e);
    lo += f32x2_t{v.x, v.y};
    hi += f32x2_t{v.z, v.w};
  }
  lo *= ep.alpha;
  hi *= ep.alpha;
  uint16_t* cp = C + b * sC + static_cast<int64_t>(row) * ldc + col;
  if (ep.ragged) {  // rows of C at any 2-byte address, columns past N not stored
    const float f[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (col + i >= N) break;
      float v = f[i];
      if (ep.bias) v += ep.beta * bias_at(ep, row, col + i);
      else if (ep.beta != 0.0f) v += ep.beta * hk::bf16_to_f32(cp[i]);
      cp[i] = hk::f32_to_bf16(v);
    }
    return;
  }
  uint2* dst = reinterpret_cast<uint2*>(cp);
  if (ep.bias) {
    lo += ep.beta * f32x2_t{bias_at(ep, row, col), bias_at(ep, row, col + 1)};
    hi += ep.beta * f32x2_t{bias_at(ep, row, col + 2), bias_at(ep, row, col + 3)};
  } else if (ep.beta != 0.0f) {
    const float beta = ep.beta;
    const uint2 old = *dst;
    lo += beta * f32x2_t{__uint_as_float(old.x << 16), __uint_as_float(old.x & 0xffff0000u)};
    hi += beta * f32x2_t{__uint_as_float(old.y << 16), __uint_as_float(old.y & 0xffff0000u)};
  }
  const bf16x2_t blo = __builtin_convertvector(lo, bf16x2_t);
  const bf16x2_t bhi = __builtin_convertvector(hi, bf16x2_t);
  uint2 v;
  __builtin_memcpy(&v.x, &blo, 4);
  __builtin_memcpy(&v.y, &bhi, 4);
  *dst = v;
}

hipError_t launch_splitk_finalize(hipStream_t stream, const float* part, int used, int batch,
                                         int M, int N, const Epi& ep, uint16_t* C, int64_t ldc,
                                         int64_t sC) {
  const int64_t total = static_cast<int64_t>(M) * part_pitch(N) * batch;
  const dim3 grid(static_cast<unsigned>(hk::ceil_div(total, 1024)));
  if (total < (int64_t{1} << 31))
    hipLaunchKernelGGL(bgemm_splitk_finalize<uint32_t>, grid, dim3(256), 0, stream, part, used,
                       batch, M, N, ep, C, ldc, sC);
  else
    hipLaunchKernelGGL(bgemm_splitk_finalize<int64_t>, grid, dim3(256), 0, stream, part, used,
                       batch, M, N, ep, C, ldc, sC);
  return hk::launch_status();
}

// Fallback: one thread per output, fp32 accumulation in k order.
__global__ __launch_bounds__(256) void bgemm_simple(int ta, int tb, int M, int N, int K, Epi ep,
                                                    const uint16_t* __restrict__ A,
                                                    int64_t lda, int64_t sA,
                                                    const uint16_t* __restrict__ B, int64_t ldb,
                                                    int64_t sB, uint16_t* __restrict__ C,
                                                    int64_t ldc, int64_t sC) {
  const int col = blockIdx.x * 16 + (threadIdx.x & 15);
  const int row = blockIdx.y * 16 + (threadIdx.x >> 4);
  const int b = blockIdx.z;
  if (row >= M || col >= N) return;
  const uint16_t* Ab = A + b * sA;
  const uint16_t* Bb = B + b * sB;
  float acc = 0.f;
  for (int k = 0; k < K; ++k) {
    const float a = hk::bf16_to_f32(ta ? Ab[static_cast<int64_t>(k) * lda + row]
                                       : Ab[static_cast<int64_t>(row) * lda + k]);
    const float v = hk::bf16_to_f32(tb ? Bb[static_cast<int64_t>(col) * ldb + k]
                                       : Bb[static_cast<int64_t>(k) * ldb + col]);
    acc += a * v;
  }
  uint16_t* dst = C + b * sC + static_cast<int64_t>(row) * ldc + col;
  float f = ep.alpha * acc;
  if (ep.bias) f += ep.beta * bias_at(ep, row, col);
  else if (ep.beta != 0.0f) f += ep.beta * hk::bf16_to_f32(*dst);
  *dst = hk::f32_to_bf16(f);
}

// Split-K chosen by the library when the caller gives none, at most `most`: the split with the least modelled
// time (us), summed over the rounds of 256 x 256 work items on the CUs:
//   - a round costs (k-tiles per split) x t(busy) plus a fixed prologue / epilogue (8 us with
//     bf16 C, 12 us with a 256 KiB fp32 partial per tile);
//   - t, a workgroup's time per k-tile, grows with the share of the CUs that are busy (clock
//     and shared-cache headroom): ~0.875 us with 100 of 256 CUs busy, ~1.62 us with all;
//   - splits add the finalize, an HBM pass over the partials (4 s + 2 bytes per output at
//     ~6 TB/s).
// Calibrated on the 8192 x 1280 x 5120 and 1280 x 5120 x 8192 products (160 and 100 tiles):
// measured 123 / 149 / 131 us at 1 / 2 / 3 splits for the first, 120 / 115 / 151 / 137 / 135
// us at 1 to 5 for the second; the model picks 1 and 2.
int auto_split_k(int64_t work_tiles, int64_t ktiles, int64_t outputs, int most, double* best_cost) {
  const int64_t cus = hk::device_cu_count();
  auto t_kt = [&](int64_t busy) {
    const double f = static_cast<double>(busy) / static_cast<double>(cus);
    const double x = (f - 0.39) / 0.61;
    return 0.875 + 0.745 * (x < 0.0 ? 0.0 : x > 1.0 ? 1.0 : x);
  };
  double best = 0.0;
  int best_s = 1;
  for (int s = 1; s <= most; ++s) {
    if (s > 1 && ktiles / s < 4) break;
    const int64_t items = work_tiles * s, kps = hk::ceil_div(ktiles, static_cast<int64_t>(s));
    const double fixed = s > 1 ? 12.0 : 8.0;
    double cost = 0.0;
    for (int64_t done = 0; done < items; done += cus) {
      const int64_t busy = items - done < cus ? items - done : cus;
      cost += static_cast<double>(kps) * t_kt(busy) + fixed;
    }
    if (s > 1) cost += static_cast<double>(4 * s + 2) * static_cast<double>(outputs) / 6.0e6;
    if (s == 1 || cost < best) {
      best = cost;
      best_s = s;
    }
  }
  if (best_cost) *best_cost = best;
  return best_s;
}

constexpr int kMostSplits = 8;      // of the library's own choice on the 256-wide tiles
constexpr int kMaxGridZ = 65535;  // batches x k splits of one launch

using Rows = hk::GemmRows;
Rows row_kind(bool ta, bool tb, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
              int64_t sA, int64_t sB, int64_t sC, int batch, bool a16, bool b16, bool c16) {
  if (K <= 0 || lda >= (1 << 22) || ldb >= (1 << 22)) return Rows::kNone;
  const int contig_a = ta ? M : K, contig_b = tb ? K : N;
  const bool ab = contig_a % 8 == 0 && contig_b % 8 == 0 && lda % 8 == 0 && ldb % 8 == 0 &&
                  sA % 8 == 0 && sB % 8 == 0 && a16 && b16;
  if (ab && N % 8 == 0 && ldc % 8 == 0 && sC % 8 == 0 && c16) return Rows::kAligned;
  if (batch > kMaxGridZ) return Rows::kNone;
  if (ab) return Rows::kRaggedC;
  return lda >= 8 && ldb >= 8 ? Rows::kRagged : Rows::kNone;
}
// The same for contiguous, 16-byte aligned operands (the planning queries).
Rows packed_rows(bool ta, bool tb, int M, int N, int K, int batch) {
  const int64_t lda = ta ? M : K, ldb = tb ? K : N;
  return row_kind(ta, tb, M, N, K, lda, ldb, N, lda * (ta ? K : M), ldb * (tb ? N : K),
                  static_cast<int64_t>(M) * N, batch, true, true, true);
}

using Plan = hk::GemmPlan;

// Modelled time (us) of the 256-wide tiles' plan for one k split (auto_split_k covers the others),
// with the tile shape run_regions picks.
double wide_cost(bool ta, bool tb, int M, int N, int K, int batch, int splits, double split_cost) {
  if (splits > 1) return split_cost;
  const double kt = static_cast<double>(hk::ceil_div(K, BK));
  if (N <= 128) {
    // one column of 128-wide tiles: less per k-tile on a busy device and per further round (MI355X, us:
    // 200 x 104 x 2176 in 200 batches 41, by auto_split_k's figures 54; 1216 x 112 x 24 in 400, 41 and 77)
    const int64_t cus = hk::device_cu_count(), items = hk::ceil_div(M, BM) * batch;
    auto t_kt = [&](int64_t busy) {
      const double x = (static_cast<double>(busy) / static_cast<double>(cus) - 0.39) / 0.61;
      return 0.79 + 0.25 * (x < 0.0 ? 0.0 : x);
    };
    const int64_t full = items / cus, last = items % cus;
    return 8.0 + 4.0 * static_cast<double>(full + (last > 0) - 1) +
           kt * (static_cast<double>(full) * t_kt(cus) + (last > 0 ? t_kt(last) : 0.0));
  }
  if (w160_plan(ta, tb, M, N, K, batch, 1)) return 8.0 + 0.99 * kt;
  if (row_tile(ta, M, N, batch, 1) == 192) return 8.0 + (split_cost - 8.0) * 0.85;
  return split_cost;
}

// The library's choice between the two families (split_k == 0): the smaller modelled time, the
// 256-wide tiles kept unless the other is 5% faster. An explicit split keeps the 256-wide tiles
// where they take the operands.
Plan make_plan(bool ta, bool tb, int M, int N, int K, int batch, int split_k, Rows rows) {
  const bool ragged = rows == Rows::kRagged;
  Plan wide{0, 1, K};
  double cost = 0.0;
  if (!ragged) {
    hk::bgemm_split_plan(M, N, K, batch, split_k, &wide.used, &wide.kps, &cost);
    if (split_k > 0) return wide;
    cost = wide_cost(ta, tb, M, N, K, batch, wide.used, cost);
  }
  const hk::FlexPlan f = hk::bgemm_flex_plan(M, N, K, batch, split_k, ragged);
  if (!ragged && f.cost > 0.95 * cost) return wide;
  return Plan{f.tile, f.used, f.kps};
}

size_t partial_bytes(int used, int M, int N, int batch) {
  return static_cast<size_t>(used) * batch * M * part_pitch(N) * sizeof(float);
}

// The better of the two families where partials may take `held` bytes at most: the small and
// any-alignment tiles with one k split, the 256-wide ones with as many of their splits as fit.
Plan lean_plan(bool ta, bool tb, int M, int N, int K, int batch, Rows rows, size_t held) {
  const bool ragged = rows == Rows::kRagged;
  const hk::FlexPlan f = hk::bgemm_flex_plan(M, N, K, batch, 1, ragged);
  if (!ragged) {
    const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
    const size_t fit = held / partial_bytes(1, M, N, batch);
    const int most = fit < 2 ? 1 : fit < kMostSplits ? static_cast<int>(fit) : kMostSplits;
    double cost = 0.0;
    const int s = auto_split_k(tiles * batch, hk::ceil_div(K, BK),
                               static_cast<int64_t>(M) * N * batch, most, &cost);
    Plan wide{0, 1, K};
    if (s > 1) {
      wide.kps = static_cast<int>(hk::ceil_div(hk::ceil_div(K, s), BK) * BK);
      wide.used = static_cast<int>(hk::ceil_div(K, wide.kps));
    }
    // one chain over a deep k runs up to 1.6 times the modelled time (176 x 312 x 6152 TN, unaligned to
    // cache lines: 37 us for 23), so splits are given up for it only where it looks far better
    const double margin = wide.used > 1 ? 0.65 : 0.95;
    if (f.cost > margin * wide_cost(ta, tb, M, N, K, batch, wide.used, cost)) return wide;
  }
  return Plan{f.tile, 1, K};
}

// bias == NULL: C = alpha * op(A) op(B) + beta * C. Otherwise C = alpha * op(A) op(B) +
// beta * bias with bias_numel N (per column), M (per row), 1 (scalar) or M*N (full, shared by
// all batches), tested in that order; C is then only written.
hipError_t bgemm_run(int transA, int transB, int M, int N, int K, hk_bf16 alpha_bits,
                     const hk_bf16* A, int lda, long long strideA, const hk_bf16* B, int ldb,
                     long long strideB, hk_bf16 beta_bits, const hk_bf16* bias,
                     int64_t bias_numel, hk_bf16* C, int ldc, long long strideC, int batchCount,
                     int splitK, hipStream_t stream) {
  HK_CHECK_ARG(transA >= 0 && transA <= 2 && transB >= 0 && transB <= 2);
  // splitK == 0: the library picks the split (auto_split_k)
  HK_CHECK_ARG(M >= 0 && N >= 0 && K >= 0 && batchCount >= 0 && splitK >= 0);
  if (M == 0 || N == 0 || batchCount == 0) return hipSuccess;
  HK_CHECK_ARG(C != nullptr && ldc >= N);
  const bool ta = transA != 0, tb = transB != 0;  // OP_C is OP_T for real bf16
  HK_CHECK_ARG(K == 0 || (A != nullptr && B != nullptr));
  HK_CHECK_ARG(lda >= (ta ? M : K) && ldb >= (tb ? K : N));
  if (!bias && splitK == 0 && (M == 1 || N == 1)) {
    // A one-row or one-column product streams one operand once: the GEMV kernels
    if (M == 1)  // C[0][n] = sum_k op(A)[0][k] op(B)[k][n]
      return hk::bgemv_run(tb, N, K, alpha_bits, beta_bits, B, ldb, strideB, A, ta ? lda : 1,
                           strideA, C, 1, strideC, batchCount, stream);
    // C[m][0] = sum_k op(A)[m][k] op(B)[k][0]
    return hk::bgemv_run(!ta, M, K, alpha_bits, beta_bits, A, lda, strideA, B, tb ? 1 : ldb,
                         strideB, C, ldc, strideC, batchCount, stream);
  }
  Epi ep{hk::bf16_bits_to_float(alpha_bits), hk::bf16_bits_to_float(beta_bits), bias, 0, 0, false};
  if (bias) {
    if (bias_numel == N) ep.bcol = 1;
    else if (bias_numel == M) ep.brow = 1;
    else if (bias_numel == 1) { /* scalar: (0, 0) */ }
    else if (bias_numel == static_cast<int64_t>(M) * N) { ep.brow = N; ep.bcol = 1; }
    else return hipErrorInvalidValue;
  }

  const Rows rows = row_kind(ta, tb, M, N, K, lda, ldb, ldc, strideA, strideB, strideC,
                             batchCount, hk::aligned16(A), hk::aligned16(B), hk::aligned16(C));
  if (rows == Rows::kNone) {
    dim3 grid((N + 15) / 16, (M + 15) / 16, batchCount);
    hipLaunchKernelGGL(bgemm_simple, grid, dim3(256), 0, stream, ta ? 1 : 0, tb ? 1 : 0, M, N,
                       K, ep, A, static_cast<int64_t>(lda), static_cast<int64_t>(strideA), B,
                       static_cast<int64_t>(ldb), static_cast<int64_t>(strideB), C,
                       static_cast<int64_t>(ldc), static_cast<int64_t>(strideC));
    return hk::launch_status();
  }
  ep.ragged = rows != Rows::kAligned;
  Plan plan = make_plan(ta, tb, M, N, K, batchCount, splitK, rows);
  // The small tiles' splits and those of unaligned rows are left out where the grid or the memory
  // does not take them, and under capture: such calls need no workspace then, whose size the capture
  // could not change and which replays would share with the stream's eager calls. Aligned rows may
  // still take the 256-wide tiles' splits there, in the workspace that the stream has.
  const bool optional = plan.flex || ep.ragged;
  if (plan.used > 1 && optional) {
    const bool capturing = hk::stream_capturing(stream);
    if (capturing || static_cast<int64_t>(batchCount) * plan.used > kMaxGridZ)
      plan = lean_plan(ta, tb, M, N, K, batchCount, rows,
                       capturing && !ep.ragged ? hk::device_workspace_bytes(stream) : 0);
  }
  const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  HK_CHECK_ARG(2 * tiles <= INT32_MAX && static_cast<int64_t>(batchCount) * plan.used <= kMaxGridZ);
  void* ws = nullptr;
  if (plan.used > 1) {
    // room for the 256-wide tiles' splits, too, which a captured call of the shape falls back on
    int room = plan.used, wide = 1, kps = K;
    if (plan.flex && !ep.ragged) {
      hk::bgemm_split_plan(M, N, K, batchCount, 0, &wide, &kps);
      if (wide > room) room = wide;
    }
    const hipError_t e = hk::device_workspace(partial_bytes(room, M, N, batchCount), stream, &ws);
    if (e == hipErrorOutOfMemory && optional) {
      (void)hipGetLastError();
      plan = lean_plan(ta, tb, M, N, K, batchCount, rows, 0);
    } else {
      HK_RETURN_IF_ERROR(e);
    }
  }
  float* part = static_cast<float*>(ws);
  if (plan.flex) {
    HK_RETURN_IF_ERROR(hk::bgemm_flex_run(
        plan.flex, hk::FlexCall{ta, tb, M, N, K, batchCount, A, lda, strideA, B, ldb, strideB, C,
                                ldc, strideC, &ep, plan.used, plan.kps, part, nullptr},
        stream));
  } else if (plan.used == 1) {
    return run_regions<false>(ta, tb, batchCount, stream, M, N, K, ep, A, lda, strideA, B, ldb,
                              strideB, C, ldc, strideC, 1, K, nullptr, hk::F32Out{});
  } else {
    HK_RETURN_IF_ERROR(run_regions<true>(ta, tb, batchCount * plan.used, stream, M, N, K, ep, A,
                                         lda, strideA, B, ldb, strideB, C, ldc, strideC,
                                         plan.used, plan.kps, part, hk::F32Out{}));
  }
  if (plan.used == 1) return hipSuccess;
  return launch_splitk_finalize(stream, part, plan.used, batchCount, M, N, ep, C,
                                static_cast<int64_t>(ldc), static_cast<int64_t>(strideC));
}

}  // namespace

namespace hk {

void bgemm_split_plan(int M, int N, int K, int batch, int split_k, int* used, int* kps,
                      double* cost) {
  const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  const int s = split_k > 0 ? split_k
                            : auto_split_k(tiles * batch, hk::ceil_div(K, BK),
                                           static_cast<int64_t>(M) * N * batch, kMostSplits, cost);
  *kps = static_cast<int>(hk::ceil_div(hk::ceil_div(K, s), BK) * BK);
  *used = static_cast<int>(hk::ceil_div(K, *kps));
}

GemmPlan bgemm_plan(bool ta, bool tb, int M, int N, int K, int batch, int split_k) {
  return make_plan(ta, tb, M, N, K, batch, split_k, Rows::kAligned);
}

GemmPlan bgemm_lean_plan(bool ta, bool tb, int M, int N, int K, int batch, size_t held) {
  return lean_plan(ta, tb, M, N, K, batch, Rows::kAligned, held);
}

GemmRows bgemm_rows(bool ta, bool tb, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                    int64_t sA, int64_t sB, int64_t sC, int batch, bool a16, bool b16, bool c16) {
  return row_kind(ta, tb, M, N, K, lda, ldb, ldc, sA, sB, sC, batch, a16, b16, c16);
}

GemmPlan bgemm_rows_plan(bool ta, bool tb, int M, int N, int K, int batch, GemmRows rows,
                         bool may_split) {
  const Plan p = make_plan(ta, tb, M, N, K, batch, 0, rows);
  if (p.used == 1 || (may_split && static_cast<int64_t>(batch) * p.used <= kMaxGridZ)) return p;
  return lean_plan(ta, tb, M, N, K, batch, rows, 0);
}

size_t bgemm_partial_bytes(int used, int M, int N, int batch) {
  return partial_bytes(used, M, N, batch);
}

hipError_t bgemm_write_partials(bool ta, bool tb, int M, int N, int K, const hk_bf16* A, int64_t lda,
                                int64_t sA, const hk_bf16* B, int64_t ldb, int64_t sB, int batch,
                                const GemmPlan& plan, float* part, hipStream_t stream) {
  HK_CHECK_ARG(plan.used > 1 && part != nullptr);
  if (plan.flex)
    return bgemm_flex_run(plan.flex,
                          FlexCall{ta, tb, M, N, K, batch, A, lda, sA, B, ldb, sB, nullptr, 0, 0,
                                   nullptr, plan.used, plan.kps, part, nullptr},
                          stream);
  const Epi ep{1.0f, 0.0f, nullptr, 0, 0, false};
  return run_regions<true>(ta, tb, batch * plan.used, stream, M, N, K, ep, A, lda, sA, B, ldb, sB,
                           nullptr, 0, 0, plan.used, plan.kps, part, F32Out{});
}

hipError_t bgemm_partials(bool ta, bool tb, int M, int N, int K, const hk_bf16* A, int64_t lda,
                          int64_t sA, const hk_bf16* B, int64_t ldb, int64_t sB, int batch,
                          const GemmPlan& plan, float* part, const F32Out* out,
                          hipStream_t stream) {
  const int used = plan.used, kps = plan.kps;
  const int contig_a = ta ? M : K, contig_b = tb ? K : N;
  HK_CHECK_ARG(M > 0 && N > 0 && K > 0 && batch > 0 && used >= 1 && (used == 1 || kps % BK == 0));
  HK_CHECK_ARG(contig_a % 8 == 0 && contig_b % 8 == 0 && N % 8 == 0 && lda % 8 == 0 &&
               ldb % 8 == 0 && sA % 8 == 0 && sB % 8 == 0 && hk::aligned16(A) &&
               hk::aligned16(B) && lda < (1 << 22) && ldb < (1 << 22));
  const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  HK_CHECK_ARG(2 * tiles <= INT32_MAX && static_cast<int64_t>(batch) * used <= 65535);
  if (plan.flex)
    return bgemm_flex_run(plan.flex,
                          FlexCall{ta, tb, M, N, K, batch, A, lda, sA, B, ldb, sB, nullptr, 0, 0,
                                   nullptr, used, kps, part, out},
                          stream);
  const Epi ep{1.0f, 0.0f, nullptr, 0, 0, false};
  const F32Out fo = used == 1 && out ? *out : F32Out{};
  return run_regions<true>(ta, tb, batch * used, stream, M, N, K, ep, A, lda, sA, B, ldb, sB,
                           nullptr, 0, 0, used, used == 1 ? K : kps, part, fo);
}

}  // namespace hk

// 0: empty, -1: invalid, 1: the GEMV kernels or the fallback, 2: the MFMA tiles.
static int query_kind(int transA, int transB, int M, int N, int K, int batchCount, int splitK) {
  if (transA < 0 || transA > 2 || transB < 0 || transB > 2 || M < 0 || N < 0 || K < 0 ||
      batchCount < 0 || splitK < 0)
    return -1;
  if (M == 0 || N == 0 || batchCount == 0) return 0;
  if (splitK == 0 && (M == 1 || N == 1)) return 1;
  return packed_rows(transA != 0, transB != 0, M, N, K, batchCount) == Rows::kNone ? 1 : 2;
}

extern "C" int hk_bgemm_split_count(int transA, int transB, int M, int N, int K, int batchCount,
                                    int splitK) {
  const int kind = query_kind(transA, transB, M, N, K, batchCount, splitK);
  if (kind < 2) return kind;
  const bool ta = transA != 0, tb = transB != 0;
  return make_plan(ta, tb, M, N, K, batchCount, splitK, packed_rows(ta, tb, M, N, K, batchCount)).used;
}

extern "C" int hk_bgemm_small_tile(int transA, int transB, int M, int N, int K, int batchCount,
                                   int splitK) {
  const int kind = query_kind(transA, transB, M, N, K, batchCount, splitK);
  if (kind < 2) return kind < 0 ? -1 : 0;
  const bool ta = transA != 0, tb = transB != 0;
  return hk::bgemm_flex_tile_rows(
      make_plan(ta, tb, M, N, K, batchCount, splitK, packed_rows(ta, tb, M, N, K, batchCount)).flex);
}

// The 256-wide tiles' own plan for a product whose operands they take; splits: its k splits.
static int wide_tile(int transA, int transB, int M, int N, int K, int batchCount, int splitK,
                     bool cols) {
  const int kind = query_kind(transA, transB, M, N, K, batchCount, splitK);
  if (kind <= 0) return kind;
  const bool ta = transA != 0, tb = transB != 0;
  if (kind == 1 || packed_rows(ta, tb, M, N, K, batchCount) == Rows::kRagged) return 0;
  int used = 1, kps = 0;
  hk::bgemm_split_plan(M, N, K, batchCount, splitK, &used, &kps);
  if (w160_plan(ta, tb, M, N, K, batchCount * used, used)) return cols ? w160::kBN : w160::kBM;
  return cols ? BN : row_tile(ta, M, N, batchCount * used, used);
}

extern "C" int hk_bgemm_tile_rows(int transA, int transB, int M, int N, int K, int batchCount,
                                  int splitK) {
  return wide_tile(transA, transB, M, N, K, batchCount, splitK, false);
}

extern "C" int hk_bgemm_tile_cols(int transA, int transB, int M, int N, int K, int batchCount,
                                  int splitK) {
  return wide_tile(transA, transB, M, N, K, batchCount, splitK, true);
}

extern "C" hipError_t hk_bgemm(int transA, int transB, int M, int N, int K, hk_bf16 alpha,
                               const hk_bf16* A, int lda, long long strideA, const hk_bf16* B,
                               int ldb, long long strideB, hk_bf16 beta, hk_bf16* C, int ldc,
                               long long strideC, int batchCount, hipStream_t stream) {
  return bgemm_run(transA, transB, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, beta,
                   nullptr, 0, C, ldc, strideC, batchCount, 0, stream);
}

extern "C" hipError_t hk_bgemm_core(int layout, int splitK, int M, int N, int K, hk_bf16 alpha,
                                    const hk_bf16* A, int lda, long long strideA,
                                    const hk_bf16* B, int ldb, long long strideB, hk_bf16 beta,
                                    hk_bf16* C, int ldc, long long strideC, int batchCount,
                                    hipStream_t stream) {
  // BgemmLayout { NT, TN, NN } (blas/bf16/bgemm_core_template.cu:59)
  HK_CHECK_ARG(layout >= HK_LAYOUT_NT && layout <= HK_LAYOUT_NN);
  HK_CHECK_ARG(splitK >= 1);
  const int ta = layout == HK_LAYOUT_TN ? 1 : 0;
  const int tb = layout == HK_LAYOUT_NT ? 1 : 0;
  return bgemm_run(ta, tb, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, beta, nullptr, 0,
                   C, ldc, strideC, batchCount, splitK, stream);
}

extern "C" hipError_t hk_bgemm_nt_backward(int M, int N, int K, hk_bf16 alpha, const hk_bf16* A,
                                           int lda, long long strideA, const hk_bf16* B, int ldb,
                                           long long strideB, hk_bf16 beta, hk_bf16* C, int ldc,
                                           long long strideC, int batchCount,
                                           hipStream_t stream) {
  return bgemm_run(0, 1, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, beta, nullptr, 0,
                   C, ldc, strideC, batchCount, 0, stream);
}

extern "C" hipError_t hk_bgemm_tn_backward(int M, int N, int K, hk_bf16 alpha, const hk_bf16* A,
                                           int lda, long long strideA, const hk_bf16* B, int ldb,
                                           long long strideB, hk_bf16 beta, hk_bf16* C, int ldc,
                                           long long strideC, int batchCount,
                                           hipStream_t stream) {
  return bgemm_run(1, 0, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, beta, nullptr, 0,
                   C, ldc, strideC, batchCount, 0, stream);
}

extern "C" hipError_t hk_bgemm_addmm(int M, int N, int K, hk_bf16 alpha, const hk_bf16* A, int lda,
                                     long long strideA, const hk_bf16* B, int ldb,
                                     long long strideB, hk_bf16 beta, const hk_bf16* bias,
                                     int64_t bias_numel, hk_bf16* C, int ldc, long long strideC,
                                     int batchCount, hipStream_t stream) {
  // C is only written: without a bias the product is C = alpha * A B (bgemm_addmm…:214-300)
  if (!bias) beta = 0;
  return bgemm_run(0, 0, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, beta, bias,
                   bias_numel, C, ldc, strideC, batchCount, 0, stream);
}

extern "C" hipError_t hk_bgemm_core_bias(int layout, int splitK, int M, int N, int K, hk_bf16 alpha,
                                         const hk_bf16* A, int lda, long long strideA,
                                         const hk_bf16* B, int ldb, long long strideB,
                                         hk_bf16 beta, const hk_bf16* bias, int64_t bias_numel,
                                         hk_bf16* C, int ldc, long long strideC, int batchCount,
                                         hipStream_t stream) {
  HK_CHECK_ARG(layout >= HK_LAYOUT_NT && layout <= HK_LAYOUT_NN);
  HK_CHECK_ARG(splitK >= 1);
  const int ta = layout == HK_LAYOUT_TN ? 1 : 0;
  const int tb = layout == HK_LAYOUT_NT ? 1 : 0;
  return bgemm_run(ta, tb, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, beta, bias,
                   bias_numel, C, ldc, strideC, batchCount, splitK, stream);
}

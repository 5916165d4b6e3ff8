// bgemm_wide.h - the 256-wide tiles of the BF16 GEMM (see bgemm.hip for the design): the kernels, templated
// on the epilogue E of a bf16 C (Epi, or ActEpi of bgemm_act.h), and how a product is cut into them.
#pragma once

#include <mutex>
#include <type_traits>

#include "bgemm_tile.h"

namespace hk {
namespace gemm {

constexpr int BM = 256, BN = 256;                      // BN: the full tile width
constexpr int kStages = 2;                             // LDS ring depth (k-tiles)
constexpr int kWaves = 8;                              // 2 x 4 over the tile, 2 per SIMD
constexpr int kThreads = kWaves * 64;

// Tile height BMT (256, or 192 for products whose 256-row tiles would leave many CUs idle, see
// row_tile; 192 only with a k-major A): each wave owns BMT / 2 rows of C, kBlkM MFMA tiles of
// 32 rows.
template <int BMT>
struct TileM {
  static_assert(BMT == 256 || BMT == 192, "tile heights");
  static constexpr int kWaveM = BMT / 2;
  static constexpr int kBlkM = kWaveM / 32;
  static constexpr int kStageBytes = BMT * BK * 2;                   // A, one k-tile
  static constexpr int kLoadsPerWave = kStageBytes / 1024 / kWaves;  // 16-byte lane copies of A
};

// Tile width BNT (256, or 128 for the half-width tiles that fill a last round, see
// column_split): each wave owns BMT / 2 x BNT / 4 of C, kBlkN MFMA tiles of 32 columns.
template <int BNT, int BMT = 256>
struct TileN {
  static constexpr int kWaveN = BNT / 4;
  static constexpr int kBlkN = kWaveN / 32;
  static constexpr int kStageBytesB = BNT * BK * 2;
  static constexpr int kLoadsB = kStageBytesB / 1024 / kWaves;
  static constexpr size_t kLdsBytes =
      static_cast<size_t>(kStages) * (TileM<BMT>::kStageBytes + kStageBytesB);
  // the LDS of a kernel whose waves stage `blocks` block rows at a time
  static constexpr size_t lds_bytes(int blocks) {
    const size_t staging = static_cast<size_t>(kWaves) * blocks * 32 * (kWaveN * 4 + 16);
    return staging > kLdsBytes ? staging : kLdsBytes;
  }
};

// Main loop per k-tile kt (ring slot kt % 2), 4 k steps of 16 MFMAs each:
//   steps 0-2: operands of step s+1 are read from LDS between the MFMAs of step s; steps 0
//              and 1 first issue the second half of tile kt+1's copies (into slot (kt+1) % 2,
//              free since the barrier that ended tile kt-1);
//   step 3:    wait for this wave's copies of tile kt+1, barrier (tile kt+1 visible to all,
//              every wave done reading slot kt % 2), read step 0 of tile kt+1, and issue the
//              first half of tile kt+2's copies into slot kt % 2 between the MFMAs.
// A copy instruction (1 KiB) keeps the CU's address unit busy ~25 cycles (TA_TA_BUSY on
// MI355X), so a k-tile's 64 take ~1,600 of its ~2,048 MFMA cycles. Issued all in step 3 they
// held that step at ~1,160 cycles against 512 of MFMA work; split over steps 3, 0 and 1 the
// product runs ~1.5% faster (8192^3: 733 -> 721 us).
// The operands are swapped in the MFMA (B block as the "A" input), so each lane ends up
// holding 4 consecutive output columns of one output row per register quad; the epilogue
// hands them to the output through LDS (staged_rows).
// One workgroup's tile: tile `wg` of the BMT x BNT tiles that cover the columns
// [n_base, n_end) of C (N bounds the stores).
template <bool A_KMAJOR, bool B_KMAJOR, bool PARTIAL, int BNT, int BMT, class E>
__device__ __forceinline__ void tile_body(
    int M, int N, int K, const E& ep, const uint16_t* __restrict__ A, int64_t lda, int64_t sA,
    const uint16_t* __restrict__ B, int64_t ldb, int64_t sB, uint16_t* __restrict__ C,
    int64_t ldc, int64_t sC, int split_k, int k_per_split, float* __restrict__ part,
    const hk::F32Out& fo, int n_base, int n_end, int wg) {
  static_assert(BMT == 256 || A_KMAJOR, "192-row tiles need a k-major A");
  using OA = TileOperand<A_KMAJOR>;
  using OB = TileOperand<B_KMAJOR, BNT>;
  constexpr int kWaveN = TileN<BNT, BMT>::kWaveN, kBlkN = TileN<BNT, BMT>::kBlkN;
  constexpr int kStageBytesB = TileN<BNT, BMT>::kStageBytesB, kLoadsB = TileN<BNT, BMT>::kLoadsB;
  constexpr int kWaveM = TileM<BMT>::kWaveM, kBlkM = TileM<BMT>::kBlkM;
  constexpr int kStageBytes = TileM<BMT>::kStageBytes, kLoadsPerWave = TileM<BMT>::kLoadsPerWave;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  unsigned char HK_LDS* ldsA = (unsigned char HK_LDS*)lds_raw;
  unsigned char HK_LDS* ldsB = ldsA + kStages * kStageBytes;

  const int batch = blockIdx.z / split_k;
  const int split = blockIdx.z - batch * split_k;
  const int tiles_m = (M + BMT - 1) / BMT, tiles_n = (n_end - n_base + BNT - 1) / BNT;
  int tm, tn;
  tile_coords(wg, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BMT, n0 = n_base + tn * BNT;
  const int kbeg = split * k_per_split;
  const int klen = min(K, kbeg + k_per_split) - kbeg;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;

  // Tile bases at k = kbeg (wave-uniform) and per-lane source offsets of this wave's copy
  // instructions. Rows past M (N) are clamped to the last row: they only feed outputs that
  // are not stored. k past the split's end is zero-filled on the last k-tile (tail_fill).
  const unsigned char* gA = reinterpret_cast<const unsigned char*>(
      A + static_cast<int64_t>(batch) * sA +
      (A_KMAJOR ? static_cast<int64_t>(m0) * lda + kbeg : static_cast<int64_t>(kbeg) * lda + m0));
  const unsigned char* gB = reinterpret_cast<const unsigned char*>(
      B + static_cast<int64_t>(batch) * sB +
      (B_KMAJOR ? static_cast<int64_t>(n0) * ldb + kbeg : static_cast<int64_t>(kbeg) * ldb + n0));
  int offA[kLoadsPerWave], offB[kLoadsB];
  int kA[kLoadsPerWave], kB[kLoadsB];
#pragma unroll
  for (int i = 0; i < kLoadsPerWave; ++i) {
    int row, k;
    OA::source(wave * kLoadsPerWave + i, lane, row, k);
    row = min(row, (A_KMAJOR ? M - 8 + 7 : M - 8) - m0);  // k-major: a row; else an 8-row chunk
    offA[i] = static_cast<int>(OA::byte_offset(row, k, lda));
    kA[i] = k;
  }
#pragma unroll
  for (int i = 0; i < kLoadsB; ++i) {
    int row, k;
    OB::source(wave * kLoadsB + i, lane, row, k);
    row = min(row, (B_KMAJOR ? N - 8 + 7 : N - 8) - n0);
    offB[i] = static_cast<int>(OB::byte_offset(row, k, ldb));
    kB[i] = k;
  }
  const int64_t stepA = 2 * OA::ktile_step(lda), stepB = 2 * OB::ktile_step(ldb);
  const unsigned ldsA_addr = static_cast<unsigned>(reinterpret_cast<uintptr_t>(ldsA));
  const unsigned ldsB_addr = static_cast<unsigned>(reinterpret_cast<uintptr_t>(ldsB));
  const int ktiles = (klen + BK - 1) / BK;
  const bool tail = (klen % BK) != 0;  // last k-tile is partial

  // Copy q (0 .. kLoadsPerWave + kLoadsB - 1) of k-tile kt into ring slot `slot`. On a partial
  // last k-tile (fill), lanes whose 8 k values lie past the split's end store zeros instead.
  auto copy = [&](int kt, int slot, int q, bool fill) {
    const bool isA = q < kLoadsPerWave;
    const int i = isA ? q : q - kLoadsPerWave;
    const unsigned char* base = (isA ? gA + kt * stepA : gB + kt * stepB);
    const int off = isA ? offA[i] : offB[i];
    const unsigned lds = isA ? ldsA_addr + slot * kStageBytes + (wave * kLoadsPerWave + i) * 1024
                             : ldsB_addr + slot * kStageBytesB + (wave * kLoadsB + i) * 1024;
    if (!fill) {
      copy16_to_lds(base, off, lds);
    } else if (kt * BK + (isA ? kA[i] : kB[i]) < klen) {
      copy16_to_lds(base, off, lds);
    } else {
      typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
      *reinterpret_cast<u32x4_t HK_LDS*>((unsigned char HK_LDS*)(uintptr_t)lds + 16 * lane) =
          u32x4_t{0u, 0u, 0u, 0u};
    }
  };
  constexpr int kCopies = kLoadsPerWave + kLoadsB;
  // a k-tile's copies: kH3 in the last k step of the k-tile two before it, the other kRest in
  // the first two k steps of the k-tile before it
  constexpr int kH3 = (kCopies + 1) / 2, kRest = kCopies - kH3;

  f32x16_t acc[kBlkM][kBlkN];
#pragma unroll
  for (int i = 0; i < kBlkM; ++i)
#pragma unroll
    for (int j = 0; j < kBlkN; ++j) acc[i][j] = f32x16_t{};

  // The wave's rows of C, staged for the stores at the start of the ring. What the epilogue reads ahead is
  // issued before the copies, so that the waits below, which count those, cover it.
  unsigned char HK_LDS* area = ldsA + wave * (E::kWideStage * 32 * (kWaveN * 4 + 16));
  const int wrow0 = m0 + wm * kWaveM, wcol0 = n0 + wn * kWaveN;
  const WaveRows rows{C, ldc, sC, batch, M, N, wrow0, wcol0, 2 * tm + wm, area};
  const auto ahead = rows_ahead<kWaveN, E::kWideAhead>(ep, rows, lane);

#pragma unroll
  for (int p = 0; p < kStages; ++p)
    if (p < ktiles) {
      const bool fill = tail && p == ktiles - 1;
#pragma unroll
      for (int q = 0; q < kCopies; ++q) copy(p, p, q, fill);
    }
  // Wait for k-tile 0 only; k-tile 1 lands while tile 0 is multiplied (waited for at its end).
  // A partial (fill) k-tile 1 may have issued fewer copies than kCopies: wait for all then.
  if (ktiles >= 2 && !(tail && ktiles == 2))
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kCopies) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();

  bf16x8_t fa[2][kBlkM], fb[2][kBlkN];
  if (ktiles > 0) {
#pragma unroll
    for (int i = 0; i < kBlkM; ++i) fa[0][i] = OA::read(ldsA, wm * kWaveM, i, 0, lane);
#pragma unroll
    for (int j = 0; j < kBlkN; ++j) fb[0][j] = OB::read(ldsB, wn * kWaveN, j, 0, lane);
  }
  constexpr int kReadsPerStep = (A_KMAJOR ? 1 : 2) * kBlkM + (B_KMAJOR ? 1 : 2) * kBlkN;
  constexpr int kMfmaPerStep = kBlkM * kBlkN;

  // One k-tile. STEADY (compile-time): tile kt + kStages exists and is whole, so its 32 copies
  // are issued with no per-copy condition; otherwise whether it exists (more) and whether it is
  // the partial last k-tile (fill) are tested at run time.
  auto ktile = [&](int kt, auto steady_tag) {
    constexpr bool STEADY = decltype(steady_tag)::value;
    const bool more = STEADY || kt + kStages < ktiles;
    const bool fill = !STEADY && tail && kt + kStages == ktiles - 1;
    const int slot = kt & 1;
    const unsigned char HK_LDS* sa = ldsA + slot * kStageBytes;
    const unsigned char HK_LDS* sb = ldsB + slot * kStageBytesB;
    // the copies of tile kt + 1 that the previous k-tile's last step left (kt >= 1)
    const bool rest = kt > 0 && (STEADY || kt + 1 < ktiles);
    const bool rest_fill = !STEADY && tail && kt + 1 == ktiles - 1;
#pragma unroll
    for (int s = 0; s < BK / 16; ++s) {
      const int cur = s & 1, nxt = cur ^ 1;
      if (s < 2 && kRest > 0) {
        constexpr int kRest0 = (kRest + 1) / 2;
        const int q0 = kH3 + (s == 0 ? 0 : kRest0), q1 = s == 0 ? kH3 + kRest0 : kCopies;
        if (rest) {
#pragma unroll
          for (int q = q0; q < q1; ++q) copy(kt + 1, slot ^ 1, q, rest_fill);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (s + 1 < BK / 16) {
#pragma unroll
        for (int i = 0; i < kBlkM; ++i) fa[nxt][i] = OA::read(sa, wm * kWaveM, i, s + 1, lane);
#pragma unroll
        for (int j = 0; j < kBlkN; ++j) fb[nxt][j] = OB::read(sb, wn * kWaveN, j, s + 1, lane);
#pragma unroll
        for (int i = 0; i < kBlkM; ++i)
#pragma unroll
          for (int j = 0; j < kBlkN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[cur][j], fa[cur][i],
                                                                acc[i][j], 0, 0, 0);
        interleave_reads<kMfmaPerStep, kReadsPerStep>();
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (kt + 1 < ktiles) {
          const unsigned char HK_LDS* na = ldsA + (slot ^ 1) * kStageBytes;
          const unsigned char HK_LDS* nb = ldsB + (slot ^ 1) * kStageBytesB;
#pragma unroll
          for (int i = 0; i < kBlkM; ++i) fa[nxt][i] = OA::read(na, wm * kWaveM, i, 0, lane);
#pragma unroll
          for (int j = 0; j < kBlkN; ++j) fb[nxt][j] = OB::read(nb, wn * kWaveN, j, 0, lane);
        }
#pragma unroll
        for (int i = 0; i < kBlkM; ++i)
#pragma unroll
          for (int j = 0; j < kBlkN; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[cur][j], fa[cur][i],
                                                                acc[i][j], 0, 0, 0);
            const int q = i * kBlkN + j;
            if (more && q < kH3) copy(kt + kStages, slot, q, fill);
            // steady state: keep each copy next to its MFMA, so that a wave's copies are spread
            // over the step (the copies are inline asm, which the scheduler does not group)
            if constexpr (STEADY) __builtin_amdgcn_sched_barrier(0);
          }
        if (kH3 > kMfmaPerStep && more) {
#pragma unroll
          for (int q = kMfmaPerStep; q < kH3; ++q) copy(kt + kStages, slot, q, fill);
        }

      }
    }
  };
  // steady state: every k-tile kt < steady has a whole k-tile kt + kStages to copy
  const int steady = ktiles - kStages - (tail ? 1 : 0);
  int kt = 0;
  for (; kt < steady; ++kt) ktile(kt, std::true_type{});
  for (; kt < ktiles; ++kt) ktile(kt, std::false_type{});

  // Epilogue. Lane l holds, for MFMA block (i, j) and quad q, output row
  // wm*128 + 32 i + l % 32 and columns wn*kWaveN + 32 j + 8 q + 4 (l / 32) .. +3; the rows go
  // out through LDS (staged_rows).
  // every wave is done with the LDS ring: its start becomes the waves' staging areas
  __syncthreads();
  if (PARTIAL && fo.C) {
    // one split: fp32 C with alpha, beta and the bias applied here
    store_f32<kWaveN, kBlkM>(acc, area, lane, fo, batch, M, N, wrow0, wcol0);
    return;
  }
  if (PARTIAL) {
    store_partial<kWaveN, kBlkM>(
        acc, area, lane,
        part + (static_cast<int64_t>(split) * (gridDim.z / split_k) + batch) * M * part_pitch(N), M,
        N, wrow0, wcol0);
    return;
  }
  store_bf16<kWaveN, kBlkM, E::kWideStage>(acc, lane, ep, rows, ahead);
}

// One column region: workgroup x takes tile x.
template <bool A_KMAJOR, bool B_KMAJOR, bool PARTIAL, int BNT, int BMT, class E>
__global__ __launch_bounds__(kThreads, 1) void bgemm_tiled(
    int M, int N, int K, E ep, const uint16_t* __restrict__ A, int64_t lda, int64_t sA,
    const uint16_t* __restrict__ B, int64_t ldb, int64_t sB, uint16_t* __restrict__ C,
    int64_t ldc, int64_t sC, int split_k, int k_per_split, float* __restrict__ part,
    hk::F32Out fo, int n_base, int n_end) {
  tile_body<A_KMAJOR, B_KMAJOR, PARTIAL, BNT, BMT>(M, N, K, ep, A, lda, sA, B, ldb, sB, C, ldc,
                                                  sC, split_k, k_per_split, part, fo, n_base,
                                                  n_end, blockIdx.x);
}

// Both column regions in one launch (column_split): workgroups [0, nfull) take the 256-wide
// tiles of columns [0, n_split), the rest the 128-wide tiles of [n_split, N). The 128-wide
// tiles start on CUs as the 256-wide ones finish, with no drain and launch between two
// kernels (about 2% of the 8192 x 5120 x 1280 product on MI355X). tile_coords' XCD grouping
// of the 128-wide region assumes that its first workgroup sits on XCD 0, which holds when
// nfull is a multiple of 8; otherwise only that region's L2 grouping is off, not which tiles
// it covers.
template <bool A_KMAJOR, bool B_KMAJOR, bool PARTIAL, class E>
__global__ __launch_bounds__(kThreads, 1) void bgemm_mixed(
    int M, int N, int K, E ep, const uint16_t* __restrict__ A, int64_t lda, int64_t sA,
    const uint16_t* __restrict__ B, int64_t ldb, int64_t sB, uint16_t* __restrict__ C,
    int64_t ldc, int64_t sC, int split_k, int k_per_split, float* __restrict__ part,
    hk::F32Out fo, int n_split, int nfull) {
  const int wg = blockIdx.x;
  if (wg < nfull)
    tile_body<A_KMAJOR, B_KMAJOR, PARTIAL, 256, 256>(M, N, K, ep, A, lda, sA, B, ldb, sB, C, ldc, sC,
                                               split_k, k_per_split, part, fo, 0, n_split, wg);
  else
    tile_body<A_KMAJOR, B_KMAJOR, PARTIAL, 128, 256>(M, N, K, ep, A, lda, sA, B, ldb, sB, C, ldc, sC,
                                               split_k, k_per_split, part, fo, n_split, N,
                                               wg - nfull);
}

// ---- 256 x 160 tiles on 16 x 16 x 32 MFMAs (A and B both k-major, C = alpha A B^T + ...) ----
// For products whose 256 x 256 tiles leave CUs idle while 256 x 160 tiles fill one round
// (8192 x 1280: 160 tiles of 256 x 256, 215 of 192 x 256, 256 of 256 x 160 on 256 CUs). 160
// columns are 5 blocks of 16, so the waves sit 4 (rows) x 2 (columns), each owning 64 x 80 of C
// as 4 x 5 blocks of v_mfma_f32_16x16x32_bf16. Whole tiles only (M % 256, N % 160, K % 64 == 0).
// LDS: a 3-slot ring of k-tiles (3 x 52 KiB, which only this tile shape fits in 160 KiB), each
// A [256][64 k] then B [160][64 k], bf16, stored as the k-major TileOperand layout (128-byte
// rows, chunk c of row r at c ^ ((r >> 1) & 7)); a 16-row operand block is one ds_read_b128
// per lane (lane l: row l % 16, logical chunk 4 s + l / 16 of k step s), 16 consecutive rows
// per read cycle, conflict-free as in the 32-row form.
// Copies: A is 32 copy instructions per k-tile (4 per wave), B 20: wave w issues B copies w,
// w + 8 and, for w < 4, w + 16, so waves 0-3 issue 7 per k-tile and waves 4-7 issue 6 (their
// vmcnt waits count 6).
// Per k-tile kt (2 k steps of 32): step 0 reads step 1's operands and runs step 0's 20 MFMAs
// with the last copies of tile kt + 2 between them; step 1 waits for this wave's copies of
// tile kt + 1 (tile kt + 2's may still be in flight), meets the others at the barrier (tile
// kt + 1 visible, slot kt % 3 free), reads tile kt + 1's step-0 operands and issues the first
// two copies of tile kt + 3 into slot kt % 3 between its MFMAs. Each copy so has more than a
// k-tile to land and the address unit's work is spread over both steps. On MI355X, 8192 x 1280
// x 5120: 96.2 us on 215 tiles of 192 x 256, 96.7 with these tiles on a 2-slot ring and every
// copy in step 1, 90.1 with 3 slots, 92.8 with 3 slots and every copy in step 1, 87.5 as here.
// The MFMA takes the B block as its first operand, so lane l holds C row l % 16 of its block,
// columns 4 (l / 16) .. + 3.
namespace w160 {
constexpr int kBM = 256, kBN = 160;
constexpr int kStageA = kBM * BK * 2;  // 32 KiB
constexpr int kStageB = kBN * BK * 2;  // 20 KiB
constexpr int kStage = kStageA + kStageB;
constexpr int kRing = 3;
constexpr size_t kLdsBytes = kRing * static_cast<size_t>(kStage);  // 156 KiB
constexpr int kCopiesA = kStageA / 1024 / kWaves;                  // 4
constexpr int kCopiesB = 3;                                        // 20 over 8 waves, see above
constexpr int kCopies = kCopiesA + kCopiesB;                       // 7 (6 for waves 4-7)
constexpr int kFirst = 2;  // copies of a k-tile issued in step 1, the rest in the next step 0
constexpr int kBlkM = 4, kBlkN = 5;                             // 16 x 16 blocks per wave
constexpr int kWaveM = 16 * kBlkM, kWaveN = 16 * kBlkN;         // 64 x 80
constexpr int kPitch = kWaveN * 4 + 16;                         // fp32 staging row, bytes
static_assert(kStageB / 1024 == 20 && kCopiesA * kWaves * 1024 == kStageA, "copy split");
static_assert(kLdsBytes <= 160 * 1024, "fits gfx950's 160 KiB of LDS");
static_assert(kWaves * 16 * kPitch <= static_cast<int>(kLdsBytes), "staging fits");

// LDS byte offset of lane `lane`'s 16 bytes of the 16-row block at row `r0`, k step s (0, 1).
__device__ __forceinline__ int frag16(int r0, int s, int lane) {
  const int row = r0 + (lane & 15);
  const int c = 4 * s + (lane >> 4);
  return row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
}
}  // namespace w160

template <class E>
__global__ __launch_bounds__(kThreads, 1) void bgemm_nt_w160(
    int M, int N, int K, E ep, const uint16_t* __restrict__ A, int64_t lda, int64_t sA,
    const uint16_t* __restrict__ B, int64_t ldb, int64_t sB, uint16_t* __restrict__ C,
    int64_t ldc, int64_t sC) {
  using namespace w160;
  using OK = TileOperand<true>;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  unsigned char HK_LDS* lds = (unsigned char HK_LDS*)lds_raw;
  const int batch = blockIdx.z;
  const int tiles_m = M / kBM, tiles_n = N / kBN;
  int tm, tn;
  tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * kBM, n0 = tn * kBN;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  const unsigned char* gA = reinterpret_cast<const unsigned char*>(
      A + static_cast<int64_t>(batch) * sA + static_cast<int64_t>(m0) * lda);
  const unsigned char* gB = reinterpret_cast<const unsigned char*>(
      B + static_cast<int64_t>(batch) * sB + static_cast<int64_t>(n0) * ldb);
  // per-lane source offsets (bytes, from the tile base at k = 0) and LDS destinations of this
  // wave's copies; rows stay inside the tile (whole tiles), so no clamping is needed
  int off[kCopies];
  unsigned dst[kCopies];
  const unsigned lds_addr = static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds));
#pragma unroll
  for (int q = 0; q < kCopies; ++q) {
    int row, k;
    if (q < kCopiesA) {
      const int ii = wave * kCopiesA + q;
      OK::source(ii, lane, row, k);
      off[q] = static_cast<int>(OK::byte_offset(row, k, lda));
      dst[q] = lds_addr + ii * 1024;
    } else {
      int ii = wave + 8 * (q - kCopiesA);
      if (ii >= 20) ii = wave + 8;  // waves 4-7 have no third B copy (never issued)
      OK::source(ii, lane, row, k);
      off[q] = static_cast<int>(OK::byte_offset(row, k, ldb));
      dst[q] = lds_addr + kStageA + ii * 1024;
    }
  }
  const int ktiles = K / BK;
  const bool six = wave >= 4;  // waves 4-7 issue 6 copies per k-tile
  auto copy = [&](int kt, int slot, int q) {
    if (q == kCopies - 1 && six) return;
    const unsigned char* base = (q < kCopiesA ? gA : gB) + kt * (2 * BK);
    copy16_to_lds(base, off[q], dst[q] + slot * kStage);
  };
  // wait until at most n k-tiles of this wave's copies are in flight
  auto wait_tiles = [&](int n) {
    if (n == 2) {
      if (six) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * kCopies - 2) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * kCopies) : "memory");
    } else if (n == 1) {
      if (six) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kCopies - 1) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kCopies) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
  };

  f32x4_t acc[kBlkM][kBlkN];
#pragma unroll
  for (int i = 0; i < kBlkM; ++i)
#pragma unroll
    for (int j = 0; j < kBlkN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int p = 0; p < kRing; ++p)
    if (p < ktiles) {
#pragma unroll
      for (int q = 0; q < kCopies; ++q) copy(p, p, q);
    }
  wait_tiles(ktiles >= 3 ? 2 : ktiles - 1);  // k-tile 0 landed
  __builtin_amdgcn_s_barrier();

  bf16x8_t fa[2][kBlkM], fb[2][kBlkN];
  auto read_ops = [&](int slot, int s, int buf) {
    const unsigned char HK_LDS* sa = lds + slot * kStage;
    const unsigned char HK_LDS* sb = sa + kStageA;
#pragma unroll
    for (int i = 0; i < kBlkM; ++i)
      fa[buf][i] = *reinterpret_cast<const bf16x8_t HK_LDS*>(
          sa + frag16(wm * kWaveM + 16 * i, s, lane));
#pragma unroll
    for (int j = 0; j < kBlkN; ++j)
      fb[buf][j] = *reinterpret_cast<const bf16x8_t HK_LDS*>(
          sb + frag16(wn * kWaveN + 16 * j, s, lane));
  };
  read_ops(0, 0, 0);
  int slot = 0;
  for (int kt = 0; kt < ktiles; ++kt) {
    const int nslot = slot == kRing - 1 ? 0 : slot + 1;
    const int slot2 = nslot == kRing - 1 ? 0 : nslot + 1;
    // step 0: operands of step 1 read while step 0 multiplies, with the rest of tile kt + 2's
    // copies between the MFMAs (its first kFirst went out in tile kt - 1's step 1; tile 2's
    // all in the prologue)
    const bool rest = kt >= 1 && kt + 2 < ktiles;
    read_ops(slot, 1, 1);
#pragma unroll
    for (int i = 0; i < kBlkM; ++i)
#pragma unroll
      for (int j = 0; j < kBlkN; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[0][j], fa[0][i], acc[i][j], 0, 0,
                                                            0);
        const int q = kFirst + 2 * (i * kBlkN + j);
        if (q < kCopies && rest) copy(kt + 2, slot2, q);
        if (q + 1 < kCopies && rest) copy(kt + 2, slot2, q + 1);
      }
    // step 1: tile kt + 1 landed (tile kt + 2's copies may still be in flight), slot free
    wait_tiles(kt + 2 < ktiles ? 1 : 0);
    __builtin_amdgcn_s_barrier();
    if (kt + 1 < ktiles) read_ops(nslot, 0, 0);
    const bool more = kt + kRing < ktiles;
#pragma unroll
    for (int i = 0; i < kBlkM; ++i)
#pragma unroll
      for (int j = 0; j < kBlkN; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[1][j], fa[1][i], acc[i][j], 0, 0,
                                                            0);
        const int q = i * kBlkN + j;
        if (q < kFirst && more) copy(kt + kRing, slot, q);
        __builtin_amdgcn_sched_barrier(0);
      }
    slot = nslot;
  }

  // Epilogue: each wave stages one 16-row block row (16 x 80 fp32) in its own LDS area and
  // reads it back as 8 consecutive columns per lane (10 lanes per row, 6 rows per pass), so the
  // bf16 outputs go out 16 bytes per lane in row segments.
  __syncthreads();
  unsigned char HK_LDS* area = lds + wave * (16 * kPitch);
  const int wrow0 = m0 + wm * kWaveM, wcol0 = n0 + wn * kWaveN;
  auto emit = [&](auto&& out) {
#pragma unroll
    for (int i = 0; i < kBlkM; ++i) {
#pragma unroll
      for (int j = 0; j < kBlkN; ++j)
        *reinterpret_cast<f32x4_t HK_LDS*>(area + (lane & 15) * kPitch +
                                          (16 * j + 4 * (lane >> 4)) * 4) = acc[i][j];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const int rr = 6 * p + lane / 10, cc = (lane % 10) * 8;
        out.pass(3 * i + p);
        if (lane < 60 && rr < 16) {
          const f32x4_t a = *reinterpret_cast<const f32x4_t HK_LDS*>(area + rr * kPitch + cc * 4);
          const f32x4_t b =
              *reinterpret_cast<const f32x4_t HK_LDS*>(area + rr * kPitch + cc * 4 + 16);
          out(16 * i + rr, cc, a, b);
        }
      }
    }
  };
  emit_rows<kWaveN / 8, 16, 3 * kBlkM>(
      ep, WaveRows{C, ldc, sC, batch, M, N, wrow0, wcol0, 4 * tm + wm, area}, lane, emit);
}

// BNT 256 or 128: one column region (bgemm_tiled); BNT 0: both regions (bgemm_mixed), with
// n_base = n_split and n_end = nfull.
template <bool AK, bool BKM, bool P, int BNT, int BMT, class E>
hipError_t launch_tiled(dim3 grid, hipStream_t stream, int M, int N, int K, const E& ep,
                        const uint16_t* A, int64_t lda, int64_t sA, const uint16_t* B,
                        int64_t ldb, int64_t sB, uint16_t* C, int64_t ldc,
                        int64_t sC, int split_k, int kps, float* part, const hk::F32Out& fo,
                        int n_base, int n_end) {
  static_assert(BNT != 0 || BMT == 256, "the mixed-width launch uses 256-row tiles");
  constexpr size_t kLds = TileN<BNT == 0 ? 256 : BNT, BMT>::lds_bytes(E::kWideStage);
  static_assert(kLds <= 160 * 1024, "fits gfx950's 160 KiB of LDS");
  const void* fn;
  if constexpr (BNT == 0) fn = reinterpret_cast<const void*>(&bgemm_mixed<AK, BKM, P, E>);
  else fn = reinterpret_cast<const void*>(&bgemm_tiled<AK, BKM, P, BNT, BMT, E>);
  static std::once_flag once;
  static hipError_t attr_status = hipSuccess;
  std::call_once(once, [fn] {
    attr_status = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(kLds));
  });
  HK_RETURN_IF_ERROR(attr_status);
  if constexpr (BNT == 0)
    hipLaunchKernelGGL((bgemm_mixed<AK, BKM, P, E>), grid, dim3(kThreads), kLds, stream, M, N, K, ep,
                       A, lda, sA, B, ldb, sB, C, ldc, sC, split_k, kps, part, fo, n_base, n_end);
  else
    hipLaunchKernelGGL((bgemm_tiled<AK, BKM, P, BNT, BMT, E>), grid, dim3(kThreads), kLds, stream, M,
                       N, K, ep, A, lda, sA, B, ldb, sB, C, ldc, sC, split_k, kps, part, fo,
                       n_base, n_end);
  return hk::launch_status();
}

template <bool P, int BNT, int BMT, class E>
hipError_t dispatch_layout(bool ta, bool tb, dim3 grid, hipStream_t stream, int M, int N, int K,
                           const E& ep, const uint16_t* A, int64_t lda, int64_t sA,
                           const uint16_t* B, int64_t ldb, int64_t sB, uint16_t* C,
                           int64_t ldc, int64_t sC, int split_k, int kps, float* part,
                           const hk::F32Out& fo, int n_base, int n_end) {
  // A is k-major unless transposed; B is k-major only when transposed.
  if (!ta && !tb)
    return launch_tiled<true, false, P, BNT, BMT>(grid, stream, M, N, K, ep, A, lda, sA, B, ldb,
                                                  sB, C, ldc, sC, split_k, kps, part, fo, n_base,
                                                  n_end);
  if (!ta && tb)
    return launch_tiled<true, true, P, BNT, BMT>(grid, stream, M, N, K, ep, A, lda, sA, B, ldb,
                                                 sB, C, ldc, sC, split_k, kps, part, fo, n_base,
                                                 n_end);
  if constexpr (BMT != 256) {
    return hipErrorInvalidValue;  // row_tile keeps 256-row tiles for an M-major A
  } else {
    if (ta && !tb)
      return launch_tiled<false, false, P, BNT, BMT>(grid, stream, M, N, K, ep, A, lda, sA, B, ldb,
                                                sB, C, ldc, sC, split_k, kps, part, fo, n_base,
                                                n_end);
    return launch_tiled<false, true, P, BNT, BMT>(grid, stream, M, N, K, ep, A, lda, sA, B, ldb, sB,
                                             C, ldc, sC, split_k, kps, part, fo, n_base, n_end);
  }
}

// Columns [0, n_split) of C take 256 x 256 tiles and [n_split, N) 256 x 128 tiles. One
// workgroup runs per CU (its LDS ring is 128 KiB), so a launch takes ceil(tiles / CUs) rounds;
// when the last round of 256-wide tiles would be partly empty, the trailing tile columns run
// as twice as many 128-wide tiles, which fill a round of half the length (8192 x 5120: 640
// tiles are 3 rounds, 512 tiles + 256 half tiles are 2.5). Costs in full-tile rounds, a half
// tile counted as 0.55 of one; a split is taken only if it saves at least 3%. Returns N for
// no split.
inline int column_split(int M, int N, int work_per_tile) {
  const int64_t cus = hk::device_cu_count();
  const int64_t tiles_m = (M + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
  auto rounds = [&](int64_t tiles) { return static_cast<double>(hk::ceil_div(tiles * work_per_tile, cus)); };
  const double whole = rounds(tiles_m * tiles_n);
  double best = whole;
  int64_t best_c = 0;
  for (int64_t c = 1; c <= tiles_n; ++c) {
    const int64_t n_split = (tiles_n - c) * BN;
    const double cost = rounds(tiles_m * (tiles_n - c)) +
                        0.55 * rounds(tiles_m * hk::ceil_div(N - n_split, int64_t{128}));
    if (cost < best) {
      best = cost;
      best_c = c;
    }
  }
  if (best_c == 0 || best > 0.97 * whole) return N;
  return static_cast<int>((tiles_n - best_c) * BN);
}

// Rows per tile. 256 x 256 tiles that do not fill one round of the CUs leave the rest idle
// (8192 x 1280: 160 tiles on 256 CUs). 192-row tiles cut each workgroup's work to 3/4 and
// raise the tile count (215 there), so they are used when their rounds, each costed 0.75 of a
// 256-row round, save at least 10%. They need a k-major A (the M-major LDS layout holds 256 or
// 128 rows) and a single k split.
inline int row_tile(bool ta, int M, int N, int grid_z, int split_k) {
  if (ta || split_k != 1) return 256;
  const int64_t cus = hk::device_cu_count();
  const int64_t tiles_n = (N + BN - 1) / BN;
  const int64_t t256 = static_cast<int64_t>((M + 255) / 256) * tiles_n * grid_z;
  if (t256 >= cus) return 256;
  const int64_t t192 = static_cast<int64_t>((M + 191) / 192) * tiles_n * grid_z;
  return 0.75 * static_cast<double>(hk::ceil_div(t192, cus)) <= 0.9 ? 192 : 256;
}

// 256 x 160 tiles (bgemm_nt_w160): both operands k-major, one k split, bf16 C, whole tiles,
// when 256 x 256 tiles leave CUs idle and 256 x 160 tiles fit one round. Each such workgroup
// carries 5/8 of a 256 x 256 tile's work (3/4 for the 192-row tiles, which then give way).
inline bool w160_plan(bool ta, bool tb, int M, int N, int K, int grid_z, int split_k) {
  if (ta || !tb || split_k != 1) return false;
  if (M % w160::kBM != 0 || N % w160::kBN != 0 || K % BK != 0) return false;
  const int64_t cus = hk::device_cu_count();
  const int64_t t256 = static_cast<int64_t>((M + 255) / 256) * ((N + BN - 1) / BN) * grid_z;
  const int64_t t160 = static_cast<int64_t>(M / w160::kBM) * (N / w160::kBN) * grid_z;
  return t256 < cus && t160 <= cus;
}

template <class E>
hipError_t launch_w160(int grid_z, hipStream_t stream, int M, int N, int K, const E& ep,
                       const uint16_t* A, int64_t lda, int64_t sA, const uint16_t* B,
                       int64_t ldb, int64_t sB, uint16_t* C, int64_t ldc, int64_t sC) {
  static std::once_flag once;
  static hipError_t attr_status = hipSuccess;
  std::call_once(once, [] {
    attr_status = hipFuncSetAttribute(reinterpret_cast<const void*>(&bgemm_nt_w160<E>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(w160::kLdsBytes));
  });
  HK_RETURN_IF_ERROR(attr_status);
  const dim3 grid(static_cast<unsigned>((M / w160::kBM) * (N / w160::kBN)), 1, grid_z);
  hipLaunchKernelGGL(bgemm_nt_w160<E>, grid, dim3(kThreads), w160::kLdsBytes, stream, M, N, K, ep,
                     A, lda, sA, B, ldb, sB, C, ldc, sC);
  return hk::launch_status();
}

// The product over its column regions (column_split), in one launch; grid.z covers batches
// and splits. A split into partials (P with split_k > 1) keeps one region.
template <bool P, class E>
hipError_t run_regions(bool ta, bool tb, int grid_z, hipStream_t stream, int M, int N, int K,
                       const E& ep, const uint16_t* A, int64_t lda, int64_t sA,
                       const uint16_t* B, int64_t ldb, int64_t sB, uint16_t* C, int64_t ldc,
                       int64_t sC, int split_k, int kps, float* part, const hk::F32Out& fo) {
  if constexpr (!P) {
    if (w160_plan(ta, tb, M, N, K, grid_z, split_k))
      return launch_w160(grid_z, stream, M, N, K, ep, A, lda, sA, B, ldb, sB, C, ldc, sC);
  }
  if (row_tile(ta, M, N, grid_z, split_k) == 192) {
    const int64_t tiles = static_cast<int64_t>((M + 191) / 192) * ((N + BN - 1) / BN);
    const dim3 grid(static_cast<unsigned>(tiles), 1, grid_z);
    return dispatch_layout<P, 256, 192>(ta, tb, grid, stream, M, N, K, ep, A, lda, sA, B, ldb, sB,
                                        C, ldc, sC, split_k, kps, part, fo, 0, N);
  }
  const int64_t tiles_m = (M + BM - 1) / BM;
  const int n_split = split_k == 1 ? column_split(M, N, grid_z) : N;
  const int64_t nfull = tiles_m * ((n_split + BN - 1) / BN);
  const int64_t nhalf = tiles_m * hk::ceil_div(N - n_split, int64_t{128});
  if (nhalf == 0) {
    const dim3 grid(static_cast<unsigned>(nfull), 1, grid_z);
    return dispatch_layout<P, 256, 256>(ta, tb, grid, stream, M, N, K, ep, A, lda, sA, B, ldb, sB, C,
                                   ldc, sC, split_k, kps, part, fo, 0, N);
  }
  if (nfull == 0) {
    const dim3 grid(static_cast<unsigned>(nhalf), 1, grid_z);
    return dispatch_layout<P, 128, 256>(ta, tb, grid, stream, M, N, K, ep, A, lda, sA, B, ldb, sB, C,
                                   ldc, sC, split_k, kps, part, fo, 0, N);
  }
  const dim3 grid(static_cast<unsigned>(nfull + nhalf), 1, grid_z);
  return dispatch_layout<P, 0, 256>(ta, tb, grid, stream, M, N, K, ep, A, lda, sA, B, ldb, sB, C,
                               ldc, sC, split_k, kps, part, fo, n_split,
                               static_cast<int>(nfull));
}

}  // namespace gemm
}  // namespace hk

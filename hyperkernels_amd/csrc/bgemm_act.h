// bgemm_act.h - the epilogue of the BF16 GEMM's tiles with bias, activation and residual, and the one of
// its backward product (bgemm_act.hip).
#pragma once

#include "activation.h"
#include "bgemm_tile.h"

namespace hk {
namespace gemm {

// forward:  z = alpha acc + bias[col], stored in bf16 where z is not NULL; C = act(z) + residual
// backward: d = alpha acc act'(z); C = d, and the column sums of d over each wave's rows where sums is
//           not NULL: row (batch, wave row) of [batch][sum_rows][pitch]
// Everything is fp32 until C and z are rounded, once each, to nearest even.
struct ActEpi {
  float alpha;
  Activation act;
  bool backward, ragged;  // ragged: C, z or residual are no whole number of aligned 16-byte vectors
  const uint16_t* bias;
  int64_t sBias;
  const uint16_t* residual;
  int64_t ldr, sR;
  uint16_t* z;  // read in the backward pass
  int64_t ldz, sZ;
  float* sums;
  int sum_rows, pitch;
  static constexpr int kWideAhead = 4;  // passes whose inputs are in flight there
  static constexpr bool kShareRows = true;
  static constexpr int kWideStage = 2;  // block rows that a wave of the 256-wide tiles stages at a time
};

// Eight bf16 of a row, n of them inside it. The whole vectors of rows that are not ragged are aligned, and
// read once: non-temporal (8192 x 1280 -> 5120: residual and GELU' 1 us less).
template <bool RAGGED>
__device__ __forceinline__ uint4 load_row8(const uint16_t* p, int n) {
  if (!RAGGED) return ld_nt(reinterpret_cast<const uint4*>(p));
  uint32_t w[4];
  if (n == 8) {
    __builtin_memcpy(w, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = (2 * e < n ? p[2 * e] : 0u) |
             (2 * e + 1 < n ? static_cast<uint32_t>(p[2 * e + 1]) << 16 : 0u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Stores are non-temporal like those of the plain product: nothing here is read again by this one (GELU with
// its preact: 117.7 us; both outputs stored through the caches 131.4, preact alone 121.6).
template <bool RAGGED>
__device__ __forceinline__ void store_row8(uint16_t* p, int n, const float (&f)[8]) {
  const uint4 v = BF16::pack(f);
  if (!RAGGED) {
    st_nt(reinterpret_cast<uint4*>(p), v);
  } else if (n == 8) {
    __builtin_memcpy(p, &v, 16);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
  }
}

// What one lane reads beside the sums: the residual or, in the backward pass, z, from column col of row 0 on;
// NULL where there is neither.
struct ActInput {
  const uint16_t* p;
  int64_t ld;
  __device__ ActInput(const ActEpi& ep, const WaveRows& w, int col) {
    const uint16_t* base = ep.backward ? (ep.act.kind == HK_ACT_NONE ? nullptr : ep.z) : ep.residual;
    ld = ep.backward ? ep.ldz : ep.ldr;
    p = base ? base + w.batch * (ep.backward ? ep.sZ : ep.sR) + col : nullptr;
  }
};
__device__ __forceinline__ uint4 load_bias8(const ActEpi& ep, const WaveRows& w, int col, int n) {
  return !ep.backward && ep.bias && n > 0
             ? load_row8<true>(ep.bias + w.batch * ep.sBias + col, n)
             : make_uint4(0, 0, 0, 0);
}
// The epilogue of one lane: the 8 columns from col on of several rows, so the bias and the column sums stay
// in registers. What it reads beside the sums (residual, or z in the backward pass) is fetched ahead
// of the row's turn.
template <bool RAGGED>
struct ActLane {
  const ActEpi& ep;
  const WaveRows& w;
  int col, n;          // n: columns inside N, 0 for none
  ActInput in;
  float reg[8];        // forward: bias, backward: column sums
  __device__ ActLane(const ActEpi& e, const WaveRows& rows, int cc, const uint4& bias)
      : ep(e), w(rows), col(rows.wcol0 + cc), n(min(8, max(0, rows.N - col))), in(e, rows, col) {
    BF16::unpack(bias, reg);  // zeros in the backward pass
  }
  __device__ ActLane(const ActEpi& e, const WaveRows& rows, int cc)
      : ActLane(e, rows, cc,
                load_bias8(e, rows, rows.wcol0 + cc, min(8, max(0, rows.N - rows.wcol0 - cc)))) {}
  __device__ bool has(int row) const { return row < w.M && n > 0; }
  __device__ uint4 fetch(int row) const {
    return in.p && has(row) ? load_row8<RAGGED>(in.p + row * in.ld, n) : make_uint4(0, 0, 0, 0);
  }
  __device__ void row(int row, const uint4& extra, const f32x4_t& a, const f32x4_t& b) {
    if (!has(row)) return;
    // one VALU slot of an element is 1 us of 8192 x 5120 outputs: nothing is done that a call does not ask for
    float v[8], x[8];
    if (ep.backward) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < 4 ? a[e] : b[e - 4];
      if (ep.alpha != 1.0f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= ep.alpha;
      }
      if (in.p) {
        BF16::unpack(extra, x);
        scale_by_grad(ep.act, x, v);
      }
      if (ep.sums) {
#pragma unroll
        for (int e = 0; e < 8; ++e) reg[e] += v[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(ep.alpha, e < 4 ? a[e] : b[e - 4], reg[e]);
      if (ep.z) store_row8<RAGGED>(ep.z + w.batch * ep.sZ + row * ep.ldz + col, n, v);
      activate(ep.act, v);
      if (in.p) {
        BF16::unpack(extra, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += x[e];
      }
    }
    store_row8<RAGGED>(w.C + w.batch * w.sC + row * w.ldc + col, n, v);
  }
  // Adds the lanes' column sums of one wave, in a fixed order, and stores its row of them. The LPR lanes
  // of a row hold 8 columns each; a wave has 64 / LPR rows, the last lanes idle where LPR is no power
  // of two.
  template <int LPR>
  __device__ void store_sums(int lane) {
    if (!ep.sums || w.wrow0 >= w.M) return;  // a wave without rows is not counted in sum_rows
    const int cc = (lane % LPR) * 8;
    if constexpr ((LPR & (LPR - 1)) == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int step = LPR; step < HK_WAVE; step *= 2) reg[e] += __shfl_xor(reg[e], step);
    } else {
      float HK_LDS* area = reinterpret_cast<float HK_LDS*>(w.area);
      constexpr int kRows = HK_WAVE / LPR;
      if (lane < kRows * LPR) {
#pragma unroll
        for (int e = 0; e < 8; ++e) area[(lane / LPR) * (8 * LPR) + cc + e] = reg[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        reg[e] = 0.f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) reg[e] += area[r * (8 * LPR) + cc + e];
      }
    }
    if (lane < LPR && n > 0) {
      // pitch is a multiple of 8: a lane's columns past N lie in its padding
      float4* dst = reinterpret_cast<float4*>(
          ep.sums + (static_cast<int64_t>(w.batch) * ep.sum_rows + w.wave_row) * ep.pitch + col);
      dst[0] = make_float4(reg[0], reg[1], reg[2], reg[3]);
      dst[1] = make_float4(reg[4], reg[5], reg[6], reg[7]);
    }
  }
};

// The rows of a wave are worked on two passes of the wave at a time, with the inputs of DEPTH in flight. Those of
// the first, and the bias, are read before the k loop: behind it they were a latency of memory that
// nothing hid (8192 x 1280 -> 5120, bias: 103.5 us with the plain epilogue at 101.1, now the same to
// 0.4). One workgroup runs on a CU, so all tiles of a round read their inputs at once: two passes in
// flight a wave are 16 KiB a CU, too little for the memory's latency, eight do not fit the registers
// (8192 x 1280 -> 5120, residual: two 123, four 116, six 117, eight 126 us; GELU' 128, 125, 125, 134).
template <int kWaveN, int DEPTH>
struct ActAhead {
  static constexpr int LPR = kWaveN / 8;  // lanes per row
  static constexpr int RPP = 64 / LPR;    // rows per pass
  uint4 bias, first[DEPTH];
};
template <int kWaveN, int DEPTH>
__device__ __forceinline__ ActAhead<kWaveN, DEPTH> rows_ahead(const ActEpi& ep, const WaveRows& w,
                                                              int lane) {
  using A = ActAhead<kWaveN, DEPTH>;
  A a;
  const int col = w.wcol0 + (lane % A::LPR) * 8, n = min(8, max(0, w.N - col));
  const ActInput in(ep, w, col);
  a.bias = load_bias8(ep, w, col, n);
#pragma unroll
  for (int p = 0; p < DEPTH; ++p) {
    const int row = w.wrow0 + p * A::RPP + lane / A::LPR;
    a.first[p] = make_uint4(0, 0, 0, 0);
    if (in.p && row < w.M && n > 0)
      a.first[p] = ep.ragged ? load_row8<true>(in.p + row * in.ld, n)
                             : load_row8<false>(in.p + row * in.ld, n);
  }
  return a;
}

// As staged_rows: 32-row MFMA block rows through LDS, kStage of them at a time (kStage x 32 rows of the wave's
// staging area). The code of a row is long, so the blocks and passes are loops: the accumulators of a
// block are picked by uniform branches, and the next passes' reads are in flight while two are worked on.
template <int kWaveN, int kBlkM, bool RAGGED, int kStage, int DEPTH>
__device__ __forceinline__ void act_rows(const f32x16_t (&acc)[kBlkM][kWaveN / 32], int lane,
                                         const ActEpi& ep, const WaveRows& w,
                                         const ActAhead<kWaveN, DEPTH>& ahead) {
  constexpr int kBlkN = kWaveN / 32;
  constexpr int P = kWaveN * 4 + 16;  // staging pitch (bytes)
  constexpr int LPR = ActAhead<kWaveN, DEPTH>::LPR, RPP = ActAhead<kWaveN, DEPTH>::RPP;
  const int r = lane & 31, h = lane >> 5;
  const int rr0 = lane / LPR, cc = (lane % LPR) * 8;
  ActLane<RAGGED> out(ep, w, cc, ahead.bias);
  uint4 next[DEPTH];
#pragma unroll
  for (int p = 0; p < DEPTH; ++p) next[p] = ahead.first[p];
#pragma unroll 1
  for (int i = 0; i < kBlkM; i += kStage) {
#pragma unroll
    for (int ii = 0; ii < kBlkM; ++ii)
      if (i == ii - ii % kStage) {
#pragma unroll
        for (int j = 0; j < kBlkN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4_t HK_LDS*>(w.area + (32 * (ii % kStage) + r) * P +
                                              (32 * j + 8 * q + 4 * h) * 4) =
                f32x4_t{acc[ii][j][4 * q], acc[ii][j][4 * q + 1], acc[ii][j][4 * q + 2],
                        acc[ii][j][4 * q + 3]};
      }
    const int end = 32 * min(kBlkM - i, kStage);
#pragma unroll 1
    for (int s = 0; s < end; s += 2 * RPP) {
      f32x4_t a[2], b[2];
      uint4 extra[2];
      const int row = w.wrow0 + 32 * i + s + rr0;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const unsigned char HK_LDS* at = w.area + (s + p * RPP + rr0) * P + cc * 4;
        a[p] = *reinterpret_cast<const f32x4_t HK_LDS*>(at);
        b[p] = *reinterpret_cast<const f32x4_t HK_LDS*>(at + 16);
        extra[p] = next[p];
      }
#pragma unroll
      for (int p = 0; p + 2 < DEPTH; ++p) next[p] = next[p + 2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        // not the rows behind the wave's last ones
        const int at = 32 * i + s + (DEPTH + p) * RPP;
        if (at < 32 * kBlkM) next[DEPTH - 2 + p] = out.fetch(w.wrow0 + at + rr0);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) out.row(row + p * RPP, extra[p], a[p], b[p]);
    }
  }
  if (ep.backward) out.template store_sums<LPR>(lane);
}
template <int kWaveN, int kBlkM, int kStage, int DEPTH>
__device__ __forceinline__ void store_bf16(const f32x16_t (&acc)[kBlkM][kWaveN / 32], int lane,
                                           const ActEpi& ep, const WaveRows& w,
                                           const ActAhead<kWaveN, DEPTH>& ahead) {
  if (ep.ragged) act_rows<kWaveN, kBlkM, true, kStage, DEPTH>(acc, lane, ep, w, ahead);
  else act_rows<kWaveN, kBlkM, false, kStage, DEPTH>(acc, lane, ep, w, ahead);
}

// Tiles of several k groups T::KG: every wave stages its sums, and those of a group, wave `wave` of T::kGroupWaves,
// then take T::kShareM of the rows that its tile part has in all groups, add the sums in group order and work
// on them. With one group at work and the others at their end it took longer (2048 x 2048 -> 2048 with bias,
// GELU and residual 25.9 us, now 24.4; 1024 x 4096 -> 1024 18.2 and 16.6; 512 x 768 -> 768 7.2 and 6.9 in a
// graph). w: the rows of the share; the inputs of all of its passes are ahead.
template <class T, bool RAGGED>
__device__ __forceinline__ void act_shared(const unsigned char HK_LDS* lds, int group, int wave, int lane,
                                           const ActEpi& ep, const WaveRows& w,
                                           const ActAhead<T::kWaveN, T::kSharePasses>& ahead) {
  constexpr int LPR = T::kWaveN / 8, RPP = 64 / LPR, NP = T::kSharePasses;
  constexpr int kAtOnce = NP > 1 ? 2 : 1;
  ActLane<RAGGED> out(ep, w, (lane % LPR) * 8, ahead.bias);
  uint4 next[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) next[p] = ahead.first[p];
#pragma unroll 1
  for (int s = 0; s < T::kShareM; s += kAtOnce * RPP) {
    f32x4_t a[kAtOnce], b[kAtOnce];
    uint4 extra[kAtOnce];
    const int row = s + lane / LPR;
#pragma unroll
    for (int p = 0; p < kAtOnce; ++p) {
      const unsigned char HK_LDS* at = lds + wave * T::kRowsArea +
                                       (group * T::kShareM + row + p * RPP) * T::kRowsPitch +
                                       (lane % LPR) * 32;
      a[p] = *reinterpret_cast<const f32x4_t HK_LDS*>(at);
      b[p] = *reinterpret_cast<const f32x4_t HK_LDS*>(at + 16);
#pragma unroll
      for (int grp = 1; grp < T::KG; ++grp) {
        at += T::kGroupWaves * T::kRowsArea;
        a[p] += *reinterpret_cast<const f32x4_t HK_LDS*>(at);
        b[p] += *reinterpret_cast<const f32x4_t HK_LDS*>(at + 16);
      }
      extra[p] = next[p];
    }
#pragma unroll
    for (int p = 0; p + kAtOnce < NP; ++p) next[p] = next[p + kAtOnce];
#pragma unroll
    for (int p = 0; p < kAtOnce; ++p) out.row(w.wrow0 + row + p * RPP, extra[p], a[p], b[p]);
  }
  if (ep.backward) out.template store_sums<LPR>(lane);
}
template <class T>
__device__ __forceinline__ void store_shared(const f32x16_t (&acc)[T::kBlkM][T::kBlkN],
                                             unsigned char HK_LDS* lds, int group, int wave, int lane,
                                             const ActEpi& ep, const WaveRows& w,
                                             const ActAhead<T::kWaveN, T::kSharePasses>& ahead) {
  const int r = lane & 31, h = lane >> 5;
  unsigned char HK_LDS* area = lds + (group * T::kGroupWaves + wave) * T::kRowsArea;
#pragma unroll
  for (int i = 0; i < T::kBlkM; ++i)
#pragma unroll
    for (int j = 0; j < T::kBlkN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4_t HK_LDS*>(area + (32 * i + r) * T::kRowsPitch +
                                          (32 * j + 8 * q + 4 * h) * 4) =
            f32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                    acc[i][j][4 * q + 3]};
  __syncthreads();
  if (group >= T::kShares) return;
  if (ep.ragged) act_shared<T, true>(lds, group, wave, lane, ep, w, ahead);
  else act_shared<T, false>(lds, group, wave, lane, ep, w, ahead);
}

// The same where the caller hands out the rows itself: the inputs of four passes are in flight.
template <int LPR, int BLOCK, int PASSES, bool RAGGED>
struct ActPasses {
  static constexpr int RPP = HK_WAVE / LPR, kPerBlock = (BLOCK + RPP - 1) / RPP;
  ActLane<RAGGED> lane_out;
  int row0;  // of the lane in a pass, in a block
  uint4 extra, next[4];
  __device__ ActPasses(const ActEpi& ep, const WaveRows& w, int lane)
      : lane_out(ep, w, (lane % LPR) * 8), row0(lane / LPR) {
#pragma unroll
    for (int n = 0; n < 4; ++n) next[n] = fetch(n);
  }
  __device__ uint4 fetch(int n) const {
    const int row = row0 + RPP * (n % kPerBlock);  // not those behind the block's and the wave's last ones
    return n < PASSES && row < BLOCK ? lane_out.fetch(lane_out.w.wrow0 + BLOCK * (n / kPerBlock) + row)
                                     : make_uint4(0, 0, 0, 0);
  }
  __device__ void pass(int n) {
    extra = next[n % 4];
    next[n % 4] = fetch(n + 4);
  }
  __device__ void operator()(int rr, int, const f32x4_t& a, const f32x4_t& b) {
    lane_out.row(lane_out.w.wrow0 + rr, extra, a, b);
  }
};
template <int LPR, int BLOCK, int PASSES, bool RAGGED, class Emit>
__device__ __forceinline__ void emit_act(const ActEpi& ep, const WaveRows& w, int lane, Emit&& emit) {
  ActPasses<LPR, BLOCK, PASSES, RAGGED> out(ep, w, lane);
  emit(out);
  if (ep.backward) out.lane_out.template store_sums<LPR>(lane);
}
template <int LPR, int BLOCK, int PASSES, class Emit>
__device__ __forceinline__ void emit_rows(const ActEpi& ep, const WaveRows& w, int lane,
                                          Emit&& emit) {
  if (ep.ragged) emit_act<LPR, BLOCK, PASSES, true>(ep, w, lane, emit);
  else emit_act<LPR, BLOCK, PASSES, false>(ep, w, lane, emit);
}

}  // namespace gemm
}  // namespace hk

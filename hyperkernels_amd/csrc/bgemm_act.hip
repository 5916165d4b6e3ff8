// bgemm_act.hip - the BF16 GEMM with bias, activation and residual in its epilogue, and the product of its
// backward pass:
//   forward   z = alpha op(A) op(B) + bias[col],  preact = bf16(z),  C = act(z) + residual
//   backward  d = alpha op(A) op(B) act'(preact),  C = d,  dbias[col] (+)= the sum of d over rows
// A feed-forward block's hidden layer is the first with A its input and B its weights, and d the
// second with A the gradient behind the next layer and B that layer's weights: what would be passes
// over [tokens, hidden] of their own (bias and activation 2 reads or writes of 2 bytes an element, the
// gradient 3, the bias gradient 1) are part of the product's stores.
//
// The products are those of bgemm.hip and bgemm_flex.hip, on the same tiles by the same choice, with the
// epilogue of bgemm_act.h in the tiles' place of the plain one; a product of one row has kernels of its own
// (below). Where K is split, a second kernel adds the fp32 partials in split order and applies the
// epilogue. The bias gradient is summed in fp32 from the values before their rounding: over the rows of
// a wave in registers, over the waves of the grid by a further kernel, in a fixed order.
#include <algorithm>

#include "bgemm_act_tiles.h"
#include "bgemm_plan.h"
#include "bgemm_wide.h"
#include "hk_overlap.h"

namespace {

using namespace hk::gemm;

constexpr int kMaxGridZ = 65535;
constexpr int kMaxSide = INT32_MAX - 0xFFFF;  // extents to which whole tiles can be added

// One element's epilogue, for the kernels that hold one at a time, and what it reads beside the sum: bias and
// residual, or z in the backward pass.
struct ActElement {
  uint16_t bias, other;  // as stored: a conversion would wait for the load
};
__device__ __forceinline__ ActElement act_inputs(const ActEpi& ep, int b, int64_t row, int col) {
  ActElement in{0, 0};
  if (ep.backward) {
    if (ep.act.kind != HK_ACT_NONE) in.other = ep.z[b * ep.sZ + row * ep.ldz + col];
  } else {
    if (ep.bias) in.bias = ep.bias[b * ep.sBias + col];
    if (ep.residual) in.other = ep.residual[b * ep.sR + row * ep.ldr + col];
  }
  return in;
}
// Returns d in the backward pass.
__device__ __forceinline__ float act_element(const ActEpi& ep, uint16_t* C, int64_t ldc, int64_t sC,
                                             int b, int64_t row, int col, float acc,
                                             const ActElement& in) {
  float v[1];
  if (ep.backward) {
    v[0] = ep.alpha * acc;
    if (ep.act.kind != HK_ACT_NONE) {
      const float z[1] = {hk::bf16_to_f32(in.other)};
      hk::scale_by_grad(ep.act, z, v);
    }
  } else {
    v[0] = __builtin_fmaf(ep.alpha, acc, hk::bf16_to_f32(in.bias));
    if (ep.z) ep.z[b * ep.sZ + row * ep.ldz + col] = hk::f32_to_bf16(v[0]);
    hk::activate(ep.act, v);
    if (ep.residual) v[0] += hk::bf16_to_f32(in.other);
  }
  C[b * sC + row * ldc + col] = hk::f32_to_bf16(v[0]);
  return v[0];
}

// The epilogue on the sums of the k splits (split order). A workgroup takes kFinalRows rows of 128
// columns, a thread 8 columns of one. Products that are split have few outputs, so this is the latency of
// its loads: two rows a thread with one split's loads at a time took 257 x 3001 -> 511 from 13.4 to 17.3 us
// (GELU and residual, in a graph), 300 x 4096 -> 304 from 12.5 to 14.9.
constexpr int kFinalRows = 16;
__global__ __launch_bounds__(256) void act_finalize(const float* __restrict__ part, int split_k,
                                                    int col_blocks, int M, int N, ActEpi ep,
                                                    uint16_t* __restrict__ C, int64_t ldc,
                                                    int64_t sC) {
  __shared__ float lds[16][128 + 4];
  const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
  const int b = blockIdx.z, batch = gridDim.z;
  const int cc = (threadIdx.x & 15) * 8, ty = threadIdx.x >> 4;
  const int64_t pitch = part_pitch(N);
  const WaveRows w{C, ldc, sC, b, M, N, rb * kFinalRows, cb * 128, rb, nullptr};
  auto rows = [&](auto&& out) {
    const int row = w.wrow0 + ty;
    const uint4 extra = out.fetch(row);
    if (out.has(row)) {
      const f32x4_t* p = reinterpret_cast<const f32x4_t*>(
          part + (static_cast<int64_t>(b) * M + row) * pitch + out.col);
      const int64_t step = static_cast<int64_t>(batch) * M * pitch / 4;
      f32x4_t lo{}, hi{};
      for (int s = 0; s < split_k; s += 4) {  // eight loads in flight, added in split order
        f32x4_t v[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool on = s + u < split_k;
          v[u][0] = on ? p[(s + u) * step] : f32x4_t{};
          v[u][1] = on ? p[(s + u) * step + 1] : f32x4_t{};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) lo += v[u][0], hi += v[u][1];
      }
      out.row(row, extra, lo, hi);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) lds[ty][cc + e] = out.reg[e];
  };
  if (ep.ragged) rows(ActLane<true>(ep, w, cc));
  else rows(ActLane<false>(ep, w, cc));
  if (!ep.backward || !ep.sums) return;
  __syncthreads();
  if (threadIdx.x < 128 && w.wcol0 + static_cast<int>(threadIdx.x) < N) {
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < 16; ++t) s += lds[t][threadIdx.x];
    ep.sums[(static_cast<int64_t>(b) * ep.sum_rows + rb) * ep.pitch + w.wcol0 + threadIdx.x] = s;
  }
}

// Fallback (K == 0, leading dimensions the tiles do not take): one thread per output and 16th row,
// fp32 accumulation in k order.
constexpr int kSimpleRows = 32;
__global__ __launch_bounds__(256) void act_simple(int ta, int tb, int col_blocks, int M, int N, int K,
                                                  ActEpi ep, const uint16_t* __restrict__ A,
                                                  int64_t lda, int64_t sA,
                                                  const uint16_t* __restrict__ B, int64_t ldb,
                                                  int64_t sB, uint16_t* __restrict__ C, int64_t ldc,
                                                  int64_t sC) {
  __shared__ float lds[16][17];
  const int block = blockIdx.y * gridDim.x + blockIdx.x;
  const int rb = block / col_blocks, cb = block - rb * col_blocks;
  if (rb * kSimpleRows >= M) return;  // the last of blockIdx.y
  const int b = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int col = cb * 16 + tx;
  const uint16_t* Ab = A + b * sA;
  const uint16_t* Bb = B + b * sB;
  float sum = 0.f;
  for (int i = 0; i < kSimpleRows / 16; ++i) {
    const int row = rb * kSimpleRows + ty + 16 * i;
    if (row >= M || col >= N) continue;
    float acc = 0.f;
    for (int k = 0; k < K; ++k) {
      const float a = hk::bf16_to_f32(ta ? Ab[static_cast<int64_t>(k) * lda + row]
                                         : Ab[static_cast<int64_t>(row) * lda + k]);
      const float v = hk::bf16_to_f32(tb ? Bb[static_cast<int64_t>(col) * ldb + k]
                                         : Bb[static_cast<int64_t>(k) * ldb + col]);
      acc += a * v;
    }
    sum += act_element(ep, C, ldc, sC, b, row, col, acc, act_inputs(ep, b, row, col));
  }
  if (!ep.backward || !ep.sums) return;
  lds[ty][tx] = sum;
  __syncthreads();
  if (ty == 0 && col < N) {
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < 16; ++t) s += lds[t][tx];
    ep.sums[(static_cast<int64_t>(b) * ep.sum_rows + rb) * ep.pitch + col] = s;
  }
}

// ---- one row: a matrix that is read once, each of its elements for one product ---------------------
// A workgroup takes some columns of B over all of k and finishes them itself, in the one launch that a short
// decoding step wants, or over a share of k, and a second kernel adds the shares (row_form says when).
// Loads are 16 bytes at any alignment, eight in flight a lane.
typedef uint32_t u32x4a2_t __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 load8_anywhere(const uint16_t* p) {
  const u32x4a2_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4a2_t*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}
constexpr int kRowUnroll = 8;

struct RowOut {
  ActEpi ep;
  uint16_t* C;
  int64_t sC;
  float* dbias;  // the bias gradient where that is this row alone (else ep.sums takes the row)
  int64_t sD;
  int accumulate;
  __device__ ActElement inputs(int b, int col) const { return act_inputs(ep, b, 0, col); }
  __device__ void operator()(int b, int col, float sum, const ActElement& in) const {
    const float d = act_element(ep, C, 0, sC, b, 0, col, sum, in);
    if (!ep.backward) return;
    if (dbias) {
      float* dst = dbias + b * sD + col;
      *dst = accumulate ? *dst + d : d;
    } else if (ep.sums) {
      ep.sums[static_cast<int64_t>(b) * ep.pitch + col] = d;
    }
  }
};

// B [K, N]: a workgroup takes COLS columns and `share` rows of k, a lane 8 columns in every ROWS-th row; the
// partial sums of a column are added over the wave's lanes, then over the waves through LDS. Neighbouring
// workgroups of 32 columns share cache lines of B, so each XCD gets a run of them. With more than one
// share (blockIdx.y) the sums go to part[batch][shares][N].
template <int COLS, int WAVES>
struct RowNn {
  static constexpr int kLanes = COLS / 8, kRows = WAVES * (HK_WAVE / kLanes);
};
template <int COLS, int WAVES>
__global__ __launch_bounds__(WAVES * HK_WAVE) void act_row_nn(int N, int K, int share,
                                                              const uint16_t* __restrict__ B,
                                                              int64_t ldb, int64_t sB,
                                                              const uint16_t* __restrict__ x,
                                                              int64_t incx, int64_t sx,
                                                              float* __restrict__ part, RowOut out) {
  constexpr int kLanes = RowNn<COLS, WAVES>::kLanes, kRows = RowNn<COLS, WAVES>::kRows;
  __shared__ float lds[WAVES][COLS];
  const int b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned xcd = blockIdx.x & 7, total = gridDim.x;
  const int block = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int c = (lane % kLanes) * 8, col = block * COLS + c;
  const unsigned k_begin = blockIdx.y * share, k_end = min(static_cast<unsigned>(K), k_begin + share);
  const int n = min(8, N - col);
  const uint16_t* xb = x + b * sx;
  const uint16_t* Bb = B + b * sB + col;
  float acc[8] = {};
  for (unsigned k0 = k_begin + wave * (kRows / WAVES) + lane / kLanes; k0 < k_end; k0 += kRowUnroll * kRows) {
    uint4 m[kRowUnroll];
    float xv[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      const unsigned k = k0 + u * kRows;
      m[u] = make_uint4(0, 0, 0, 0);
      xv[u] = 0.f;
      if (k < k_end) {
        xv[u] = hk::bf16_to_f32(xb[k * incx]);
        if (n == 8) m[u] = load8_anywhere(Bb + k * ldb);
        else m[u] = load_row8<true>(Bb + k * ldb, n);
      }
    }
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      float f[8];
      hk::BF16::unpack(m[u], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += xv[u] * f[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int step = kLanes; step < HK_WAVE; step *= 2) acc[e] += __shfl_xor(acc[e], step);
  if (lane < kLanes) {
#pragma unroll
    for (int e = 0; e < 8; ++e) lds[wave][c + e] = acc[e];
  }
  __syncthreads();
  const int i = threadIdx.x, own = block * COLS + i;
  if (i < COLS && own < N) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += lds[w][i];
    if (part) part[(static_cast<int64_t>(b) * gridDim.y + blockIdx.y) * N + own] = s;
    else out(b, own, s, out.inputs(b, own));
  }
}

// B [N, K]: a wave takes a row of B, 4 rows a workgroup, and eight waves share a SIMD, so that rows begin while
// others end (bias and GELU, in a graph: 1 x 1280 -> 5120 5.2 us, 6.8 with 16 lanes a row and two waves a
// SIMD; 2560 -> 2560 5.4 and 7.6, 1280 -> 50304 23.5 and 35.0).
constexpr int kNtRows = 4, kNtUnroll = 4, kNtStep = HK_WAVE * 8;
template <bool UNIT>  // incx == 1
__global__ __launch_bounds__(kNtRows * HK_WAVE, UNIT ? 8 : 4) void act_row_nt(
    int N, int K, const uint16_t* __restrict__ B, int64_t ldb, int64_t sB,
    const uint16_t* __restrict__ x, int64_t incx, int64_t sx, RowOut out) {
  const int b = blockIdx.z, j = threadIdx.x & 63;
  const int col = blockIdx.x * kNtRows + (threadIdx.x >> 6);
  const uint16_t* xb = x + b * sx;
  const uint16_t* row = B + b * sB + static_cast<int64_t>(min(col, N - 1)) * ldb;
  auto x8 = [&](unsigned k) {
    if (UNIT) return load_row8<true>(xb + k, 8);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = xb[(k + 2 * e) * incx] | static_cast<uint32_t>(xb[(k + 2 * e + 1) * incx]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  // read ahead of the loop, whose latency hides theirs
  ActElement in{};
  if (j == 0 && col < N) in = out.inputs(b, col);
  float acc = 0.f;
  const unsigned kvec = K & ~7;
  for (unsigned k0 = 8 * j; k0 < kvec; k0 += kNtUnroll * kNtStep) {
    uint4 m[kNtUnroll], v[kNtUnroll];
#pragma unroll
    for (int u = 0; u < kNtUnroll; ++u) {
      const unsigned k = k0 + u * kNtStep;
      m[u] = v[u] = make_uint4(0, 0, 0, 0);
      if (k < kvec) {
        m[u] = load8_anywhere(row + k);
        v[u] = x8(k);
      }
    }
#pragma unroll
    for (int u = 0; u < kNtUnroll; ++u) {
      float fa[8], fb[8];
      hk::BF16::unpack(m[u], fa);
      hk::BF16::unpack(v[u], fb);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += fa[e] * fb[e];
      acc += s;
    }
  }
  if (kvec + j < static_cast<unsigned>(K)) acc += hk::bf16_to_f32(row[kvec + j]) * hk::bf16_to_f32(xb[(kvec + j) * incx]);
  acc = hk::wave_sum(acc);
  if (j == 0 && col < N) out(b, col, acc, in);
}

// The epilogue on the partials [batch][nsplit][N] of a product that is split over k.
__global__ __launch_bounds__(256) void act_row_sum(const float* __restrict__ part, int nsplit, int N,
                                                   RowOut out) {
  const int col = blockIdx.x * 256 + threadIdx.x, b = blockIdx.z;
  if (col >= N) return;
  const float* p = part + static_cast<int64_t>(b) * nsplit * N + col;
  const ActElement in = out.inputs(b, col);
  float s = 0.f;
  // eight loads in flight, added in split order
  for (int k = 0; k < nsplit; k += 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = k + u < nsplit ? p[static_cast<int64_t>(k + u) * N] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
  out(b, col, s, in);
}

// dst[y * stride + col] (+)= the sum of `rows` rows of sums[y][rows][pitch]: 32 columns a workgroup, each
// of its 8 groups of lanes every 8th row.
__global__ __launch_bounds__(256) void act_column_sums(const float* __restrict__ sums, int64_t rows,
                                                       int pitch, int N, float* __restrict__ dst,
                                                       int64_t stride, int accumulate) {
  __shared__ float lds[8][33];
  const int tx = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + tx;
  const float* p = sums + static_cast<int64_t>(blockIdx.y) * rows * pitch + col;
  float v = 0.f;
  if (col < N) {
    for (int64_t r0 = grp; r0 < rows; r0 += 64) {  // eight loads in flight
      float f[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = r0 + 8 * u < rows ? p[(r0 + 8 * u) * pitch] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) v += f[u];
    }
  }
  lds[grp][tx] = v;
  __syncthreads();
  if (grp == 0 && col < N) {
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) s += lds[t][tx];
    float* d = dst + blockIdx.y * stride + col;
    *d = accumulate ? *d + s : s;
  }
}

// ---- host ------------------------------------------------------------------------------------------
struct Call {
  bool ta, tb;
  int M, N, K, batch;
  const hk_bf16* A;
  int64_t lda, sA;
  const hk_bf16* B;
  int64_t ldb, sB;
  ActEpi ep;
  hk_bf16* C;
  int64_t ldc, sC;
  float* dbias;
  int64_t sD;
  bool accumulate;
};

// How a product of one row runs: over `splits` shares of k, and for B [K, N] on which workgroup.
struct RowForm {
  int splits;
  int nn;  // 0: 32 columns, 16 waves; 1: 64 columns, 16 waves; 2: 64 columns, 8 waves
};

// How a call runs, and what it needs: the column sums of `sum_rows` blocks of rows and matrix, and the
// partials of its k splits.
struct Plan {
  enum Kind { kRow, kSimple, kTiles } kind;
  hk::GemmPlan gemm{0, 1, 0};
  hk::GemvPlan gemv{1, 0};
  RowForm row{1, 0};
  bool ragged = false;
  int sum_rows = 0;
  size_t sum_bytes = 0, part_bytes = 0;
  size_t bytes() const { return sum_bytes + part_bytes; }
};

// One CU reads some 20 bytes a nanosecond, so what counts is that all of them get equal parts of B, and what
// a second launch costs, some 2 us of a graph and 2.6 of the host's time (bias and GELU, B from
// memory, in a graph, us).
// B [K, N]: enough columns for a workgroup of 64 on nearly every CU are left whole (K 2560, N 16000: 17.6
// with 16 waves, 26.8 with 8, four shares 20.3; N 50304, K 1280: 34.3, 31.2 and 29.1). A short k, too:
// 32 columns and one trip of the loop (N 5120, K 1280: 8.65 in one launch, 8.05 in two, 5.6 against
// 7.4 for K 512 to 768). Everything else is cut to some 640 workgroups of 64 columns, two or three a CU, of
// at least 160 rows (N 5120, K 2048: 11.8 whole, 9.3 cut; K 5120: 24.6 and 14.6; K 10240: 45.8 and 22.8).
// B [N, K]: rows are left whole unless they are few and very long (N 256, K 10240: 6.7 whole, 6.0 cut, K 5120:
// 4.8 and 5.1; N 1280, K 10240: 8.0 and 9.5, K 50304: 31 and 24; N 5120, K 5120: 11.1 and 12.2).
RowForm row_form(const Call& c, const hk::GemvPlan& gemv) {
  if (c.tb) {
    const bool cut = c.K > 8192 && int64_t{16} * c.N * c.batch <= c.K;
    return {cut ? gemv.nsplit : 1, 0};
  }
  const int64_t groups = hk::ceil_div(c.N, 64) * c.batch;
  if (groups >= 224) return {1, groups >= 512 ? 2 : 1};
  if (c.K <= 1536) return {1, 0};
  return {static_cast<int>(std::min<int64_t>(640 / groups, c.K / 160)), 2};
}
int row_share(const Call& c, const RowForm& f) { return static_cast<int>(hk::ceil_div(c.K, f.splits)); }

// may_split false: k splits only where the product needs them (one row).
Plan make_plan(const Call& c, bool may_split) {
  Plan p;
  const bool sums = c.ep.backward && c.dbias;
  if (c.M == 1 && c.K > 0) {
    p.kind = Plan::kRow;
    if (c.tb) p.gemv = hk::bgemv_plan(true, c.N, c.K, c.batch);
    p.row = row_form(c, p.gemv);
    if (p.row.splits > 1)
      p.part_bytes = static_cast<size_t>(c.batch) * p.row.splits * c.N * sizeof(float);
    p.sum_rows = sums && c.batch > 1 && c.sD == 0 ? 1 : 0;
  } else {
    using hk::aligned16;
    hk::GemmRows rows = hk::bgemm_rows(c.ta, c.tb, c.M, c.N, c.K, c.lda, c.ldb, c.ldc, c.sA, c.sB,
                                       c.sC, c.batch, aligned16(c.A), aligned16(c.B), aligned16(c.C));
    if (rows == hk::GemmRows::kNone) {
      p.kind = Plan::kSimple;
      p.sum_rows = static_cast<int>(hk::ceil_div(c.M, kSimpleRows));
    } else {
      p.kind = Plan::kTiles;
      p.ragged = rows != hk::GemmRows::kAligned ||
                 (c.ep.z && (c.ep.ldz % 8 != 0 || c.ep.sZ % 8 != 0 || !aligned16(c.ep.z))) ||
                 (c.ep.residual &&
                  (c.ep.ldr % 8 != 0 || c.ep.sR % 8 != 0 || !aligned16(c.ep.residual)));
      p.gemm = hk::bgemm_rows_plan(c.ta, c.tb, c.M, c.N, c.K, c.batch, rows, may_split);
      int block = kFinalRows;
      if (p.gemm.used > 1) {
        p.part_bytes = hk::bgemm_partial_bytes(p.gemm.used, c.M, c.N, c.batch);
      } else if (p.gemm.flex) {
        block = act_flex_wave_rows(p.gemm.flex);
      } else {
        block = w160_plan(c.ta, c.tb, c.M, c.N, c.K, c.batch, 1) ? w160::kWaveM
                                                                 : row_tile(c.ta, c.M, c.N, c.batch, 1) / 2;
      }
      p.sum_rows = static_cast<int>(hk::ceil_div(c.M, block));
    }
    if (!sums) p.sum_rows = 0;
  }
  // both parts begin on 16 bytes: the pitch is a multiple of 8 floats
  p.sum_bytes = static_cast<size_t>(c.batch) * p.sum_rows * part_pitch(c.N) * sizeof(float);
  return p;
}

hipError_t column_sums(const Call& c, const float* sums, int64_t rows, hipStream_t stream) {
  const bool shared = c.sD == 0 || c.batch == 1;
  if (rows == 0 && c.accumulate) return hipSuccess;
  HK_CHECK_ARG(shared || c.batch <= 65535);
  hipLaunchKernelGGL(act_column_sums, dim3((c.N + 31) / 32, shared ? 1 : c.batch), dim3(256), 0,
                     stream, sums, shared ? rows * c.batch : rows, part_pitch(c.N), c.N, c.dbias,
                     c.sD, c.accumulate ? 1 : 0);
  return hk::launch_status();
}

hipError_t run_piece(Call c, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (c.N == 0) return hipSuccess;
  if (c.M == 0 || c.batch == 0)  // no rows: a bias gradient of zero
    return c.ep.backward && c.dbias && (c.batch > 0 || c.sD == 0)
               ? column_sums(c, nullptr, 0, stream)
               : hipSuccess;
  Plan p = make_plan(c, true);
  char* ws = static_cast<char*>(workspace);
  if (ws) {
    HK_CHECK_ARG(workspace_bytes >= static_cast<int64_t>(p.bytes()) && hk::aligned16(ws));
  } else if (p.bytes() > 0) {
    // a graph would keep the stream's workspace, which other graphs and eager calls write too
    if (hk::stream_capturing(stream)) return hipErrorStreamCaptureUnsupported;
    void* got = nullptr;
    hipError_t e = hk::device_workspace(p.bytes(), stream, &got);
    if (e == hipErrorOutOfMemory && p.kind == Plan::kTiles && p.part_bytes > 0) {
      (void)hipGetLastError();
      p = make_plan(c, false);  // no memory for the partials
      e = p.bytes() > 0 ? hk::device_workspace(p.bytes(), stream, &got) : hipSuccess;
    }
    HK_RETURN_IF_ERROR(e);
    ws = static_cast<char*>(got);
  }
  float* part = reinterpret_cast<float*>(ws + p.sum_bytes);
  ActEpi& ep = c.ep;
  ep.ragged = p.ragged;
  ep.sums = p.sum_bytes > 0 ? reinterpret_cast<float*>(ws) : nullptr;
  ep.sum_rows = p.sum_rows;
  ep.pitch = part_pitch(c.N);

  if (p.kind == Plan::kRow) {
    // C[0][n] = sum_k op(A)[0][k] op(B)[k][n]
    const int64_t incx = c.ta ? c.lda : 1;
    const RowOut out{ep, c.C, c.sC, ep.sums ? nullptr : c.dbias, c.sD, c.accumulate ? 1 : 0};
    const bool split = p.row.splits > 1;
    if (c.tb && split) {
      HK_RETURN_IF_ERROR(hk::bgemv_partials(c.N, c.K, c.B, c.ldb, c.sB, c.A, incx, c.sA, c.batch,
                                            p.gemv, part, stream));
    } else if (c.tb) {
      hipLaunchKernelGGL(incx == 1 ? act_row_nt<true> : act_row_nt<false>,
                         dim3((c.N + kNtRows - 1) / kNtRows, 1, c.batch),
                         dim3(kNtRows * HK_WAVE), 0, stream, c.N, c.K, c.B, c.ldb, c.sB, c.A, incx,
                         c.sA, out);
    } else {
      const int cols = p.row.nn == 0 ? 32 : 64, waves = p.row.nn == 2 ? 8 : 16;
      const auto kernel = p.row.nn == 0   ? act_row_nn<32, 16>
                          : p.row.nn == 1 ? act_row_nn<64, 16>
                                          : act_row_nn<64, 8>;
      hipLaunchKernelGGL(kernel, dim3((c.N + cols - 1) / cols, p.row.splits, c.batch),
                         dim3(waves * HK_WAVE), 0, stream, c.N, c.K, row_share(c, p.row), c.B, c.ldb,
                         c.sB, c.A, incx, c.sA, split ? part : nullptr, out);
    }
    if (split) {
      HK_RETURN_IF_ERROR(hk::launch_status());
      hipLaunchKernelGGL(act_row_sum, dim3((c.N + 255) / 256, 1, c.batch), dim3(256), 0, stream, part,
                         p.row.splits, c.N, out);
    }
    HK_RETURN_IF_ERROR(hk::launch_status());
    return ep.sums ? column_sums(c, ep.sums, 1, stream) : hipSuccess;
  }
  if (p.kind == Plan::kSimple) {
    const int cols = (c.N + 15) / 16;
    const int64_t blocks = hk::ceil_div(c.M, kSimpleRows) * cols;
    HK_CHECK_ARG(blocks <= INT32_MAX);
    // under 2^32 threads in x
    const auto gx = static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 23));
    const auto gy = static_cast<unsigned>(hk::ceil_div(blocks, gx));
    hipLaunchKernelGGL(act_simple, dim3(gx, gy, c.batch), dim3(256), 0, stream, c.ta ? 1 : 0,
                       c.tb ? 1 : 0, cols, c.M, c.N, c.K, ep, c.A, c.lda, c.sA, c.B, c.ldb, c.sB, c.C,
                       c.ldc, c.sC);
    HK_RETURN_IF_ERROR(hk::launch_status());
  } else if (p.gemm.used > 1) {
    const int cols = (c.N + 127) / 128;
    const int64_t blocks = hk::ceil_div(c.M, kFinalRows) * cols;
    HK_CHECK_ARG(blocks < 1 << 24);  // 2^32 threads
    HK_RETURN_IF_ERROR(hk::bgemm_write_partials(c.ta, c.tb, c.M, c.N, c.K, c.A, c.lda, c.sA, c.B, c.ldb,
                                                c.sB, c.batch, p.gemm, part, stream));
    hipLaunchKernelGGL(act_finalize, dim3(static_cast<unsigned>(blocks), 1, c.batch), dim3(256), 0,
                       stream, part, p.gemm.used, cols, c.M, c.N, ep, c.C, c.ldc, c.sC);
    HK_RETURN_IF_ERROR(hk::launch_status());
  } else if (p.gemm.flex) {
    FlexArgs<ActEpi> g{};
    g.M = c.M, g.N = c.N, g.K = c.K;
    g.ep = ep;
    g.a = Operand{c.A, c.lda, c.sA};
    g.b = Operand{c.B, c.ldb, c.sB};
    g.C = c.C, g.ldc = c.ldc, g.sC = c.sC;
    g.split_k = 1, g.k_per_split = c.K;
    HK_RETURN_IF_ERROR(act_flex_run(p.gemm.flex, c.ta, c.tb, g, c.batch, stream));
  } else {
    const int64_t tiles = hk::ceil_div(c.M, BM) * hk::ceil_div(c.N, BN);
    HK_CHECK_ARG(2 * tiles <= INT32_MAX);
    HK_RETURN_IF_ERROR(act_wide_run(c.ta, c.tb, c.batch, stream, c.M, c.N, c.K, ep, c.A, c.lda, c.sA,
                                    c.B, c.ldb, c.sB, c.C, c.ldc, c.sC));
  }
  return ep.sums ? column_sums(c, ep.sums, p.sum_rows, stream) : hipSuccess;
}

// A dimension of a grid has under 2^32 threads, and more of them run as their number modulo 2^32, with no error.
// One row takes up to 64 threads a column, the smallest tiles of many rows 16 a row, so products of more than
// kPieceSide rows or columns run as several; whole tiles and vectors.
constexpr int kPieceSide = 1 << 25;

hipError_t run(const Call& c, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (c.M <= kPieceSide && c.N <= kPieceSide) return run_piece(c, workspace, workspace_bytes, stream);
  for (int64_t n0 = 0; n0 < c.N; n0 += kPieceSide) {
    for (int64_t m0 = 0; m0 == 0 || m0 < c.M; m0 += kPieceSide) {  // no rows: a bias gradient of zero
      Call p = c;
      p.M = static_cast<int>(std::min<int64_t>(kPieceSide, c.M - m0));
      p.N = static_cast<int>(std::min<int64_t>(kPieceSide, c.N - n0));
      if (c.K > 0) {
        p.A += c.ta ? m0 : m0 * c.lda;
        p.B += c.tb ? n0 * c.ldb : n0;
      }
      p.C += m0 * c.ldc + n0;
      if (c.ep.bias) p.ep.bias += n0;
      if (c.ep.residual) p.ep.residual += m0 * c.ep.ldr + n0;
      if (c.ep.z) p.ep.z += m0 * c.ep.ldz + n0;
      if (c.dbias) p.dbias += n0;
      p.accumulate = c.accumulate || m0 > 0;  // the bias gradients of the rows before are there
      HK_RETURN_IF_ERROR(run_piece(p, workspace, workspace_bytes, stream));
    }
  }
  return hipSuccess;
}

// The arguments that both entry points share.
hipError_t check(int transA, int transB, int M, int N, int K, const void* A, int lda, const void* B,
                 int ldb, int activation, const void* C, int ldc, long long strideC, int batchCount) {
  HK_CHECK_ARG(transA >= 0 && transA <= 2 && transB >= 0 && transB <= 2);
  HK_CHECK_ARG(M >= 0 && N >= 0 && K >= 0 && batchCount >= 0 && batchCount <= kMaxGridZ);
  HK_CHECK_ARG(M <= kMaxSide && N <= kMaxSide && K <= kMaxSide);
  HK_CHECK_ARG(activation >= HK_ACT_NONE && activation <= HK_ACT_SILU);
  if (M == 0 || N == 0 || batchCount == 0) return hipSuccess;
  HK_CHECK_ARG(C != nullptr && ldc >= N && (batchCount == 1 || strideC != 0));
  HK_CHECK_ARG(K == 0 || (A != nullptr && B != nullptr));
  HK_CHECK_ARG(lda >= (transA ? M : K) && ldb >= (transB ? K : N));
  return hipSuccess;
}

// A matrix, or a batch of them, as memory.
hk::Rows memory(const void* p, int rows, int cols, int64_t ld, int64_t stride, int batch) {
  return hk::Rows(p, 2, cols).along(batch, 2 * stride).along(rows, 2 * ld);
}
// Whether C lies apart from the other output and from all inputs, but for `same` (the residual, or a preact that is
// read), which may be C itself.
bool outputs_apart(const Call& c, const hk::Rows& out, const hk::Rows& same) {
  const hk::Rows C = memory(c.C, c.M, c.N, c.ldc, c.sC, c.batch);
  const hk::Rows bias = hk::Rows(c.ep.bias, 2, c.N).along(c.batch, 2 * c.ep.sBias);
  if (hk::overlaps_itself(C) || hk::overlap_unless_same(C, same) || hk::overlap(out, same)) return false;
  if (hk::overlap(C, out) || hk::overlap(C, bias) || hk::overlap(out, bias)) return false;
  if (c.K == 0) return true;
  const hk::Rows A = memory(c.A, c.ta ? c.K : c.M, c.ta ? c.M : c.K, c.lda, c.sA, c.batch);
  const hk::Rows B = memory(c.B, c.tb ? c.N : c.K, c.tb ? c.K : c.N, c.ldb, c.sB, c.batch);
  return !hk::overlap(C, A) && !hk::overlap(C, B) && !hk::overlap(out, A) && !hk::overlap(out, B);
}

Call forward_call(int transA, int transB, int M, int N, int K, hk_bf16 alpha, const hk_bf16* A, int lda,
                  long long strideA, const hk_bf16* B, int ldb, long long strideB,
                  const hk_bf16* bias, long long strideBias, int activation,
                  const hk_bf16* residual, int ldr, long long strideR, hk_bf16* preact, int ldz,
                  long long strideZ, hk_bf16* C, int ldc, long long strideC, int batchCount) {
  ActEpi ep{};
  ep.alpha = hk::bf16_bits_to_float(alpha);
  ep.act = hk::make_activation(activation);
  ep.bias = bias, ep.sBias = strideBias;
  ep.residual = residual, ep.ldr = ldr, ep.sR = strideR;
  ep.z = preact, ep.ldz = ldz, ep.sZ = strideZ;
  return Call{transA != 0, transB != 0, M, N, K, batchCount, A, lda, strideA, B, ldb, strideB,
              ep, C, ldc, strideC, nullptr, 0, false};
}

}  // namespace

extern "C" hipError_t hk_bgemm_act(int transA, int transB, int M, int N, int K, hk_bf16 alpha,
                                   const hk_bf16* A, int lda, long long strideA, const hk_bf16* B,
                                   int ldb, long long strideB, const hk_bf16* bias,
                                   long long strideBias, int activation, const hk_bf16* residual,
                                   int ldr, long long strideR, hk_bf16* preact, int ldz,
                                   long long strideZ, hk_bf16* C, int ldc, long long strideC,
                                   int batchCount, void* workspace, int64_t workspace_bytes,
                                   hipStream_t stream) {
  HK_RETURN_IF_ERROR(check(transA, transB, M, N, K, A, lda, B, ldb, activation, C, ldc, strideC,
                           batchCount));
  HK_CHECK_ARG(!residual || ldr >= N);
  HK_CHECK_ARG(!preact || (ldz >= N && (batchCount <= 1 || strideZ != 0)));
  const Call c = forward_call(transA, transB, M, N, K, alpha, A, lda, strideA, B, ldb, strideB, bias,
                              strideBias, activation, residual, ldr, strideR, preact, ldz, strideZ, C, ldc,
                              strideC, batchCount);
  const hk::Rows z = memory(preact, M, N, ldz, strideZ, batchCount);
  HK_CHECK_ARG(!hk::overlaps_itself(z) &&
               outputs_apart(c, z, memory(residual, M, N, ldr, strideR, batchCount)));
  return run(c, workspace, workspace_bytes, stream);
}

extern "C" hipError_t hk_bgemm_act_backward(int transA, int transB, int M, int N, int K, hk_bf16 alpha,
                                            const hk_bf16* A, int lda, long long strideA,
                                            const hk_bf16* B, int ldb, long long strideB,
                                            int activation, const hk_bf16* preact, int ldz,
                                            long long strideZ, hk_bf16* C, int ldc,
                                            long long strideC, float* dbias, long long strideDbias,
                                            int accumulate, int batchCount, void* workspace,
                                            int64_t workspace_bytes, hipStream_t stream) {
  HK_RETURN_IF_ERROR(check(transA, transB, M, N, K, A, lda, B, ldb, activation, C, ldc, strideC,
                           batchCount));
  const bool empty = M == 0 || N == 0 || batchCount == 0;
  HK_CHECK_ARG(activation == HK_ACT_NONE || empty || (preact != nullptr && ldz >= N));
  HK_CHECK_ARG((reinterpret_cast<uintptr_t>(dbias) & 3u) == 0);
  HK_CHECK_ARG(batchCount <= 1 || strideDbias == 0 || strideDbias >= N || strideDbias <= -N);
  ActEpi ep{};
  ep.alpha = hk::bf16_bits_to_float(alpha);
  ep.act = hk::make_activation(activation);
  ep.backward = true;
  ep.z = activation == HK_ACT_NONE ? nullptr : const_cast<hk_bf16*>(preact);
  ep.ldz = ldz, ep.sZ = strideZ;
  const Call c{transA != 0, transB != 0, M, N, K, batchCount, A, lda, strideA, B, ldb, strideB,
               ep, C, ldc, strideC, dbias, strideDbias, accumulate != 0};
  HK_CHECK_ARG(outputs_apart(
      c, hk::Rows(dbias, 4, N).along(strideDbias != 0 ? batchCount : 1, 4 * int64_t{strideDbias}),
      memory(ep.z, M, N, ldz, strideZ, batchCount)));
  return run(c, workspace, workspace_bytes, stream);
}

extern "C" int64_t hk_bgemm_act_workspace(int transA, int transB, int M, int N, int K, int batchCount,
                                          int dbias) {
  if (transA < 0 || transA > 2 || transB < 0 || transB > 2 || M < 0 || N < 0 || K < 0 ||
      batchCount < 0 || batchCount > kMaxGridZ || M > kMaxSide || N > kMaxSide || K > kMaxSide)
    return -1;
  if (M == 0 || N == 0 || batchCount == 0) return 0;
  // the most of what the rows' alignments make of the call, and of its whole and last pieces
  Call c{};
  c.ta = transA != 0, c.tb = transB != 0;
  c.K = K, c.batch = batchCount;
  c.ep.backward = dbias != 0;
  float none;
  c.dbias = dbias ? &none : nullptr;  // compared with NULL only
  size_t most = 0;
  for (int piece = 0; piece < 4; ++piece) {
    if ((piece & 1 && M <= kPieceSide) || (piece & 2 && N <= kPieceSide)) continue;
    c.M = piece & 1 ? (M - 1) % kPieceSide + 1 : std::min(M, kPieceSide);
    c.N = piece & 2 ? (N - 1) % kPieceSide + 1 : std::min(N, kPieceSide);
    for (int odd = 0; odd < 4; ++odd) {
      // aligned, unaligned C, unaligned A and B, and the fallback's leading dimensions
      c.lda = (odd == 3 ? int64_t{1} << 22 : hk::ceil_div(c.ta ? M : K, 8) * 8) + (odd == 2 ? 1 : 0);
      c.ldb = hk::ceil_div(c.tb ? K : N, 8) * 8;
      c.ldc = hk::ceil_div(N, 8) * 8 + (odd == 1 ? 1 : 0);
      most = std::max(most, make_plan(c, true).bytes());
    }
  }
  return static_cast<int64_t>(most);
}

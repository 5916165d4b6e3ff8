// embedding.hip - embedding lookup, out[i] = scale table[token_i] + residual[i], and the table's gradient,
// grad_table[v] (+)= scale sum of grad[i] over the i with token_i = v. fp32, bf16 and fp16, any d, strides, alignment.
//
// Both are bound by memory. The gradient has to be the same whatever the order in which workgroups run, and texts repeat a
// few words very often, so rows are neither added atomically nor owned by one workgroup each:
//   embedding_sort     workgroup b of 2^bits has the table rows b, b + 2^bits, .. (frequent words lie side by side in most
//                      vocabularies). It reads all tokens (from L2), counts those of the workgroups before it, which is
//                      where its part of the order begins, and places its own by row, in the tokens' order.
//   embedding_sum      the sorted order in equal chunks, a wave each and 64 units of columns: rows that lie inside a chunk
//                      are written, the parts of those that go on across its ends are left as partial sums,
//   embedding_combine  which are added in order where such a row begins.
// All three are latency, and clearing the table is bandwidth: each launch clears a part of it beside its own work.
// Few tokens take one launch: each workgroup finds its rows' tokens and sums them itself.
//
// Measured: 8192 rows of 768 of an fp32 table, added to bf16 rows, 7.8 us; their table's gradient (50257 rows, 154 MB
// written) 43 us (17 + 15 + 11 as profiled), 6.1 TB/s of it 26: the three are chains of dependent loads; 333 tokens over
// 1009 x 131 6.0 us, launch and loads.
#include <algorithm>
#include <initializer_list>

#include "hk_device.h"
#include "hk_host.h"
#include "hk_overlap.h"

namespace hk {
namespace {

__device__ __forceinline__ int64_t token_of(const void* tokens, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(tokens)[i] : static_cast<const int32_t*>(tokens)[i];
}

// E elements of a row as fp32: whole vectors where E > 1.
template <class F, int E>
__device__ __forceinline__ void load(const void* p, int64_t at, float* f) {
  using S = typename F::storage;
  const S* x = static_cast<const S*>(p) + at;
  if constexpr (E == 1) {
    f[0] = F::load(x, 0);
  } else if constexpr (E * sizeof(S) == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(x);
    float t[8];
    F::unpack(make_uint4(w.x, w.y, 0, 0), t);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = t[i];
  } else {
#pragma unroll
    for (int i = 0; i < E; i += F::kPerVec) F::unpack(*reinterpret_cast<const uint4*>(x + i), f + i);
  }
}
template <class F, int E>
__device__ __forceinline__ void store(void* p, int64_t at, const float* f) {
  using S = typename F::storage;
  S* x = static_cast<S*>(p) + at;
  if constexpr (E == 1) {
    F::store(x, 0, f[0]);
  } else if constexpr (E * sizeof(S) == 8) {
    *reinterpret_cast<uint2*>(x) = make_uint2(F::pack2(f[0], f[1]), F::pack2(f[2], f[3]));
  } else {
#pragma unroll
    for (int i = 0; i < E; i += F::kPerVec) st_nt(reinterpret_cast<uint4*>(x + i), F::pack(f + i));
  }
}

// ---- lookup ------------------------------------------------------------------------------------------------
struct Lookup {
  const void *table, *tokens, *residual;
  void* out;
  int wide_tokens;
  int64_t vocab, table_stride, residual_stride, out_stride;
  float scale;
  int units;       // a row, of E elements
  int64_t first;   // row of this launch's first unit
  uint32_t total;  // units of this launch
};

template <class FT, class FO, int E>
__global__ __launch_bounds__(256) void embedding_lookup(Lookup a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.total) return;
  const uint32_t r = i / a.units;
  const int64_t row = a.first + r;
  const int col = static_cast<int>(i - r * a.units) * E;
  const int64_t t = token_of(a.tokens, a.wide_tokens, row);
  float f[E], g[E];
  if (static_cast<uint64_t>(t) < static_cast<uint64_t>(a.vocab)) {
    load<FT, E>(a.table, t * a.table_stride + col, f);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= a.scale;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = __uint_as_float(0x7fc00000u);
  }
  if (a.residual) {
    load<FO, E>(a.residual, row * a.residual_stride + col, g);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] += g[e];
  }
  store<FO, E>(a.out, row * a.out_stride + col, f);
}

// ---- gradient ----------------------------------------------------------------------------------------------
struct Grad {
  const void *grad, *tokens;
  void* table;
  int wide_tokens;
  int64_t n, vocab, grad_stride, table_stride;
  int d;
  float scale;
  int accumulate;
  int bits;         // workgroup b that sorts (or of `few`) has rows b, b + 2^bits, ..
  int range;        // their bits in `used`
  int ranges;       // workgroups that sort
  int sums;         // workgroups that sum, and that combine
  int clear;        // table rows that each of the workgroups behind these clears:
  int64_t clear_sum, clear_sort;  // combine from row 0, sum from clear_sum, sort from clear_sort
  int table_elem;   // bytes
  int chunk;        // positions a chunk
  int col_blocks;   // waves a chunk
  uint2* sorted;    // (token's place, its table row), the places of a row side by side; row ~0 behind the last
  uint64_t* used;   // a bit for each table row, `range` a workgroup: some token is it
  float* part;      // [chunk][2][d]: of the row that goes on from before, of the one that goes on behind
};

// Zeros one row of the table: all lanes of a group of `lanes`.
__device__ __forceinline__ void zero_row(const Grad& a, int64_t row, int lane, int lanes) {
  char* p = static_cast<char*>(a.table) + row * a.table_stride * a.table_elem;
  const int64_t bytes = static_cast<int64_t>(a.d) * a.table_elem;
  const uintptr_t both = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(bytes);
  if ((both & 15) == 0) {
    for (int64_t i = lane * 16; i < bytes; i += lanes * 16) st_nt(reinterpret_cast<uint4*>(p + i), make_uint4(0, 0, 0, 0));
  } else if ((both & 3) == 0) {
    for (int64_t i = lane * 4; i < bytes; i += lanes * 4) *reinterpret_cast<uint32_t*>(p + i) = 0;
  } else {
    for (int64_t i = lane * 2; i < bytes; i += lanes * 2) *reinterpret_cast<uint16_t*>(p + i) = 0;
  }
}

// Zeros a workgroup's part of the rows from `first` to `end`; without those that have tokens if their bits are known.
__device__ __forceinline__ void clear_rows(const Grad& a, int block, int64_t first, int64_t end, bool known) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  first += static_cast<int64_t>(block) * a.clear;
  end = min(end, first + a.clear);
  for (int64_t r = first + wave; r < end; r += waves) {
    const int64_t bit = (r & ((int64_t(1) << a.bits) - 1)) * a.range + (r >> a.bits);
    if (!known || !(a.used[bit >> 6] >> (bit & 63) & 1)) zero_row(a, r, threadIdx.x & 63, 64);
  }
}

constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kRounds = 8;                             // tokens a lane and tile
constexpr int kTileTokens = kSortThreads * kRounds;    // 4096
constexpr int kMaxRange = 1024;

__global__ __launch_bounds__(kSortThreads) void embedding_sort(Grad a) {
  __shared__ int count[kMaxRange];             // of each row, then where its next token goes
  __shared__ int wave_at[kSortWaves][kMaxRange];
  __shared__ uint2 list[kTileTokens];
  __shared__ int sums[kSortWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  if (static_cast<int>(blockIdx.x) >= a.ranges) {
    clear_rows(a, blockIdx.x - a.ranges, a.clear_sort, a.vocab, false);
    return;
  }
  const uint32_t mask_of = (1u << a.bits) - 1, me = blockIdx.x;
  const int rows = static_cast<int>((a.vocab - me + mask_of) >> a.bits);
  // the row of one of this workgroup's tokens, ~0 for others
  auto row_of = [&](uint64_t t) {
    return t < static_cast<uint64_t>(a.vocab) && (t & mask_of) == me ? static_cast<uint32_t>(t >> a.bits) : ~0u;
  };

  for (int i = tid; i < rows; i += kSortThreads) count[i] = 0;
  __syncthreads();
  int below = 0;
  for (int64_t i = tid; i < a.n; i += kSortThreads * 4) {
    uint64_t t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = i + u * kSortThreads;
      t[u] = at < a.n ? static_cast<uint64_t>(token_of(a.tokens, a.wide_tokens, at)) : ~uint64_t(0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      below += t[u] < static_cast<uint64_t>(a.vocab) && (t[u] & mask_of) < me;
      const uint32_t r = row_of(t[u]);
      if (r != ~0u) atomicAdd(&count[r], 1);
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) below += __shfl_xor(below, s);
  if (lane == 0) sums[wave] = below;
  __syncthreads();
  below = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) below += sums[w];
  if (!a.accumulate)
    for (int r = wave * 64; r < rows; r += kSortThreads) {
      const uint64_t some = __ballot(r + lane < rows && count[min(r + lane, rows - 1)] > 0);
      if (lane == 0) a.used[(static_cast<int64_t>(me) * a.range + r) >> 6] = some;
    }
  __syncthreads();

  // count[r]: the first place of row r in the sorted order
  {
    constexpr int kPer = kMaxRange / kSortThreads;
    int mine[kPer], sum = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int r = tid * kPer + u;
      mine[u] = r < rows ? count[r] : 0;
      sum += mine[u];
    }
    int incl = sum;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const int up = __shfl_up(incl, s);
      if (lane >= s) incl += up;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int at = below + incl - sum;
    for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int r = tid * kPer + u;
      if (r < rows) count[r] = at;
      at += mine[u];
    }
    // the last workgroup knows where the valid tokens end
    int total = below;
    for (int w = 0; w < kSortWaves; ++w) total += sums[w];
    if (static_cast<int>(me) == a.ranges - 1)
      for (int64_t i = total + tid; i < a.n; i += kSortThreads) a.sorted[i] = make_uint2(0, ~0u);
    if (total == below) return;  // none of these rows
  }

  int bits = 1;
  while ((1 << bits) < rows) ++bits;
  for (int64_t base = 0; base < a.n; base += kTileTokens) {
    // this range's tokens of the tile in order: each wave looks through 64 x kRounds of them
    uint32_t row[kRounds];
    uint64_t mask[kRounds];
    int found = 0;
    const int64_t w0 = base + wave * (64 * kRounds) + lane;
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
      const int64_t at = w0 + 64 * u;
      row[u] = at < a.n ? row_of(static_cast<uint64_t>(token_of(a.tokens, a.wide_tokens, at))) : ~0u;
    }
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
      mask[u] = __ballot(row[u] != ~0u);
      found += __popcll(mask[u]);
    }
    __syncthreads();  // the tile before is done with list and sums
    if (lane == 0) sums[wave] = found;
    for (int i = tid; i < kSortWaves * rows; i += kSortThreads) wave_at[i / rows][i % rows] = 0;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      if (w < wave) at += sums[w];
      total += sums[w];
    }
    if (total == 0) continue;
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
      const int before = __popcll(mask[u] & ((uint64_t(1) << lane) - 1));
      if (row[u] != ~0u) list[at + before] = make_uint2(static_cast<uint32_t>(w0 + 64 * u), row[u]);
      at += __popcll(mask[u]);
    }
    __syncthreads();
    // each wave takes an equal part of the list: how many of each row it has, where they go, and there
    const int per = ((total + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
    const int from = wave * per, to = min(from + per, total);
    for (int i = from + lane; i < to; i += 64) atomicAdd(&wave_at[wave][list[i].y], 1);
    __syncthreads();
    for (int r = tid; r < rows; r += kSortThreads) {
      int next = count[r];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = wave_at[w][r];
        wave_at[w][r] = next;
        next += c;
      }
      count[r] = next;
    }
    __syncthreads();
    for (int i0 = from; i0 < to; i0 += 64) {
      const int i = i0 + lane;
      const bool some = i < to;
      const uint2 e = some ? list[i] : make_uint2(0, 0);
      uint64_t same = __ballot(some);
      for (int b = 0; b < bits; ++b) {
        const bool bit = (e.y >> b) & 1;
        const uint64_t with = __ballot(some && bit);
        same &= bit ? with : ~with;
      }
      const int before = __popcll(same & ((uint64_t(1) << lane) - 1));
      int place = 0;
      if (some) place = wave_at[wave][e.y] + before;
      if (some && (same >> lane) == 1) wave_at[wave][e.y] = place + 1;  // the last of them
      if (some) a.sorted[place] = make_uint2(e.x, (e.y << a.bits) + me);
    }
  }
}

template <class FT, int E>
__device__ __forceinline__ void put_row(const Grad& a, uint32_t row, int col, float* f) {
  const int64_t at = static_cast<int64_t>(row) * a.table_stride + col;
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] *= a.scale;
  if (a.accumulate) {
    float g[E];
    load<FT, E>(a.table, at, g);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] += g[e];
  }
  store<FT, E>(a.table, at, f);
}

constexpr int kAhead = 16;   // rows in flight
constexpr int kWindow = 32;  // positions that a wave reads at once

// The wave's chunk and columns. All but the column is the same for the whole wave, and kept in scalar registers.
struct Place {
  int64_t chunk, from, to;
  int col;
  __device__ Place(const Grad& a, int unit) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    chunk = item / a.col_blocks;
    col = (static_cast<int>(item - chunk * a.col_blocks) * 64 + (threadIdx.x & 63)) * unit;
    from = chunk * a.chunk, to = min(from + a.chunk, a.n);
  }
};
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
  return __builtin_amdgcn_readlane(v, lane);
}

template <class FG, class FT, int E>
__global__ __launch_bounds__(256) void embedding_sum(Grad a) {
  if (static_cast<int>(blockIdx.x) >= a.sums) {
    clear_rows(a, blockIdx.x - a.sums, a.clear_sum, a.clear_sort, true);
    return;
  }
  const Place w(a, E);
  if (w.from >= a.n) return;
  const int lane = threadIdx.x & 63;
  const bool mine = w.col < a.d;
  float acc[E] = {};
  uint32_t before = ~0u, row = ~0u;
  auto flush = [&](bool partial) {
    if (row == ~0u || !mine) return;
    if (row == before || partial) {
      float* p = a.part + (w.chunk * 2 + (row == before ? 0 : 1)) * a.d + w.col;
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = acc[e];
    } else {
      put_row<FT, E>(a, row, w.col, acc);
    }
  };
  for (int64_t p0 = w.from; p0 < w.to; p0 += kWindow) {
    // lane l: position p0 + l - 1, from the one before the window to the one behind it
    const int64_t at = p0 + lane - 1;
    const uint2 s = lane <= kWindow + 1 && at >= 0 && at < a.n ? a.sorted[at] : make_uint2(0, ~0u);
    if (p0 == w.from) before = lane_value(s.y, 0);
    const int count = static_cast<int>(min(w.to - p0, static_cast<int64_t>(kWindow)));
    for (int half = 0; half < kWindow / kAhead; ++half) {
      const int q0 = half * kAhead;
      if (q0 >= count) break;
      float x[kAhead][E];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t r = q0 + u < count ? lane_value(s.y, q0 + u + 1) : ~0u;
        if (r != ~0u && mine)
          load<FG, E>(a.grad, static_cast<int64_t>(lane_value(s.x, q0 + u + 1)) * a.grad_stride + w.col, x[u]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t r = q0 + u < count ? lane_value(s.y, q0 + u + 1) : ~0u;
        if (r == ~0u) continue;
        if (r != row) {
          flush(false);
          row = r;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += x[u][e];
      }
    }
    if (p0 + count == w.to) flush(row == lane_value(s.y, count + 1));
  }
}

// The row that begins in a chunk and goes on behind it: its part of this chunk, and of the chunks that it goes on into.
template <class FT, int E>
__global__ __launch_bounds__(256) void embedding_combine(Grad a) {
  if (static_cast<int>(blockIdx.x) >= a.sums) {
    clear_rows(a, blockIdx.x - a.sums, 0, a.clear_sum, true);
    return;
  }
  const Place w(a, E);
  if (w.to >= a.n) return;
  const int lane = threadIdx.x & 63;
  const bool mine = w.col < a.d;
  // the rows at the ends of the chunk, and at the beginnings of the next ones
  const int64_t end = lane == 0 ? w.to : lane == 1 ? w.to - 1 : w.from - 1;
  const uint32_t ends = lane < 3 && end >= 0 ? a.sorted[end].y : ~0u;
  auto begins = [&](int64_t c) {
    const int64_t first = (c + lane) * a.chunk;
    return first < a.n ? a.sorted[first].y : ~0u;
  };
  uint32_t next = begins(w.chunk + 1);
  float acc[E] = {};
  if (mine)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = a.part[(w.chunk * 2 + 1) * a.d + w.col + e];
  const uint32_t row = lane_value(ends, 0);
  if (row == ~0u || lane_value(ends, 1) != row || lane_value(ends, 2) == row) return;
  for (int64_t c = w.chunk + 1;; c += 64, next = begins(c)) {
    // how many of the next chunks begin with it
    const uint64_t on = __ballot(next == row);
    const int more = ~on ? __ffsll(static_cast<unsigned long long>(~on)) - 1 : 64;
    if (mine)
      for (int i = 0; i < more; i += kAhead) {
        float x[kAhead][E];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][e] = i + u < more ? a.part[(c + i + u) * 2 * a.d + w.col + e] : 0.f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += x[u][e];
      }
    if (more < 64) break;
  }
  if (mine) put_row<FT, E>(a, row, w.col, acc);
}

// Few tokens: a workgroup finds those of its rows and sums them in order, a wave a row. Frequent words lie side by side in
// most vocabularies, so a workgroup has rows far apart; and a row of more than kLong tokens, a chain of loads, is summed by
// all four waves, each every fourth window of the list, and their parts in order.
constexpr int kFew = 2048, kFewer = 1024;  // tokens: of the two variants, by what a lane holds
constexpr int kLong = 32;
template <class FG, class FT, int E, int U>
__global__ __launch_bounds__(256) void embedding_few(Grad a) {
  __shared__ uint2 list[U * 256];
  __shared__ float parts[3][E][64];
  __shared__ int sums[4];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const uint32_t stride = 1u << a.bits;
  const int64_t rows = (a.vocab - blockIdx.x + stride - 1) >> a.bits;
  uint32_t row[U];
  uint64_t mask[U];
  int found = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (wave * U + u) * 64 + lane;
    const uint64_t t = at < a.n ? static_cast<uint64_t>(token_of(a.tokens, a.wide_tokens, at)) : ~uint64_t(0);
    const bool here = t < static_cast<uint64_t>(a.vocab) && (t & (stride - 1)) == blockIdx.x;
    row[u] = here ? static_cast<uint32_t>(t >> a.bits) : ~0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    mask[u] = __ballot(row[u] != ~0u);
    found += __popcll(mask[u]);
  }
  if (lane == 0) sums[wave] = found;
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) at += sums[w];
    total += sums[w];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row[u] != ~0u)
      list[at + __popcll(mask[u] & ((uint64_t(1) << lane) - 1))] = make_uint2((wave * U + u) * 64 + lane, row[u]);
    at += __popcll(mask[u]);
  }
  __syncthreads();
  if (a.accumulate && total == 0) return;  // none of these rows
  auto tokens_in = [&](int i, uint32_t r) { return __ballot(i + lane < total && list[min(i + lane, total - 1)].y == r); };
  auto tokens_of = [&](uint32_t r) {
    int c = 0;
    for (int i = 0; i < total; i += 64) c += __popcll(tokens_in(i, r));
    return c;
  };
  // the sum of the row's tokens in every `step`-th window of the list
  auto sum = [&](uint32_t r, int first, int step, int col, bool mine, float* acc) {
    for (int i = first * 64; i < total; i += step * 64) {
      uint64_t of = tokens_in(i, r);
      while (of) {
        float x[kAhead][E];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][e] = 0.f;
          if (of) {
            const int k = __ffsll(static_cast<unsigned long long>(of)) - 1;
            of &= of - 1;
            if (mine) load<FG, E>(a.grad, static_cast<int64_t>(list[i + k].x) * a.grad_stride + col, x[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += x[u][e];
      }
    }
  };
  for (int64_t r = wave; r < rows; r += 4) {
    const int64_t to = (r << a.bits) + blockIdx.x;
    const int of = tokens_of(static_cast<uint32_t>(r));
    if (of == 0) {
      if (!a.accumulate && r % gridDim.y == blockIdx.y) zero_row(a, to, lane, 64);
    } else if (of <= kLong) {
      for (int c0 = blockIdx.y; c0 < a.col_blocks; c0 += gridDim.y) {
        const int col = (c0 * 64 + lane) * E;
        float acc[E] = {};
        sum(static_cast<uint32_t>(r), 0, 1, col, col < a.d, acc);
        if (col < a.d) put_row<FT, E>(a, static_cast<uint32_t>(to), col, acc);
      }
    }
  }
  if (total <= kLong) return;
  for (int64_t r = 0; r < rows; ++r) {
    if (tokens_of(static_cast<uint32_t>(r)) <= kLong) continue;
    for (int c0 = blockIdx.y; c0 < a.col_blocks; c0 += gridDim.y) {
      const int col = (c0 * 64 + lane) * E;
      float acc[E] = {};
      sum(static_cast<uint32_t>(r), wave, 4, col, col < a.d, acc);
      if (wave > 0)
#pragma unroll
        for (int e = 0; e < E; ++e) parts[wave - 1][e][lane] = acc[e];
      __syncthreads();
      if (wave == 0 && col < a.d) {
#pragma unroll
        for (int w = 0; w < 3; ++w)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += parts[w][e][lane];
        put_row<FT, E>(a, static_cast<uint32_t>((r << a.bits) + blockIdx.x), col, acc);
      }
      __syncthreads();
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------
int64_t elem(int type) { return type == HK_TYPE_F32 ? 4 : 2; }
bool type_ok(int type) { return type >= HK_TYPE_F32 && type <= HK_TYPE_F16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Elements a lane takes at once: 8 where all tensors have them as 16-byte vectors (fp32: two), 4, or 1.
struct Matrix {
  const void* p;
  int64_t stride, elem;
  int64_t rows;
};
int unit(int64_t d, int most, std::initializer_list<Matrix> ts) {
  for (int e = most; e >= 4; e /= 2) {
    bool all = d % e == 0;
    for (const Matrix& t : ts) {
      const int64_t bytes = e * t.elem < 16 ? e * t.elem : 16;
      all = all && (!t.p || (aligned(t.p, bytes) && (t.rows <= 1 || t.stride * t.elem % bytes == 0)));
    }
    if (all) return e;
  }
  return 1;
}

template <class FT, class FO>
hipError_t lookup(Lookup a, int64_t n, int64_t d, int e, hipStream_t stream) {
  a.units = static_cast<int>(d / e);
  const int64_t step = std::max<int64_t>(1, (int64_t(1) << 30) / a.units);
  for (a.first = 0; a.first < n; a.first += step) {
    a.total = static_cast<uint32_t>(std::min(step, n - a.first) * a.units);
    const dim3 grid((a.total + 255) / 256);
    if (e == 8) hipLaunchKernelGGL((embedding_lookup<FT, FO, 8>), grid, dim3(256), 0, stream, a);
    else if (e == 4) hipLaunchKernelGGL((embedding_lookup<FT, FO, 4>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((embedding_lookup<FT, FO, 1>), grid, dim3(256), 0, stream, a);
    HK_RETURN_IF_ERROR(launch_status());
  }
  return hipSuccess;
}
template <class FT>
hipError_t lookup_to(const Lookup& a, int64_t n, int64_t d, int e, int out_type, hipStream_t stream) {
  return out_type == HK_TYPE_F32    ? lookup<FT, F32>(a, n, d, e, stream)
         : out_type == HK_TYPE_BF16 ? lookup<FT, BF16>(a, n, d, e, stream)
                                    : lookup<FT, F16>(a, n, d, e, stream);
}

// Positions a chunk: a wave's serial work, and the partial sums of a frequent row, both grow as the root of n.
int chunk_of(int64_t n) {
  int c = kAhead;
  while (int64_t(c) * c * 32 < n && c < 4096) c *= 2;
  return c;
}
int64_t chunks_of(int64_t n) { return ceil_div(n, chunk_of(n)); }
// One launch: up to 1024 tokens, and up to 2048 over a table that this launch clears as fast as the three (one launch and
// three: 333 tokens over 1009 x 131 8 and 26 us, 1000 over 50257 x 768 38 and 34, 2048 over 1000 x 64 12 and 28, over 5000
// x 256 18 and 19, over 50257 x 768 41 and 34, over 131072 x 512 69 and 54).
bool few(int64_t n, int64_t vocab) { return n <= kFewer || (n <= kFew && vocab <= 32768); }
// Half of the workgroups that the card holds at once, of 16 to 1024 rows.
int sort_bits(int64_t vocab) {
  int bits = 0;
  while ((bits < 8 && (vocab >> bits) > 16) || ceil_div(vocab, int64_t(1) << bits) > kMaxRange) ++bits;
  return bits;
}
int used_bits(int64_t vocab) { return static_cast<int>(ceil_div(ceil_div(vocab, int64_t(1) << sort_bits(vocab)), 64) * 64); }
struct Workspace {
  int64_t used, part, bytes;
};
Workspace gradient_workspace(int64_t n, int64_t vocab, int64_t d) {
  if (few(n, vocab)) return {0, 0, 0};
  const int64_t used = ceil_div(8 * n, 16) * 16, part = used + ceil_div(int64_t(used_bits(vocab) / 8) << sort_bits(vocab), 16) * 16;
  return {used, part, part + chunks_of(n) * 2 * d * 4};
}

template <class FG, class FT, int E>
hipError_t gradient(Grad a, hipStream_t stream) {
  a.col_blocks = static_cast<int>(ceil_div(a.d, 64 * E));
  if (few(a.n, a.vocab)) {
    // A wave a row, and workgroups for all CUs; the columns of a frequent row go to several (333 tokens, 1009 x 131: 11.7
    // -> 6.4 us).
    int64_t blocks = 1;
    while (blocks < 2048 && blocks * 4 < a.vocab) blocks *= 2, ++a.bits;
    const dim3 grid(static_cast<unsigned>(std::min(blocks, a.vocab)), std::min(a.col_blocks, 16));
    if (a.n <= kFewer)
      hipLaunchKernelGGL((embedding_few<FG, FT, E, kFewer / 256>), grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((embedding_few<FG, FT, E, kFew / 256>), grid, dim3(256), 0, stream, a);
    return launch_status();
  }
  a.bits = sort_bits(a.vocab);
  a.ranges = static_cast<int>(std::min(int64_t(1) << a.bits, a.vocab));
  a.range = used_bits(a.vocab);
  a.chunk = chunk_of(a.n);
  a.sums = static_cast<int>(ceil_div(chunks_of(a.n) * a.col_blocks, 4));
  int64_t sort = a.ranges, sum = a.sums, combine = a.sums;
  if (!a.accumulate) {
    // 64 KiB a workgroup, and not more workgroups than a launch takes; the three launches' parts by how long they are
    // without it (8192 tokens, 50257 x 768: all in the first 46.5, so 43.3 us)
    a.clear = static_cast<int>(std::max<int64_t>({kSortWaves, 65536 / (int64_t(a.d) * a.table_elem), a.vocab >> 20}));
    a.clear_sum = a.vocab * 3 / 10, a.clear_sort = a.vocab * 6 / 10;
    combine += ceil_div(a.clear_sum, a.clear);
    sum += ceil_div(a.clear_sort - a.clear_sum, a.clear);
    sort += ceil_div(a.vocab - a.clear_sort, a.clear);
  }
  hipLaunchKernelGGL(embedding_sort, dim3(static_cast<unsigned>(sort)), dim3(kSortThreads), 0, stream, a);
  HK_RETURN_IF_ERROR(launch_status());
  hipLaunchKernelGGL((embedding_sum<FG, FT, E>), dim3(static_cast<unsigned>(sum)), dim3(256), 0, stream, a);
  HK_RETURN_IF_ERROR(launch_status());
  hipLaunchKernelGGL((embedding_combine<FT, E>), dim3(static_cast<unsigned>(combine)), dim3(256), 0, stream, a);
  return launch_status();
}
template <class FG, class FT>
hipError_t gradient_by(const Grad& a, int e, hipStream_t stream) {
  return e == 4 ? gradient<FG, FT, 4>(a, stream) : gradient<FG, FT, 1>(a, stream);
}
template <class FG>
hipError_t gradient_to(const Grad& a, int e, int table_type, hipStream_t stream) {
  return table_type == HK_TYPE_F32    ? gradient_by<FG, F32>(a, e, stream)
         : table_type == HK_TYPE_BF16 ? gradient_by<FG, BF16>(a, e, stream)
                                      : gradient_by<FG, F16>(a, e, stream);
}

constexpr int64_t kMost = int64_t(1) << 31, kStride = int64_t(1) << 40;
bool sizes_ok(int64_t n, int64_t vocab, int64_t d) {
  return n >= 0 && n < kMost && vocab >= 1 && vocab < kMost && d >= 1 && d < kMost;
}
bool gradient_ok(int64_t n, int64_t vocab, int64_t d) {
  if (!sizes_ok(n, vocab, d) || n >= kMost / 2) return false;
  return chunks_of(n) * ceil_div(d, 64) < (int64_t(1) << 25);  // waves of a launch
}

}  // namespace
}  // namespace hk

extern "C" hipError_t hk_embedding_forward(const void* table, int type, int64_t vocab, int64_t d, int64_t table_stride,
                                           const void* tokens, int wide_tokens, int64_t n, float scale,
                                           const void* residual, int64_t residual_stride, void* out, int out_type,
                                           int64_t out_stride, hipStream_t stream) {
  using namespace hk;
  HK_CHECK_ARG(type_ok(type) && type_ok(out_type) && sizes_ok(n, vocab, d));
  for (int64_t s : {table_stride, residual_stride, out_stride}) HK_CHECK_ARG(s >= 0 && s < kStride);
  if (n == 0) return hipSuccess;
  const int64_t et = elem(type), eo = elem(out_type), ei = wide_tokens ? 8 : 4;
  HK_CHECK_ARG(table && tokens && out && aligned(table, et) && aligned(tokens, ei) && aligned(out, eo) &&
               aligned(residual, eo));
  const Rows o = Rows(out, eo, d).along(n, eo * out_stride);
  HK_CHECK_ARG(!overlaps_itself(o) && !overlap(o, Rows(table, et, d).along(vocab, et * table_stride)) &&
               !overlap(o, Rows(tokens, ei, n)) &&
               !overlap_unless_same(o, Rows(residual, eo, d).along(n, eo * residual_stride)));
  Lookup a{};
  a.table = table, a.tokens = tokens, a.residual = residual, a.out = out, a.wide_tokens = wide_tokens;
  a.vocab = vocab, a.table_stride = table_stride, a.residual_stride = residual_stride, a.out_stride = out_stride;
  a.scale = scale;
  const int e = unit(d, 8, {{table, table_stride, et, vocab}, {residual, residual_stride, eo, n}, {out, out_stride, eo, n}});
  return type == HK_TYPE_F32    ? lookup_to<F32>(a, n, d, e, out_type, stream)
         : type == HK_TYPE_BF16 ? lookup_to<BF16>(a, n, d, e, out_type, stream)
                                : lookup_to<F16>(a, n, d, e, out_type, stream);
}

extern "C" int64_t hk_embedding_workspace(int64_t n, int64_t vocab, int64_t d) {
  return hk::gradient_ok(n, vocab, d) ? hk::gradient_workspace(n, vocab, d).bytes : -1;
}

extern "C" hipError_t hk_embedding_backward(const void* grad, int type, int64_t n, int64_t d, int64_t grad_stride,
                                            const void* tokens, int wide_tokens, float scale, void* grad_table,
                                            int table_type, int64_t vocab, int64_t table_stride, int accumulate,
                                            void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace hk;
  HK_CHECK_ARG(type_ok(type) && type_ok(table_type) && gradient_ok(n, vocab, d));
  HK_CHECK_ARG(grad_stride >= 0 && grad_stride < kStride && table_stride >= 0 && table_stride < kStride);
  if (n == 0 && accumulate) return hipSuccess;
  const int64_t eg = elem(type), et = elem(table_type), ei = wide_tokens ? 8 : 4;
  HK_CHECK_ARG(grad_table && aligned(grad_table, et));
  HK_CHECK_ARG(n == 0 || (grad && tokens && aligned(grad, eg) && aligned(tokens, ei)));
  const Rows o = Rows(grad_table, et, d).along(vocab, et * table_stride);
  HK_CHECK_ARG(!overlaps_itself(o) && !overlap(o, Rows(grad, eg, d).along(n, eg * grad_stride)) &&
               !overlap(o, Rows(tokens, ei, n)));
  const Workspace layout = gradient_workspace(n, vocab, d);
  const int64_t need = layout.bytes;
  if (need > 0) {
    if (workspace) {
      HK_CHECK_ARG(workspace_bytes >= need && aligned16(workspace));
    } else {
      // a graph would keep the stream's workspace, which other graphs and eager calls write too
      if (stream_capturing(stream)) return hipErrorStreamCaptureUnsupported;
      HK_RETURN_IF_ERROR(device_workspace(static_cast<size_t>(need), stream, &workspace));
    }
  }
  Grad a{};
  a.grad = grad, a.tokens = tokens, a.table = grad_table, a.wide_tokens = wide_tokens;
  a.n = n, a.vocab = vocab, a.grad_stride = grad_stride, a.table_stride = table_stride, a.d = static_cast<int>(d);
  a.scale = scale, a.accumulate = accumulate, a.table_elem = static_cast<int>(et);
  a.sorted = static_cast<uint2*>(workspace);
  a.used = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + layout.used);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + layout.part);
  const int e = unit(d, 4, {{grad, grad_stride, eg, n}, {grad_table, table_stride, et, vocab}});
  return type == HK_TYPE_F32    ? gradient_to<F32>(a, e, table_type, stream)
         : type == HK_TYPE_BF16 ? gradient_to<BF16>(a, e, table_type, stream)
                                : gradient_to<F16>(a, e, table_type, stream);
}

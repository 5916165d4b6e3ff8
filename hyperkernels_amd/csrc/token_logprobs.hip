// token_logprobs.hip - log probabilities of given tokens over rows of logits, with the log-sum-exp, the entropy and the
// likeliest alternatives, and the gradient of the first and third. fp32, bf16 or fp16 logits, any row stride and
// alignment.
//
//   lse = log sum_j exp(x_j),  logp = x_token - lse,  H = -sum p log p = log s - u / s
//   with m = max x, s = sum exp(x - m), u = sum (x - m) exp(x - m);
//   dx_j = g ([j = token] - p_j) - h p_j (x_j - lse + H).
// One fp32 number has no room for log s beside a maximum far from 0: logp takes them off one after the other, and so does the
// gradient of rows whose lse is past kFar, for which one workgroup a row reads it twice (2048 rows of 50257 fp32 near
// 1000: 228 us, 140 near 0; 16 of 131072: 94, 12 near 0).
//
// Forward: a workgroup holds a row (or a piece of one) in registers, so it is read once whatever follows: the maximum, then
// both sums against it without any rescaling, then the selection. Rows that are longer than the registers, or too
// few to fill the card, are cut into pieces that a second kernel joins. 16-byte loads from the row's first
// 16-byte boundary on; the up to 2 x 7 elements beside them go one to a lane.
//
// The `top` largest: with W waves, the ceil(top / W)-th largest of each wave's 64 lane maxima is reached by that many
// elements of the wave, so the least of those over the waves is a bound that `top` elements reach and few others do (some
// 60 of 50257 for top = 20). The lanes that hold one put their vectors into LDS, 128 lanes at a time, where all lanes
// look them through and collect (value, index) keys, which are ranked by counting the larger ones. A wave of few words (of a
// short piece, or with most masked) has no such bound or a low one, which many reach: then it is the `top`-th largest of all lane
// maxima, found bit by bit. Where more reach that than the list takes even without those equal to it, `top` passes over
// the row find the next largest.
//
// Measured, rows of 50257: 4096 of bf16 with 5 alternatives 78 us (5.3 TB/s, where the bound is the memory); 8192 of bf16
// without 149 (5.5), their gradient 269 (read and write at 6.1, the copy's rate); 16 of fp32 with 20 alternatives 7.1 + 5.1 us, which is
// latency: load, maximum, sums, selection one after the other. With waves that have no words: 16 rows of bf16, 20 alternatives,
// 14.4 us (a pass for each: 40); 600 rows of 3000, 13.4 (52); 300 rows, 5 alternatives, an eighth of the words masked in a wave's
// share of each 4096, 27 (162).
#include <limits.h>

#include <type_traits>

#include "hk_device.h"
#include "hk_host.h"
#include "hk_overlap.h"

namespace hk {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 64;
constexpr int kMaxPieces = 64;
constexpr int kList = 1024;  // candidates in LDS
constexpr int kMany = 384;  // candidates that take longer to rank than fewer do to find
constexpr int kLanes = 128;  // lanes whose vectors LDS holds
constexpr int kMostVecs = 14;  // 16-byte vectors a lane: with them 80 registers, three workgroups a CU

struct Row {
  const void* x;
  int64_t stride;  // elements
  const void* tokens;
  int wide_tokens;  // int64
  int64_t vocab;
  int64_t rows;
  float *logp, *lse, *entropy, *top_logp;
  int64_t* top_index;
  int top;
  int pieces, piece;  // pieces a row, elements a piece
  // of each piece: (max, s, u, unused), and `top` keys
  float4* part;
  uint64_t* keys;
  int64_t first;  // row of this launch's first workgroup
};

__device__ __forceinline__ int64_t token_of(const void* tokens, int wide, int64_t row) {
  return wide ? static_cast<const int64_t*>(tokens)[row] : static_cast<const int32_t*>(tokens)[row];
}

// (value, index) as a number that is larger for larger values, and for the lower index of equal ones; NaN is under
// all values, and 0 stands for nothing.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);  // -0 is 0
  return v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x7fc00000u : (b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  return (static_cast<uint64_t>(ordered(v)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(uint64_t key) { return value_of(static_cast<uint32_t>(key >> 32)); }
__device__ __forceinline__ int64_t key_index(uint64_t key) {
  return 0xffffffffu - static_cast<uint32_t>(key);
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t k) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_xor(static_cast<unsigned long long>(k), d);
    k = o > k ? o : k;
  }
  return k;
}

// Ranks the n keys of `list` (all different) and hands (rank, key) of the first `top` to put. All threads.
template <int THREADS, class Put>
__device__ __forceinline__ void rank_keys(const uint64_t* list, int n, int top, Put put) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < top) put(rank, mine);
  }
}

template <class F, int THREADS, int V, bool ENT, bool TOP>
__global__ __launch_bounds__(THREADS, THREADS == 64 ? 2 : 6) void logprobs_kernel(Row a) {
  constexpr int kE = F::kPerVec, W = THREADS / 64;
  using S = typename F::storage;
  __shared__ float red[3][W];
  __shared__ uint64_t list[TOP ? kList : 1];
  __shared__ uint4 stash[TOP ? kLanes * V : 1];
  __shared__ uint16_t owner[TOP ? kLanes : 1];
  __shared__ int count, lanes, over;

  const int64_t item = blockIdx.x + a.first * a.pieces, row = a.pieces == 1 ? item : item / a.pieces;
  const int pc = static_cast<int>(item - row * a.pieces);
  const int base = pc * a.piece;  // first element of the piece
  const int n = static_cast<int>(min(a.vocab - base, static_cast<int64_t>(a.piece)));
  const S* x = static_cast<const S*>(a.x) + row * a.stride + base;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;

  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(S));
  const int head = min(off ? kE - off : 0, n), vecs = (n - head) / kE, tail0 = head + vecs * kE;
  uint4 d[V];
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    d[v] = make_uint4(0, 0, 0, 0);
    if (v * THREADS + tid < vecs) d[v] = ld_nt(xv + v * THREADS + tid);
  }
  // one of the elements beside the vectors
  const int odd = tid < head ? tid : tid >= 32 && tid - 32 < n - tail0 ? tail0 + tid - 32 : -1;
  const float x0 = odd >= 0 ? F::load(x, odd) : -INFINITY;

  // calls f(value, index in the piece) for each of the lane's elements
  auto each = [&](auto f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = v * THREADS + tid;
      if (at < vecs) {
        float e[kE];
        F::unpack(d[v], e);
#pragma unroll
        for (int i = 0; i < kE; ++i) f(e[i], head + at * kE + i);
      }
    }
  };
  float mx = x0;
  each([&](float e, int) { mx = fmaxf(mx, e); });

  float m = wave_max(mx);
  if (TOP && tid == 0) count = lanes = over = 0;
  if (W > 1) {
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = red[0][lane & (W - 1)];
    m = row16_reduce(m, MaxOp{});  // W <= 16, and every lane of the row has one of the values
  }
  const float ref = m == -INFINITY ? 0.f : m;  // nothing above -inf: the sums are 0
  float s = 0.f, u = 0.f;
  // as far as the compiler can see these are new: else it keeps the first pass's fp32 values of 16-bit rows
#pragma unroll
  for (int v = 0; v < V; ++v) asm("" : "+v"(d[v].x), "+v"(d[v].y), "+v"(d[v].z), "+v"(d[v].w));
  auto add = [&](float e) {
    const float t = (e - ref) * kLog2e;  // log2 of the term; as one fma it would overflow at fp32's lowest values
    const float p = __builtin_amdgcn_exp2f(t);
    s += p;
    // -inf has p = 0 and counts for nothing; a NaN is in s
    if (ENT) u = __builtin_fmaf(fmaxf(t, -1000.f), p, u);
  };
  if (odd >= 0) add(x0);
  each([&](float e, int) { add(e); });
  s = wave_sum(s);
  if (ENT) u = wave_sum(u);
  if (W > 1) {
    if (lane == 0) red[1][wave] = s, red[2][wave] = u;
    __syncthreads();
    s = u = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += red[1][w], u += red[2][w];
  }
  u *= kLn2;
  const float log_s = __logf(s), lse = ref + log_s;
  if (tid == 0) {
    if (a.pieces > 1) {
      a.part[item] = make_float4(m, s, u, 0.f);
    } else {
      if (a.lse) a.lse[row] = lse;
      if (ENT) a.entropy[row] = log_s - u / s;
      const int64_t t = token_of(a.tokens, a.wide_tokens, row);
      a.logp[row] = t >= 0 && t < n ? F::load(x, t) - ref - log_s : __uint_as_float(0x7fc00000u);
    }
  }
  if constexpr (TOP) {
    auto put = [&](int rank, uint64_t key) {
      if (a.pieces > 1) {
        a.keys[item * a.top + rank] = key;
      } else {
        a.top_logp[row * a.top + rank] = key_value(key) - ref - log_s;
        a.top_index[row * a.top + rank] = key_index(key);
      }
    };
    // the bound
    float left = mx, bound = -INFINITY;
    for (int r = (a.top + W - 1) / W; r > 0; --r) {
      bound = wave_max(left);
      const uint64_t who = __ballot(left == bound);
      if (who == 0 || lane == __ffsll(static_cast<unsigned long long>(who)) - 1) left = -INFINITY;
    }
    if (W > 1) {
      if (lane == 0) red[0][wave] = bound;
      __syncthreads();
      bound = row16_reduce(red[0][lane & (W - 1)], [](float p, float q) { return fminf(p, q); });
    }
    // Where too many are equal to the bound (masked words), those above it are all there are, and then the first of those
    // equal to it. So it is at -inf from the start: fewer lanes than are asked for have any word above that.
    bool above = bound == -INFINITY && s - s == 0.f;
    const auto passes = [&](float e) { return above ? e > bound : !(e < bound); };
    auto collect = [&](float e, int i) {
      if (passes(e)) {
        const int at = atomicAdd(&count, 1);
        if (at < kList) list[at] = key_of(e, base + i);
      }
    };
    int slot = INT_MAX;
    if (mx > bound) atomicAdd(&over, 1);
    if (passes(mx)) {
      slot = atomicAdd(&lanes, 1);
      if (odd >= 0) collect(x0, odd);
    }
    __syncthreads();
    // Where fewer lanes are over it, the bound is the `top`-th largest of all lanes' maxima already, as that of one wave is.
    bool searched = W == 1 || over < a.top;
    const int held = lanes;
    int found = kList + 1;
    if (held <= 2 * kLanes) {  // of more there is a better bound, or too many are equal to it
      for (int from = 0; from < held; from += kLanes) {
        if (slot >= from && slot < from + kLanes) {
          owner[slot - from] = static_cast<uint16_t>(tid);
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (v * THREADS + tid < vecs) stash[(slot - from) * V + v] = d[v];
        }
        __syncthreads();
        for (int i = tid; i < min(held - from, kLanes) * V; i += THREADS) {
          const int at = (i % V) * THREADS + owner[i / V];
          if (at < vecs) {
            float e[kE];
            F::unpack(stash[i], e);
#pragma unroll
            for (int j = 0; j < kE; ++j) collect(e[j], head + at * kE + j);
          }
        }
        __syncthreads();
        if (count > kList) break;
      }
      __syncthreads();
      found = count;
    }
    while (found > kMany) {
      if (!searched) {
        // The `top`-th largest, or a value that a few more reach, four bits at a time: lane t of each wave counts its
        // lanes that reach the number with t there.
        int* const counts = reinterpret_cast<int*>(stash);  // two rounds' [wave][16]
        const uint32_t mine = ordered(mx);
        uint32_t least = 0;
        for (int shift = 28; shift >= 0; shift -= 4) {
          int* const of = counts + (shift & 4) * (4 * W);
          int reach = 0;
#pragma unroll 5
          for (uint32_t t = 1; t < 16; ++t) {
            const int c = __popcll(__ballot(mine >= (least | t << shift)));
            reach = lane == static_cast<int>(t) ? c : reach;
          }
          if (lane < 16) of[16 * wave + lane] = reach;
          __syncthreads();
          reach = 0;
#pragma unroll
          for (int w = 0; w < W; ++w) reach += of[16 * w + (lane & 15)];
          const int digit = __popcll(__ballot(lane > 0 && lane < 16 && reach >= a.top));  // fewer reach more
          least |= static_cast<uint32_t>(digit) << shift;
          if (digit > 0 && __builtin_amdgcn_readlane(reach, digit) <= a.top + W) break;
        }
        bound = value_of(least);
        searched = true;
        above = bound == -INFINITY && s - s == 0.f;
      } else if (!above && bound > -INFINITY) {
        above = true;
      } else {
        break;
      }
      // once more from memory: held until here, the row's registers would spill
      constexpr int kLoads = 8;
      __syncthreads();
      if (tid == 0) count = 0;
      __syncthreads();
      for (int i0 = tid; i0 < n; i0 += kLoads * THREADS) {
        float e[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) e[u] = F::load(x, min(i0 + u * THREADS, n - 1));
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
          if (i0 + u * THREADS < n) collect(e[u], i0 + u * THREADS);
      }
      __syncthreads();
      found = count;
    }
    if (found <= kList) {
      rank_keys<THREADS>(list, found, a.top, put);
      if (tid < 64) {
        int got = found;
        if (above)
          for (int i0 = 0; i0 < n && got < a.top; i0 += 64) {
            const bool it = i0 + lane < n && F::load(x, i0 + lane) == bound;
            const uint64_t those = __ballot(it);
            const int rank = got + __popcll(those & ((uint64_t(1) << lane) - 1));
            if (it && rank < a.top) put(rank, key_of(bound, base + i0 + lane));
            got += __popcll(those);
          }
        // a piece of fewer elements
        for (int i = got + lane; i < a.top; i += 64) put(i, 0);
      }
    } else {
      uint64_t last = ~uint64_t(0);
      for (int r = 0; r < a.top; ++r) {
        uint64_t best = 0;
        for (int i = tid; i < n; i += THREADS) {
          const uint64_t k = key_of(F::load(x, i), base + i);
          if (k < last && k > best) best = k;
        }
        best = wave_max_u64(best);
        if (W > 1) {
          __syncthreads();  // the round before is done with the list
          if (lane == 0) list[wave] = best;
          __syncthreads();
          best = list[0];
#pragma unroll
          for (int w = 1; w < W; ++w) best = list[w] > best ? list[w] : best;
        }
        last = best;
        if (tid == 0) put(r, best);
      }
    }
  }
}

// The same without alternatives, which need no second look at a row: each lane streams over its vectors, four ahead of
// those it adds up, with a maximum of its own that the sums are moved to where it rises. Half the registers, loads
// under way all the time (8192 rows of 50257 bf16, with the gradient: 423 -> 405 us).
constexpr int kAhead = 4;
template <class F, bool ENT>
__global__ __launch_bounds__(512, 8) void logprobs_stream(Row a) {
  constexpr int kE = F::kPerVec, W = 8;
  using S = typename F::storage;
  __shared__ float red[3][W];
  const int64_t item = blockIdx.x + a.first * a.pieces, row = a.pieces == 1 ? item : item / a.pieces;
  const int pc = static_cast<int>(item - row * a.pieces), base = pc * a.piece;
  const int n = static_cast<int>(min(a.vocab - base, static_cast<int64_t>(a.piece)));
  const S* x = static_cast<const S*>(a.x) + row * a.stride + base;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(S));
  const int head = min(off ? kE - off : 0, n), vecs = (n - head) / kE, tail0 = head + vecs * kE;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const int odd = tid < head ? tid : tid >= 32 && tid - 32 < n - tail0 ? tail0 + tid - 32 : -1;

  float m = odd >= 0 ? F::load(x, odd) : -INFINITY;  // NaN: the sums get it below
  const float x0 = m;
  m = m != m ? -INFINITY : m;
  float s = 0.f, u = 0.f, r = m == -INFINITY ? 0.f : m;
  auto add = [&](float e) {
    // not one fma: x log2 e may be past fp32, and loses 2^-24 of a large x
    const float t = (e - r) * kLog2e, p = __builtin_amdgcn_exp2f(t);
    s += p;
    if (ENT) u = __builtin_fmaf(fmaxf(t, -1000.f), p, u);
  };
  if (odd >= 0) add(x0);
  auto load4 = [&](int v0, uint4 (&d)[kAhead]) {
#pragma unroll
    for (int v = 0; v < kAhead; ++v)
      if (v0 + v * 512 + tid < vecs) d[v] = ld_nt(xv + v0 + v * 512 + tid);
  };
  auto take4 = [&](int v0, const uint4 (&d)[kAhead]) {
#pragma unroll
    for (int v = 0; v < kAhead; ++v) {
      if (v0 + v * 512 + tid >= vecs) continue;
      float e[kE];
      F::unpack(d[v], e);
      float top = e[0];
#pragma unroll
      for (int i = 1; i < kE; ++i) top = fmaxf(top, e[i]);
      if (top > m) {
        const float by = (m - top) * kLog2e, f = __builtin_amdgcn_exp2f(by);
        if (ENT) u = m == -INFINITY ? u : f * __builtin_fmaf(fmaxf(by, -1000.f), s, u);
        s = m == -INFINITY ? s : s * f;  // of nothing but a NaN
        m = top;
        r = m;
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) add(e[i]);
    }
  };
  uint4 d0[kAhead], d1[kAhead];
  load4(0, d0);
  for (int v0 = 0; v0 < vecs; v0 += 2 * kAhead * 512) {
    load4(v0 + kAhead * 512, d1);
    take4(v0, d0);
    load4(v0 + 2 * kAhead * 512, d0);
    take4(v0 + kAhead * 512, d1);
  }
  float all = wave_max(m);
  if (lane == 0) red[0][wave] = all;
  __syncthreads();
  all = row16_reduce(red[0][lane & (W - 1)], MaxOp{});
  const float ref = all == -INFINITY ? 0.f : all;
  // to the row's maximum; a lane of nothing above -inf has sums of 0, or NaN
  const float by = (m - ref) * kLog2e, f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(by);
  if (ENT) u = wave_sum(m == -INFINITY ? u : f * __builtin_fmaf(fmaxf(by, -1000.f), s, u));
  s = wave_sum(s * f);
  if (lane == 0) red[1][wave] = s, red[2][wave] = u;
  __syncthreads();
  if (tid != 0) return;
  s = u = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) s += red[1][w], u += red[2][w];
  u *= kLn2;
  if (a.pieces > 1) {
    a.part[item] = make_float4(all, s, u, 0.f);
    return;
  }
  const float log_s = __logf(s);
  if (a.lse) a.lse[row] = ref + log_s;
  if (ENT) a.entropy[row] = log_s - u / s;
  const int64_t t = token_of(a.tokens, a.wide_tokens, row);
  a.logp[row] = t >= 0 && t < n ? F::load(x, t) - ref - log_s : __uint_as_float(0x7fc00000u);
}

// Joins the pieces of a row.
template <class F>
__global__ __launch_bounds__(256) void logprobs_join(Row a) {
  extern __shared__ uint64_t list[];
  __shared__ int count;
  const int64_t row = a.first + blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const bool some = lane < a.pieces;
  const float4 p = some ? a.part[row * a.pieces + lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  const float m = wave_max(p.x), ref = m == -INFINITY ? 0.f : m;
  // a piece of nothing above -inf has sums of 0 against 0
  const float shift = fmaxf(p.x - ref, -1000.f);  // of the piece's reference
  const float f = p.x == -INFINITY ? 0.f : __expf(p.x - ref);
  const float s = wave_sum(p.x == -INFINITY ? p.y : f * p.y);
  const float u = wave_sum(p.x == -INFINITY ? 0.f : f * __builtin_fmaf(shift, p.y, p.z));
  const float log_s = __logf(s);
  if (tid == 0) {
    if (a.lse) a.lse[row] = ref + log_s;
    if (a.entropy) a.entropy[row] = log_s - u / s;
    using S = typename F::storage;
    const int64_t t = token_of(a.tokens, a.wide_tokens, row);
    a.logp[row] = t >= 0 && t < a.vocab ? F::load(static_cast<const S*>(a.x) + row * a.stride, t) - ref - log_s
                                        : __uint_as_float(0x7fc00000u);
    count = 0;
  }
  if (a.top == 0) return;
  __syncthreads();
  // each piece's keys fall: its ceil(top / pieces)-th bounds what can be among the first, as the waves' do above
  const uint64_t* keys = a.keys + row * a.pieces * a.top;
  const int r = (a.top + a.pieces - 1) / a.pieces;
  uint64_t bound = some ? keys[lane * a.top + r - 1] : ~uint64_t(0);
  bound = ~wave_max_u64(~bound);
  for (int i = tid; i < a.pieces * a.top; i += 256) {
    const uint64_t k = keys[i];
    if (k >= bound && k != 0) list[atomicAdd(&count, 1)] = k;
  }
  __syncthreads();
  rank_keys<256>(list, count, a.top, [&](int rank, uint64_t key) {
    a.top_logp[row * a.top + rank] = key_value(key) - ref - log_s;
    a.top_index[row * a.top + rank] = key_index(key);
  });
}

struct Grad {
  const void* x;
  void* dx;
  int64_t stride, dstride;  // elements
  const void* tokens;
  int wide_tokens;
  int vocab;
  const float *lse, *entropy, *g, *h;
  int segments;  // workgroups a row
  int64_t first;
};

constexpr int kGradVecs = 2;  // 16-byte vectors a lane
// p = exp(x - lse) is off by half a step of lse, relative. Below these that is a sixteenth of the result's rounding, or 2^-18 of fp32's;
// past them it has no bound: a row of words at the type's lowest value has an lse with no room for log s.
template <class F>
constexpr float kFar = F::kPerVec == 4 ? 128.f : std::is_same_v<F, F16> ? 1024.f : 4096.f;

// Where a row's elements lie: up to 7 before its first 16-byte boundary, vectors, and up to 7 behind them.
template <class F>
struct Span {
  int head, vecs, odd;  // odd: the one of the others that this lane has, or -1
  __device__ __forceinline__ Span(const typename F::storage* x, int n) {
    constexpr int kE = F::kPerVec;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(*x)), tid = threadIdx.x;
    head = min(off ? kE - off : 0, n), vecs = (n - head) / kE;
    const int tail0 = head + vecs * kE;
    odd = tid < head ? tid : tid >= 32 && tid - 32 < n - tail0 ? tail0 + tid - 32 : -1;
  }
};

// A row's maximum, and the logarithm of its sum of exponentials against that, by all of the workgroup's 256 lanes.
constexpr int kFarVecs = 4;  // in flight
template <class F>
__device__ __forceinline__ void row_parts(const typename F::storage* x, const Span<F>& at, float& ref, float& log_s) {
  constexpr int kE = F::kPerVec;
  __shared__ float red[2][4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint4* xv = reinterpret_cast<const uint4*>(x + at.head);
  float m = at.odd >= 0 ? F::load(x, at.odd) : -INFINITY;
  float s = m == -INFINITY ? 0.f : 1.f;
  for (int v0 = tid; v0 < at.vecs; v0 += 256 * kFarVecs) {
    uint4 d[kFarVecs];
#pragma unroll
    for (int u = 0; u < kFarVecs; ++u)
      if (v0 + 256 * u < at.vecs) d[u] = xv[v0 + 256 * u];
#pragma unroll
    for (int u = 0; u < kFarVecs; ++u) {
      if (v0 + 256 * u >= at.vecs) continue;
      float e[kE], top = m;
      F::unpack(d[u], e);
#pragma unroll
      for (int i = 0; i < kE; ++i) top = fmaxf(top, e[i]);
      if (top > m) {
        s *= __builtin_amdgcn_exp2f((m - top) * kLog2e);
        m = top;
      }
      const float r = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < kE; ++i) s += __builtin_amdgcn_exp2f((e[i] - r) * kLog2e);
    }
  }
  const float wm = wave_max(m);
  if (lane == 0) red[0][wave] = wm;
  __syncthreads();
  ref = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  s = wave_sum(m == -INFINITY ? s : s * __builtin_amdgcn_exp2f((m - ref) * kLog2e));
  if (lane == 0) red[1][wave] = s;
  __syncthreads();
  log_s = __logf((red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
}

// VEC: rows of x and dx have the same place within 16 bytes, so the vectors of one are vectors of the other.
template <class F, bool VEC>
__global__ __launch_bounds__(256) void logprobs_grad(Grad a) {
  constexpr int kE = F::kPerVec;
  using S = typename F::storage;
  const int64_t item = blockIdx.x + a.first, row = item / a.segments;
  const int seg = static_cast<int>(item - row * a.segments), tid = threadIdx.x;
  const S* x = static_cast<const S*>(a.x) + row * a.stride;
  S* dx = static_cast<S*>(a.dx) + row * a.dstride;
  const float lse = a.lse[row];
  const int64_t token = token_of(a.tokens, a.wide_tokens, row);
  float g = a.g ? a.g[row] : 0.f;
  const float h = a.h ? a.h[row] : 0.f, ent = a.h ? a.entropy[row] : 0.f;
  // a row without a softmax has no gradient either: what the terms below leave out would hide it
  const float all = lse - lse == 0.f ? g : __uint_as_float(0x7fc00000u);
  auto from_log = [&](float log_p, int i) {
    const float d = fmaxf(log_p, -200.f);  // exp of less is 0, and -inf has to be no factor
    const float p = __builtin_amdgcn_exp2f(d * kLog2e);
    const float t = p * __builtin_fmaf(h, d + ent, all);
    return (i == token ? g : 0.f) - t;
  };
  const Span<F> at(x, a.vocab);
  const uint4* xv = reinterpret_cast<const uint4*>(x + at.head);
  uint4* ov = reinterpret_cast<uint4*>(dx + at.head);
  if (fabsf(lse) >= kFar<F> && fabsf(lse) < INFINITY) {
    // the row's first workgroup does all of it: what the others would write may lie on what this one reads
    if (seg > 0) return;
    float ref, log_s;
    row_parts<F>(x, at, ref, log_s);
    auto one = [&](float e, int i) { return from_log((e - ref) - log_s, i); };
    if (!VEC) {
      for (int i = tid; i < a.vocab; i += 256) F::store(dx, i, one(F::load(x, i), i));
      return;
    }
    if (at.odd >= 0) F::store(dx, at.odd, one(F::load(x, at.odd), at.odd));
    for (int v0 = tid; v0 < at.vecs; v0 += 256 * kFarVecs) {
      uint4 d[kFarVecs];
#pragma unroll
      for (int u = 0; u < kFarVecs; ++u)
        if (v0 + 256 * u < at.vecs) d[u] = xv[v0 + 256 * u];
#pragma unroll
      for (int u = 0; u < kFarVecs; ++u) {
        const int v = v0 + 256 * u;
        if (v >= at.vecs) continue;
        float e[kE];
        F::unpack(d[u], e);
#pragma unroll
        for (int i = 0; i < kE; ++i) e[i] = one(e[i], at.head + v * kE + i);
        st_nt(ov + v, F::pack(e));
      }
    }
    return;
  }
  auto one = [&](float e, int i) { return from_log(e - lse, i); };
  if (VEC) {
    uint4 d[kGradVecs];
    const int v0 = seg * (256 * kGradVecs) + tid;
#pragma unroll
    for (int v = 0; v < kGradVecs; ++v)
      if (v0 + 256 * v < at.vecs) d[v] = ld_nt(xv + v0 + 256 * v);
    if (seg == 0 && at.odd >= 0) F::store(dx, at.odd, one(F::load(x, at.odd), at.odd));
#pragma unroll
    for (int v = 0; v < kGradVecs; ++v) {
      const int i0 = v0 + 256 * v;
      if (i0 < at.vecs) {
        float e[kE];
        F::unpack(d[v], e);
#pragma unroll
        for (int i = 0; i < kE; ++i) e[i] = one(e[i], at.head + i0 * kE + i);
        st_nt(ov + i0, F::pack(e));
      }
    }
  } else {
    const int per = 256 * kGradVecs * kE, from = seg * per;
    for (int i = from + tid; i < min(from + per, a.vocab); i += 256) F::store(dx, i, one(F::load(x, i), i));
  }
}

// ---- host --------------------------------------------------------------------------------------------------
size_t elem(int type) { return type == HK_TYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
constexpr int64_t kMaxVocab = int64_t(1) << 20;
constexpr int64_t kGrid = int64_t(1) << 22;  // workgroups a launch

bool shape_ok(int type, int64_t rows, int64_t vocab, int64_t stride) {
  return type >= HK_TYPE_F32 && type <= HK_TYPE_F16 && rows >= 0 && rows < (int64_t(1) << 31) && vocab >= 1 &&
         vocab <= kMaxVocab && stride >= 0 && stride < (int64_t(1) << 40);
}

struct Plan {
  int threads, vecs, pieces, piece;
};
// One wave a row where it holds it and there are rows for all, else 512 lanes. Rows are cut where they pass 14 vectors a
// lane, and where they leave CUs idle, into pieces of 2048 elements at least.
Plan plan(int type, int64_t rows, int64_t vocab, bool top) {
  const int e = 16 / static_cast<int>(elem(type)), cus = device_cu_count();
  Plan p{512, 4, 1, static_cast<int>(vocab)};
  // a piece may begin anywhere within 16 bytes: its vectors are no more than those of its elements
  if (vocab <= 64 * 4 * e && (rows >= 2 * cus || vocab <= 256)) {
    p.threads = 64;
    return p;
  }
  int64_t pieces = top ? ceil_div(vocab, int64_t(512) * kMostVecs * e) : 1;
  if (rows < cus) {
    const int64_t fill = ceil_div(cus, rows > 0 ? rows : 1), most = vocab / 2048;
    pieces = pieces > (fill < most ? fill : most) ? pieces : (fill < most ? fill : most);
  }
  if (pieces > kMaxPieces) pieces = kMaxPieces;
  p.pieces = static_cast<int>(pieces < 1 ? 1 : pieces);
  p.piece = static_cast<int>(ceil_div(ceil_div(vocab, p.pieces), e) * e);
  p.pieces = static_cast<int>(ceil_div(vocab, p.piece));
  p.vecs = p.piece <= 512 * 4 * e ? 4 : kMostVecs;
  return p;
}
int64_t workspace_bytes_of(const Plan& p, int64_t rows, int top) {
  return p.pieces > 1 ? rows * p.pieces * (16 + 8 * int64_t(top)) : 0;
}

template <class F, int THREADS, int V>
hipError_t launch(const Row& a, int64_t blocks, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(blocks)), block(THREADS);
  if (a.top > 0) {
    if (a.entropy) hipLaunchKernelGGL((logprobs_kernel<F, THREADS, V, true, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((logprobs_kernel<F, THREADS, V, false, true>), grid, block, 0, stream, a);
  } else if constexpr (THREADS == 64) {
    if (a.entropy) hipLaunchKernelGGL((logprobs_kernel<F, THREADS, V, true, false>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((logprobs_kernel<F, THREADS, V, false, false>), grid, block, 0, stream, a);
  }
  return launch_status();
}
template <class F>
hipError_t stream_rows(const Row& a, int64_t blocks, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(blocks));
  if (a.entropy) hipLaunchKernelGGL((logprobs_stream<F, true>), grid, dim3(512), 0, stream, a);
  else hipLaunchKernelGGL((logprobs_stream<F, false>), grid, dim3(512), 0, stream, a);
  return launch_status();
}
template <class F>
hipError_t run(Row a, const Plan& p, hipStream_t stream) {
  const int64_t step = kGrid / p.pieces;
  for (a.first = 0; a.first < a.rows; a.first += step) {
    const int64_t rows = a.rows - a.first < step ? a.rows - a.first : step, blocks = rows * p.pieces;
    HK_RETURN_IF_ERROR(p.threads == 64 ? (launch<F, 64, 4>(a, blocks, stream))
                       : a.top == 0    ? stream_rows<F>(a, blocks, stream)
                       : p.vecs == 4   ? (launch<F, 512, 4>(a, blocks, stream))
                                       : (launch<F, 512, kMostVecs>(a, blocks, stream)));
    if (p.pieces > 1) {
      hipLaunchKernelGGL(logprobs_join<F>, dim3(static_cast<unsigned>(rows)), dim3(256),
                         static_cast<size_t>(8) * p.pieces * a.top, stream, a);
      HK_RETURN_IF_ERROR(launch_status());
    }
  }
  return hipSuccess;
}

template <class F>
hipError_t run_grad(Grad a, int64_t rows, bool vec, hipStream_t stream) {
  const int64_t items = rows * a.segments;
  for (a.first = 0; a.first < items; a.first += kGrid) {
    const dim3 grid(static_cast<unsigned>(items - a.first < kGrid ? items - a.first : kGrid));
    if (vec) hipLaunchKernelGGL((logprobs_grad<F, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((logprobs_grad<F, false>), grid, dim3(256), 0, stream, a);
    HK_RETURN_IF_ERROR(launch_status());
  }
  return hipSuccess;
}

}  // namespace
}  // namespace hk

extern "C" int64_t hk_token_logprobs_workspace(int type, int64_t rows, int64_t vocab, int top) {
  if (!hk::shape_ok(type, rows, vocab, vocab) || top < 0 || top > hk::kMaxTop || top > vocab) return -1;
  return hk::workspace_bytes_of(hk::plan(type, rows, vocab, top > 0), rows, top);
}

extern "C" hipError_t hk_token_logprobs(const void* logits, int type, int64_t rows, int64_t vocab, int64_t row_stride,
                                        const void* tokens, int wide_tokens, float* logp, float* lse, float* entropy,
                                        int top, float* top_logp, int64_t* top_index, void* workspace,
                                        int64_t workspace_bytes, hipStream_t stream) {
  HK_CHECK_ARG(hk::shape_ok(type, rows, vocab, row_stride) && top >= 0 && top <= hk::kMaxTop && top <= vocab);
  if (rows == 0) return hipSuccess;
  const int64_t es = static_cast<int64_t>(hk::elem(type)), et = wide_tokens ? 8 : 4;
  HK_CHECK_ARG(logits && tokens && logp && hk::aligned(logits, es) && hk::aligned(tokens, et) && hk::aligned(logp, 4) &&
               hk::aligned(lse, 4) && hk::aligned(entropy, 4));
  HK_CHECK_ARG(top == 0 || (top_logp && top_index && hk::aligned(top_logp, 4) && hk::aligned(top_index, 8)));
  const hk::Rows in[2] = {hk::Rows(logits, es, vocab).along(rows, es * row_stride), hk::Rows(tokens, et, rows)};
  const hk::Rows out[5] = {hk::Rows(logp, 4, rows), hk::Rows(lse, 4, rows), hk::Rows(entropy, 4, rows),
                           hk::Rows(top ? top_logp : nullptr, 4, rows * top),
                           hk::Rows(top ? top_index : nullptr, 8, rows * top)};
  for (int i = 0; i < 5; ++i) {
    HK_CHECK_ARG(!hk::overlap(out[i], in[0]) && !hk::overlap(out[i], in[1]));
    for (int j = 0; j < i; ++j) HK_CHECK_ARG(!hk::overlap(out[i], out[j]));
  }
  const hk::Plan p = hk::plan(type, rows, vocab, top > 0);
  hk::Row a{};
  a.x = logits, a.stride = row_stride, a.tokens = tokens, a.wide_tokens = wide_tokens;
  a.vocab = vocab, a.rows = rows, a.logp = logp, a.lse = lse, a.entropy = entropy;
  a.top_logp = top_logp, a.top_index = top_index, a.top = top, a.pieces = p.pieces, a.piece = p.piece;
  if (const int64_t need = hk::workspace_bytes_of(p, rows, top)) {
    if (workspace) {
      HK_CHECK_ARG(workspace_bytes >= need && hk::aligned16(workspace));
    } else {
      // a graph would keep the stream's workspace, which other graphs and eager calls write too
      if (hk::stream_capturing(stream)) return hipErrorStreamCaptureUnsupported;
      HK_RETURN_IF_ERROR(hk::device_workspace(static_cast<size_t>(need), stream, &workspace));
    }
    a.part = static_cast<float4*>(workspace);
    a.keys = reinterpret_cast<uint64_t*>(a.part + rows * p.pieces);
  }
  return type == HK_TYPE_F32    ? hk::run<hk::F32>(a, p, stream)
         : type == HK_TYPE_BF16 ? hk::run<hk::BF16>(a, p, stream)
                                : hk::run<hk::F16>(a, p, stream);
}

extern "C" hipError_t hk_token_logprobs_backward(const void* logits, int type, int64_t rows, int64_t vocab,
                                                 int64_t row_stride, const void* tokens, int wide_tokens,
                                                 const float* lse, const float* entropy, const float* grad_logp,
                                                 const float* grad_entropy, void* grad, int64_t grad_stride,
                                                 hipStream_t stream) {
  HK_CHECK_ARG(hk::shape_ok(type, rows, vocab, row_stride) && hk::shape_ok(type, rows, vocab, grad_stride));
  if (rows == 0) return hipSuccess;
  const int64_t es = static_cast<int64_t>(hk::elem(type)), et = wide_tokens ? 8 : 4;
  HK_CHECK_ARG(logits && tokens && lse && grad && hk::aligned(logits, es) && hk::aligned(grad, es) &&
               hk::aligned(tokens, et) && hk::aligned(lse, 4) && hk::aligned(entropy, 4) && hk::aligned(grad_logp, 4) &&
               hk::aligned(grad_entropy, 4) && (!grad_entropy || entropy));
  const hk::Rows x = hk::Rows(logits, es, vocab).along(rows, es * row_stride);
  const hk::Rows dx = hk::Rows(grad, es, vocab).along(rows, es * grad_stride);
  HK_CHECK_ARG(!hk::overlaps_itself(dx) && !hk::overlap_unless_same(dx, x) &&
               !hk::overlap(dx, hk::Rows(tokens, et, rows)));
  for (const float* p : {lse, entropy, grad_logp, grad_entropy}) HK_CHECK_ARG(!hk::overlap(dx, hk::Rows(p, 4, rows)));
  hk::Grad a{};
  a.x = logits, a.dx = grad, a.stride = row_stride, a.dstride = grad_stride;
  a.tokens = tokens, a.wide_tokens = wide_tokens, a.vocab = static_cast<int>(vocab);
  a.lse = lse, a.entropy = entropy, a.g = grad_logp, a.h = grad_entropy;
  a.segments = static_cast<int>(hk::ceil_div(vocab, 256 * hk::kGradVecs * (16 / es)));
  const uintptr_t apart = reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad);
  const bool vec = (apart & 15) == 0 && (rows == 1 || (es * (row_stride - grad_stride)) % 16 == 0);
  return type == HK_TYPE_F32    ? hk::run_grad<hk::F32>(a, rows, vec, stream)
         : type == HK_TYPE_BF16 ? hk::run_grad<hk::BF16>(a, rows, vec, stream)
                                : hk::run_grad<hk::F16>(a, rows, vec, stream);
}

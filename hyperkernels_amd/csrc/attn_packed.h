// attn_packed.h - device pieces shared by the packed 16-bit attention kernels (attn_packed_fwd.hip,
// attn_packed_bwd.hip): which rows a workgroup owns, the LDS layout of a tile and the matrix products.
//
// Sequence s has queries cu_q[s] .. cu_q[s + 1] and keys cu_k[s] .. cu_k[s + 1]. The `group` query heads that share
// one key head are taken together: row r of (sequence, key head) is query r / group of head r % group, so a tile
// of rows reads each key once whatever the group is, and a single token of a large group still fills a tile.
#pragma once

#include <math.h>

#include <atomic>
#include <type_traits>

#include "hk_device.h"
#include "hk_host.h"
#include "hk_overlap.h"

namespace hk {
namespace packed {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

#define HK_LDS __attribute__((address_space(3)))

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The element types: the product of 32 x 16 and 16 x 32 (lane l of A holds row l % 32 and k = 8 (l / 32) .. + 7, of B
// column l % 32 and the same k; element i of C is row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32), and the
// rounding of two fp32 values (to nearest even).
struct TypeBF16 {
  using format = BF16;
  static constexpr bool kNarrow = false;  // fp32's exponents
  static __device__ __forceinline__ f32x16_t mfma(s16x8_t a, s16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x, y}, bf16x2_t));
  }
  static __device__ __forceinline__ f32x2_t unpack(uint32_t w) {
    return f32x2_t{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  }
};
struct TypeF16 {
  using format = F16;
  static constexpr bool kNarrow = true;
  static __device__ __forceinline__ f32x16_t mfma(s16x8_t a, s16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x, y}, f16x2_t));
  }
  static __device__ __forceinline__ f32x2_t unpack(uint32_t w) {
    return __builtin_convertvector(__builtin_bit_cast(f16x2_t, w), f32x2_t);
  }
};

// A tensor [tokens, heads, head_dim]: strides in bytes.
struct Tensor {
  char* p;
  int64_t m, h;
};

struct Args {
  Tensor q, k, v, o, dout, dq, dk, dv;
  float* lse;
  int64_t lse_stride;  // elements between heads
  const int32_t *cu_q, *cu_k;
  int64_t q_tokens, k_tokens;
  int n, group, k_heads, d;  // sequences, query heads a key head, key heads, elements a head
  int causal;
  float scale;
  int tiles;   // slots of row (or key) tiles, all sequences
  int splits;  // backward: shares of a key tile's rows, each with partial results of its own
  int chunk, most;  // forward: key tiles a share, and how many shares there are room for
  int32_t* shares;  // forward: of each row
  int cus;
  int near;  // backward: groups divide 32 rows, which lie within 2^30 bytes
  float* part;   // partial results
  float2* stat;  // forward: (max, sum) of them
  float* delta;  // backward: rowsum(dout * o), log-sum-exp in log 2 and dout's exponent, each [q head][token]
};

__host__ __device__ inline int64_t clamp64(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

// At most this many tiles of B rows, `group` rows a token, whatever the lengths of the n sequences are: the grid goes by
// the numbers of tokens and sequences alone, so nothing about the lengths has to be known on the host.
__host__ __device__ inline int64_t slots(int64_t tokens, int n, int group, int B) {
  return tokens * group / B + n;
}

struct Seq {
  int64_t q0, k0;  // first query and key
  int mq, mk;      // how many of them
  int tile, tiles; // the workgroup's tile of this sequence, and how many it has
};
// Starts outside 0 .. tokens count as the nearer of both and lengths under 0 as 0, so whatever cu holds the rows are
// some of the tensor.

__device__ __forceinline__ int wave_add(int v) {
  auto dpp = [](int x, auto ctrl) {
    return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  v += dpp(v, std::integral_constant<int, detail::kDppXor1>{});
  v += dpp(v, std::integral_constant<int, detail::kDppXor2>{});
  v += dpp(v, std::integral_constant<int, detail::kDppHalfMirror>{});
  v += dpp(v, std::integral_constant<int, detail::kDppMirror>{});
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] + r[1];
  const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(h[0] + h[1]);
}

// Workgroup L's (tile, share, key head): the tiles of all sequences by falling number within the sequence, which under
// the causal mask is by falling work, each with all its shares and heads side by side. Where the card holds all of them at
// once (per_cu a CU), workgroup L and L + P (P CUs) are likely to meet on one CU, so every other P of them run backwards:
// a CU gets heavy and light ones. (8192 tokens in 13 documents, 12 heads of 64, sequence by sequence instead: forward
// 34.6 us against 29.8, dk and dv 59 against 48.)
// More than 64 sequences, one a lane, are taken one after the other. ByQ: tiles of queries (`group` rows each), else of
// keys. cu_q and cu_k may be one array over tensors of different lengths, so the starts do not tell.
template <bool ByQ>
__device__ __forceinline__ bool find_item(const Args& a, int group, int B, int per_cu, Seq& q, int& share, int& head) {
  const int lane = threadIdx.x & 63, per_tile = a.k_heads * a.splits;
  const int32_t* const cu = ByQ ? a.cu_q : a.cu_k;
  const int64_t tokens = ByQ ? a.q_tokens : a.k_tokens;
  if (a.n > 64) {
    // slot floor(cu[s] group / B) + s is the first of sequence s, which leaves each the tiles it needs
    const int x = a.tiles - 1 - static_cast<int>(blockIdx.x) / per_tile, rest = blockIdx.x % per_tile;
    int lo = 0, hi = a.n;
    do {
      const int step = (hi - lo + 63) >> 6;
      const int i = lo + lane * step;
      const bool before = i < hi && clamp64(cu[i < hi ? i : lo], 0, tokens) * group / B + i <= x;
      const int count = __popcll(__ballot(before));
      if (count == 0) return false;
      lo += (count - 1) * step;
      hi = min(hi, lo + step);
    } while (hi - lo > 1);
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int64_t q0 = clamp64(a.cu_q[lo], 0, a.q_tokens), q1 = clamp64(a.cu_q[lo + 1], q0, a.q_tokens);
    const int64_t k0 = clamp64(a.cu_k[lo], 0, a.k_tokens), k1 = clamp64(a.cu_k[lo + 1], k0, a.k_tokens);
    q.q0 = q0, q.mq = static_cast<int>(q1 - q0);
    q.k0 = k0, q.mk = static_cast<int>(k1 - k0);
    q.tile = x - static_cast<int>((ByQ ? q0 : k0) * group / B + lo);
    q.tiles = static_cast<int>(((ByQ ? q.mq : q.mk) * static_cast<int64_t>(group) + B - 1) / B);
    share = rest / a.k_heads, head = rest - share * a.k_heads;
    return q.tile >= 0 && q.tile < q.tiles;
  }
  // all that is read, at once; numbers of rows and keys fit 32 bits, and so does a sequence's last tile's end
  const int i0 = min(lane, a.n - 1), tq = static_cast<int>(a.q_tokens), tk = static_cast<int>(a.k_tokens);
  const int cq0 = a.cu_q[i0], cq1 = a.cu_q[i0 + 1], ck0 = a.cu_k[i0], ck1 = a.cu_k[i0 + 1];
  const int q0 = min(max(cq0, 0), tq), q1 = min(max(cq1, q0), tq);
  const int k0 = min(max(ck0, 0), tk), k1 = min(max(ck1, k0), tk);
  const uint32_t len = static_cast<uint32_t>(ByQ ? q1 - q0 : k1 - k0) * group;
  const int count = lane < a.n ? static_cast<int>((len + B - 1) / B) : 0;  // the sequence's tiles
  auto over = [&](int t) { return wave_add(max(count - t, 0)); };  // tiles of number t and over
  const int total = over(0) * per_tile;
  int L = blockIdx.x;
  if (L >= total) return false;
  if (total > a.cus && total <= per_cu * a.cus) {
    const int P = a.cus, round = L / P;
    if (round & 1) L = round * P + min(P, total - round * P) - 1 - (L - round * P);
  }
  const int x = L / per_tile, rest = L - x * per_tile;
  // the last t with more than x tiles of number t and over; counts are under 2^24, which floats hold
  int lo = 0, above = 0, hi = __builtin_amdgcn_readfirstlane(static_cast<int>(wave_max(static_cast<float>(count))));
  if (a.n == 1) {
    lo = hi - 1 - x, above = x;
  } else {
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, c = over(mid);
      if (c > x) lo = mid;
      else hi = mid, above = c;
    }
  }
  // the (x - above)-th sequence with such a tile
  const uint64_t with = __ballot(count > lo);
  const bool it = count > lo && __popcll(with & ((uint64_t(1) << lane) - 1)) == x - above;
  const int s = __ffsll(static_cast<unsigned long long>(__ballot(it))) - 1;
  if (s < 0) return false;
  auto of = [&](int v) { return __builtin_amdgcn_readlane(v, s); };
  q.q0 = of(q0), q.mq = of(q1 - q0), q.k0 = of(k0), q.mk = of(k1 - k0);
  q.tile = lo, q.tiles = of(count);
  share = rest / a.k_heads, head = rest - share * a.k_heads;
  return lo >= 0 && lo < q.tiles;  // whatever sequences that overlap add up to
}

// Item L of those that give every row tile's keys in shares of a.chunk tiles of B_k keys, sequence after sequence: shares
// are alike, so their order is free. At most 64 sequences.
__device__ __forceinline__ bool find_share(const Args& a, int B, int B_k, int L, Seq& q, int& share, int& shares,
                                           int& head) {
  const int lane = threadIdx.x & 63;
  const int i0 = min(lane, a.n - 1), tq = static_cast<int>(a.q_tokens), tk = static_cast<int>(a.k_tokens);
  const int cq0 = a.cu_q[i0], cq1 = a.cu_q[i0 + 1], ck0 = a.cu_k[i0], ck1 = a.cu_k[i0 + 1];
  const int q0 = min(max(cq0, 0), tq), q1 = min(max(cq1, q0), tq);
  const int k0 = min(max(ck0, 0), tk), k1 = min(max(ck1, k0), tk);
  const int tiles = static_cast<int>((static_cast<uint32_t>(q1 - q0) * a.group + B - 1) / B);
  const int parts = max(1, (k1 - k0 + B_k * a.chunk - 1) / (B_k * a.chunk));
  const int items = lane < a.n ? tiles * parts : 0;
  int upto = items;  // of the sequences to here
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int below = __shfl_up(upto, d);
    if (lane >= d) upto += below;
  }
  const int x = L / a.k_heads;
  head = L - x * a.k_heads;
  const uint64_t behind = __ballot(upto > x);
  if (behind == 0) return false;
  const int s = __ffsll(static_cast<unsigned long long>(behind)) - 1;
  auto of = [&](int v) { return __builtin_amdgcn_readlane(v, s); };
  const int r = x - of(upto - items);
  shares = of(parts);
  q.q0 = of(q0), q.mq = of(q1 - q0), q.k0 = of(k0), q.mk = of(k1 - k0);
  q.tiles = of(tiles);
  q.tile = r / shares;
  share = r - q.tile * shares;
  return r >= 0 && q.tile < q.tiles;
}

// LDS tile: rows of D elements (2 D bytes) as they lie in memory, the 16-byte chunk c of row r at chunk c ^ swz(r).
// gfx950's LDS serves 256 bytes a cycle over 64 banks: 16 lanes of a 16-byte read, which here take 16 consecutive
// rows at one chunk, and 32 lanes of a transposing read, which take 4 consecutive rows by 4 consecutive chunks; both
// cover the banks once, so one copy of a tile serves the products over its columns and those over its rows.
template <int D>
__device__ __forceinline__ int swz(int r) {
  if (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int at_chunk(int r, int c) {
  return r * (2 * D) + ((c ^ swz<D>(r)) << 4);
}

// 16 bytes a lane from memory into LDS (1 KiB a wave at lds_addr + 16 lane), past the registers. In asm, so that the
// compiler does not wait for every copy before each LDS read: the kernel waits (vmcnt) before the barrier that
// publishes a tile. m0 is an input operand; an SGPR base just written by a VALU needs 5 wait states, which the
// compiler's own checks do not add inside asm.
__device__ __forceinline__ void copy16_to_lds(const void* sbase, int voff, unsigned lds_addr) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_addr));
}
__device__ __forceinline__ void copy16_to_lds(const void* addr, unsigned lds_addr) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(addr), "{m0}"(lds_addr));
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Copies of N consecutive tokens of one head by 4 waves. Rows behind the sequence's last and chunks behind the
// head's last element read the last one: they stay inside the sequence, and what they meet is masked (rows) or
// zero on the other side of the product (columns of queries) or not stored (columns of values). A wave's copies are 4
// kRows rows apart, at which the chunks lie alike: in whole tiles they differ by a scalar.
template <int D, int N>
struct KeyCopy {
  static constexpr int kChunks = D / 8, kRows = 64 / kChunks;  // rows a wave and instruction
  static constexpr int kCopies = N / (4 * kRows);              // instructions a wave
  const char* base;  // the sequence's first token
  int64_t step;      // of N tokens
  int stride, row, chunk16, off;
  __device__ KeyCopy(const Tensor& x, const Seq& q, int head, int wave, int lane, int d) {
    base = x.p + q.k0 * x.m + head * x.h;
    step = N * x.m;
    stride = static_cast<int>(x.m);
    row = wave * kRows + lane / kChunks;
    chunk16 = 16 * min((lane % kChunks) ^ swz<D>(row), d / 8 - 1);
    off = row * stride + chunk16;
  }
  // tile t of a sequence of n tokens
  __device__ __forceinline__ void operator()(int t, int n, int wave, unsigned lds) const {
    const char* p = base + t * step;
    const int last = n - 1 - t * N;
    if (last >= N - 1) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16_to_lds(p + i * (4 * kRows) * static_cast<int64_t>(stride), off, lds + 1024 * (wave + 4 * i));
    } else {
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        copy16_to_lds(p, min(row + 4 * kRows * i, last) * stride + chunk16, lds + 1024 * (wave + 4 * i));
    }
  }
};

// Lane offsets of a tile's reads. rows(): 16 bytes of row r at 8 (2 s + lane / 32) elements, the operand of a product
// over columns. cols(): the operand of a product over rows, elements 0 .. 3 of rows R + 4 h + {0 .. 3} and 4 .. 7 of
// rows R + 8 + 4 h + {0 .. 3} (h = lane / 32) at column 32 b + lane % 32: the order in which a C block's column holds
// its rows, so that block's values are the other operand as they are.
template <int D>
struct Reads {
  int row[D / 16];
  int col[2][D / 32];
  __device__ explicit Reads(int lane) {
    const int c = lane & 31, h = lane >> 5;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) row[s] = at_chunk<D>(c, 2 * s + h);
    // within each 16 lanes, lane j reads 4 elements of row j / 4 at columns 4 (j % 4)
    const int j = lane & 15, x = 16 * ((lane >> 4) & 1) + 4 * (j & 3);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int b = 0; b < D / 32; ++b)
        col[e][b] = at_chunk<D>(8 * e + 4 * h + (j >> 2), 4 * b + (x >> 3)) + 2 * (x & 7);
    // kept in registers: the compiler would form them anew in every tile
#pragma unroll
    for (int s = 0; s < D / 16; ++s) asm volatile("" : "+v"(row[s]));
#pragma unroll
    for (int b = 0; b < D / 32; ++b) asm volatile("" : "+v"(col[0][b]), "+v"(col[1][b]));
  }
  __device__ __forceinline__ s16x8_t rows(const char HK_LDS* tile, int first, int s) const {
    return *reinterpret_cast<const s16x8_t HK_LDS*>(tile + first * (2 * D) + row[s]);
  }
  __device__ __forceinline__ s16x8_t cols(const char HK_LDS* tile, int first, int b) const {
    const char HK_LDS* p = tile + first * (2 * D);
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t HK_LDS*)(p + col[0][b]));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t HK_LDS*)(p + col[1][b]));
    return s16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};

// A block of zeros that stays in 16 registers, for the first product of a sum: the compiler sets the sum's own registers
// to zero instead, 16 instructions a block.
__device__ __forceinline__ f32x16_t zero_block() {
  f32x16_t z = {};
  asm volatile("" : "+v"(z));
  return z;
}

// A row's operand of a product over columns from memory: element s is columns 16 s + 8 h .. + 7, zero behind d.
template <int D>
__device__ __forceinline__ void load_row(const char* p, int h, int d, s16x8_t (&x)[D / 16]) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const int c = 16 * s + 8 * h;
    x[s] = c < d ? *reinterpret_cast<const s16x8_t*>(p + 2 * c) : s16x8_t{};
  }
}

// P of two 16-row halves of a C block as operands.
template <class T>
__device__ __forceinline__ void pack_block(const f32x16_t& p, s16x8_t (&x)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = T::pack(p[8 * s + 2 * i], p[8 * s + 2 * i + 1]);
    x[s] = __builtin_bit_cast(s16x8_t, w);
  }
}

// Stores a lane's column of a C block set (32 b + 8 (i / 4) + 4 h + i % 4 of row r, elements < d) times f.
template <class T, int D>
__device__ __forceinline__ void store_row(char* p, int h, int d, const f32x16_t (&o)[D / 32], float f) {
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * b + 8 * g + 4 * h;
      if (c < d)
        *reinterpret_cast<u32x2_t*>(p + 2 * c) = u32x2_t{T::pack(o[b][4 * g] * f, o[b][4 * g + 1] * f),
                                                         T::pack(o[b][4 * g + 2] * f, o[b][4 * g + 3] * f)};
    }
}

// ---- host --------------------------------------------------------------------------------------------------
// Shapes, strides and pointers of a call. Keys' strides are bounded so that a tile's offsets fit 32 bits.
inline hipError_t check(const hk_attn_packed_params* p, int type, bool backward) {
  HK_CHECK_ARG(p != nullptr && (type == HK_TYPE_BF16 || type == HK_TYPE_F16));
  HK_CHECK_ARG(p->num_seqs >= 0 && p->q_tokens >= 0 && p->k_tokens >= 0);
  HK_CHECK_ARG(p->k_heads >= 1 && p->q_heads >= 1 && p->q_heads % p->k_heads == 0);
  HK_CHECK_ARG(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0);
  HK_CHECK_ARG(p->scale > 0.f && p->scale < INFINITY);
  constexpr int64_t kMost = INT32_MAX / 2;  // rows and keys are counted in 32 bits, a tile's worth behind the last
  HK_CHECK_ARG(p->q_tokens <= kMost / p->q_heads && p->k_tokens <= kMost);
  // workgroups of one launch, of 512 threads at most: 2^32 threads are more than it takes
  constexpr int64_t kGrid = int64_t(1) << 22;
  HK_CHECK_ARG((slots(p->q_tokens, p->num_seqs, p->q_heads / p->k_heads, 32)) <= kGrid / p->k_heads);
  HK_CHECK_ARG(slots(p->k_tokens, p->num_seqs, 1, 128) <= kGrid / p->k_heads);
  if (p->num_seqs == 0) return hipSuccess;
  HK_CHECK_ARG(p->cu_q && p->cu_k && (reinterpret_cast<uintptr_t>(p->cu_q) & 3) == 0 &&
               (reinterpret_cast<uintptr_t>(p->cu_k) & 3) == 0);
  auto tensor = [](const void* t, int64_t m, int64_t h) {
    constexpr int64_t kStride = int64_t(1) << 40;
    return t && aligned16(t) && m >= 0 && h >= 0 && m % 8 == 0 && h % 8 == 0 && m < kStride && h < kStride;
  };
  auto keys = [&](const void* t, int64_t m, int64_t h) { return tensor(t, m, h) && m <= (int64_t(1) << 23); };
  if (p->q_tokens > 0) {
    HK_CHECK_ARG(tensor(p->q, p->q_strideM, p->q_strideH) && tensor(p->o, p->o_strideM, p->o_strideH));
    HK_CHECK_ARG((reinterpret_cast<uintptr_t>(p->lse) & 3) == 0 && (!backward || p->lse));
    HK_CHECK_ARG(!p->lse || p->lse_strideH >= 0);
    HK_CHECK_ARG(!backward || (tensor(p->dout, p->do_strideM, p->do_strideH) &&
                               tensor(p->dq, p->dq_strideM, p->dq_strideH)));
  }
  if (p->k_tokens > 0) {
    HK_CHECK_ARG(keys(p->k, p->k_strideM, p->k_strideH) && keys(p->v, p->v_strideM, p->v_strideH));
    HK_CHECK_ARG(!backward || (tensor(p->dk, p->dk_strideM, p->dk_strideH) &&
                               tensor(p->dv, p->dv_strideM, p->dv_strideH)));
  }
  return hipSuccess;
}

// Whether what a call writes shares no memory with anything else of it.
inline bool outputs_apart(const hk_attn_packed_params* p, bool backward) {
  auto rows = [&](const void* t, int64_t tokens, int heads, int64_t m, int64_t h) {
    return Rows(tokens > 0 ? t : nullptr, 2, p->head_dim).along(heads, 2 * h).along(tokens, 2 * m);
  };
  const int64_t tq = p->q_tokens, tk = p->k_tokens;
  const Rows lse = Rows(p->lse, 4, tq).along(p->q_heads, 4 * p->lse_strideH);
  const Rows o = rows(p->o, tq, p->q_heads, p->o_strideM, p->o_strideH);
  const Rows in[7] = {rows(p->q, tq, p->q_heads, p->q_strideM, p->q_strideH),
                      rows(p->k, tk, p->k_heads, p->k_strideM, p->k_strideH),
                      rows(p->v, tk, p->k_heads, p->v_strideM, p->v_strideH),
                      Rows(p->cu_q, 4, p->num_seqs + 1),
                      Rows(p->cu_k, 4, p->num_seqs + 1),
                      backward ? rows(p->dout, tq, p->q_heads, p->do_strideM, p->do_strideH) : Rows(nullptr, 2, 1),
                      backward ? lse : Rows(nullptr, 4, 1)};
  const Rows out[3] = {backward ? rows(p->dq, tq, p->q_heads, p->dq_strideM, p->dq_strideH) : o,
                       backward ? rows(p->dk, tk, p->k_heads, p->dk_strideM, p->dk_strideH) : lse,
                       backward ? rows(p->dv, tk, p->k_heads, p->dv_strideM, p->dv_strideH) : Rows(nullptr, 2, 1)};
  for (int i = 0; i < 3; ++i) {
    if (overlaps_itself(out[i]) || (backward && overlap(out[i], o))) return false;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return false;
    for (const Rows& x : in)
      if (overlap(out[i], x)) return false;
  }
  return true;
}

inline Args make_args(const hk_attn_packed_params* p) {
  Args a{};
  auto t = [](const void* x, int64_t m, int64_t h) {
    return Tensor{static_cast<char*>(const_cast<void*>(x)), 2 * m, 2 * h};
  };
  a.q = t(p->q, p->q_strideM, p->q_strideH), a.k = t(p->k, p->k_strideM, p->k_strideH);
  a.v = t(p->v, p->v_strideM, p->v_strideH), a.o = t(p->o, p->o_strideM, p->o_strideH);
  a.dout = t(p->dout, p->do_strideM, p->do_strideH), a.dq = t(p->dq, p->dq_strideM, p->dq_strideH);
  a.dk = t(p->dk, p->dk_strideM, p->dk_strideH), a.dv = t(p->dv, p->dv_strideM, p->dv_strideH);
  a.lse = p->lse, a.lse_stride = p->lse_strideH;
  a.cu_q = p->cu_q, a.cu_k = p->cu_k;
  a.q_tokens = p->q_tokens, a.k_tokens = p->k_tokens;
  a.n = p->num_seqs, a.group = p->q_heads / p->k_heads, a.k_heads = p->k_heads, a.d = p->head_dim;
  a.causal = p->is_causal ? 1 : 0;
  a.scale = p->scale;
  a.splits = 1, a.cus = device_cu_count();
  return a;
}

int64_t forward_workspace(const hk_attn_packed_params* p);

// The workspace of a call: the caller's, or the stream's.
inline hipError_t workspace(int64_t need, void* given, int64_t given_bytes, hipStream_t stream, void** out) {
  *out = given;
  if (need == 0) return hipSuccess;
  if (given) {
    HK_CHECK_ARG(given_bytes >= need && aligned16(given));
    return hipSuccess;
  }
  // a graph would keep the stream's workspace, which other graphs and eager calls write too
  if (stream_capturing(stream)) return hipErrorStreamCaptureUnsupported;
  return device_workspace(static_cast<size_t>(need), stream, out);
}

// Launches one kernel, whose LDS is past the 64 KiB that need no asking.
template <auto Kernel, int kLds, int kThreads = 256>
hipError_t launch(dim3 grid, const Args& a, hipStream_t stream) {
  if constexpr (kLds > 0) {
    static std::atomic<uint64_t> asked;  // a bit a device
    int dev = 0;
    HK_RETURN_IF_ERROR(hipGetDevice(&dev));
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (dev > 63 || !(asked.load(std::memory_order_relaxed) & bit)) {
      HK_RETURN_IF_ERROR(hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
      asked.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  hipLaunchKernelGGL(Kernel, grid, dim3(kThreads), kLds, stream, a);
  return launch_status();
}

}  // namespace packed
}  // namespace hk

// attn_packed_bwd.hip - the gradients of packed 16-bit attention (attn_packed_fwd.hip): with p = exp(s - lse),
// dp = dout v^T, delta = rowsum(dout * o) and ds = p (dp - delta),
//   dv = p^T dout,  dq = scale ds k,  dk = scale ds^T q.
//
// Two kernels, each of which owns what it writes, so nothing is added atomically and every sum has a fixed order; that
// forms s and dp twice (seven products instead of five). attn_packed_dq goes by rows like the forward (S^T = K Q^T and
// dP^T = V dO^T with a row a lane, dS^T the operand of dQ^T += K^T dS^T as it lies) and leaves delta and lse for
// attn_packed_dkv, which goes by keys: S = Q K^T and dP = dO V^T with a key a lane, P and dS the operands of
// dV^T += dO^T P and dK^T += Q^T dS as they lie. The rows of a group's heads are one loop there, which sums them.
// P and dS are rounded to 16 bits for the products, as the inputs are; everything else is fp32. That makes the norm of
// the gradients' error sqrt(2) of what rounding them leaves. delta from the o that was rounded adds p (dout . o's
// error) to dS, 2 / (n - 1) of that rounding's square over n equal keys: rows of up to 128 keys, where it would be most
// of the error, take delta = sum p dp instead, from one more pass over the first one or two tiles of keys in workgroups
// that have such rows. dS is as small as P and dout together (1e-7 for a dout of 1e-3 over 1000 keys), which is under
// fp16's normal range: there it is formed for dout times a power of two, of its row in attn_packed_dq (an addend of the
// exponent), of the rows so far in attn_packed_dkv, where dK is moved to the next when it grows. Large values could
// take such a dS past fp16's end: attn_packed_dq looks at each block's largest and moves the row's power, and dQ with
// it (4096 tokens, 16 heads of 128: 126 -> 131 us; a second pass over such tiles instead, for want of registers, 139);
// attn_packed_dkv has the sum of a key's |v|, which bounds its dP before the loop. There P, as small as one over the
// number of a row's keys, is held times 2^12.
//
// Measured, causal: 13 documents, 8192 tokens, 12 heads of 64, bf16: dq 32, dk and dv 42 us; sequences of 2048, 1001 and
// 333, 16 heads on 4 of 128, fp16: 54, and 86 + 17 to join. Bound by each workgroup's chain (products, exponentials, products that
// need them) at two to three waves a SIMD. Both in one launch, every other workgroup a tile of either, took as long (7.6 for delta,
// then 84). Five products, with dS handed from one to the other, have not been tried.
#include "attn_packed.h"

namespace hk {
namespace packed {

constexpr int kLeast = -40;  // an exponent under any of fp16
constexpr int kShort = 128;  // keys of a row up to which delta is formed from p and dp
constexpr float kMost = 65504.f;  // fp16's largest number
constexpr int kUp = 12;  // fp16: P is held times 2^12, normal numbers to 2^-26: rows of more than 2^14 keys have P under 2^-14

// The exponent e of |x| < 2^e, kLeast for 0.
__device__ __forceinline__ int exponent(float x) { return x == 0.f ? kLeast : __builtin_amdgcn_frexp_expf(x); }

template <int D, int KG>
struct DqShape {
  static constexpr int kRows = 128 / KG;
  static constexpr int kKeys = KG == 4 ? 128 : 64;
  static constexpr int kBlocks = kKeys / KG / 32;
  static constexpr int kFew = kShort / kKeys;  // tiles of keys of rows whose delta is formed from p and dp
  static constexpr int kTile = kKeys * D * 2;
  static constexpr int kStage = 2 * kTile;
  static constexpr int kPitch = D + 4;
  static constexpr int kExchange = KG == 1 ? 0 : 4 * 32 * kPitch * 4;
  static constexpr int kPerCu = D == 64 ? (KG == 4 ? 2 : 3) : (KG == 4 ? 1 : 2);  // workgroups a CU
  static constexpr int kLds = 2 * kStage > kExchange ? 2 * kStage : kExchange;
};

template <class T, int D, int KG>
__global__ __launch_bounds__(256, KG == 4 ? 1 : D == 64 ? 3 : 2) void attn_packed_dq(Args a) {
  using S = DqShape<D, KG>;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  char HK_LDS* const lds = (char HK_LDS*)lds_raw;

  Seq q;
  int share, kh;
  if (!find_item<true>(a, a.group, S::kRows, S::kPerCu, q, share, kh)) return;
  const int rows = q.mq * a.group, r0 = q.tile * S::kRows;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int kg = wave % KG, w0 = r0 + 32 * (wave / KG);
  const int row = w0 + c, rr = min(row, rows - 1);
  const int tok = rr / a.group, qh = kh * a.group + rr - tok * a.group;
  const int ahead = q.mk - q.mq;
  const int lim = a.causal ? tok + ahead : q.mk - 1;
  const int lim_lo = __builtin_amdgcn_readfirstlane(lim);
  const int lim_hi = __builtin_amdgcn_readlane(lim, 31);
  const int last_tok = min(r0 + S::kRows, rows) - 1;
  const int end = a.causal ? min(q.mk, last_tok / a.group + ahead + 1) : q.mk;
  const int t1 = end > 0 ? (end + S::kKeys - 1) / S::kKeys : 0;

  const KeyCopy<D, S::kKeys> copy_k(a.k, q, kh, wave, lane, a.d), copy_v(a.v, q, kh, wave, lane, a.d);
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds));
  auto fetch = [&](int t) {
    const unsigned to = lds0 + (t & 1) * S::kStage;
    copy_k(t, q.mk, wave, to);
    copy_v(t, q.mk, wave, to + S::kTile);
  };
  const bool few = (a.causal ? r0 / a.group + ahead : q.mk - 1) < kShort;  // the first row, and so some, has few keys
  if (t1 > 0) fetch(0);
  if (few && S::kFew > 1 && t1 > 1) fetch(1);

  const Reads<D> rd(lane);
  const float sc = a.scale * kLog2e;
  const f32x16_t zero = zero_block();
  s16x8_t qx[D / 16], gx[D / 16];
  float delta = 0.f, lse2;
  // scores, with -inf where a key is masked, and dp of the 32 keys from key0 on, at kt and vt in LDS
  auto products = [&](const char HK_LDS* kt, const char HK_LDS* vt, int key0, f32x16_t& s, f32x16_t& dp) {
    s = T::mfma(rd.rows(kt, 0, 0), qx[0], zero);
#pragma unroll
    for (int i = 1; i < D / 16; ++i) s = T::mfma(rd.rows(kt, 0, i), qx[i], s);
    dp = T::mfma(rd.rows(vt, 0, 0), gx[0], zero);
#pragma unroll
    for (int i = 1; i < D / 16; ++i) dp = T::mfma(rd.rows(vt, 0, i), gx[i], dp);
    if (key0 + 31 > lim_lo) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 8 * (i >> 2) + 4 * h + (i & 3) > lim) s[i] = -INFINITY;
    }
  };
  int grow = 0;
  {
    const int64_t at = q.q0 + tok;
    load_row<D>(a.q.p + at * a.q.m + qh * a.q.h, h, a.d, qx);
    load_row<D>(a.dout.p + at * a.dout.m + qh * a.dout.h, h, a.d, gx);
    const float lse = a.lse[qh * a.lse_stride + at];
    // a row that sees nothing has exponentials of 0
    lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
    if (few) {
      wait_copies();
      barrier();
      for (int key0 = 0; lim_lo < kShort && key0 < kShort && key0 <= lim_hi; key0 += 32) {
        const char HK_LDS* kt = lds + key0 / S::kKeys * S::kStage + key0 % S::kKeys * (2 * D);
        f32x16_t s, dp;
        products(kt, kt + S::kTile, key0, s, dp);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          delta = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sc, -lse2)), dp[i], delta);
      }
    }
    if (lim_hi >= kShort) {
      s16x8_t ox[D / 16];
      load_row<D>(a.o.p + at * a.o.m + qh * a.o.h, h, a.d, ox);
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const u32x4_t x = __builtin_bit_cast(u32x4_t, ox[s]), y = __builtin_bit_cast(u32x4_t, gx[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2_t u = T::unpack(x[i]), w = T::unpack(y[i]);
          sum += u[0] * w[0] + u[1] * w[1];
        }
      }
      delta = lim < kShort ? delta : sum;
    }
    delta = half32_reduce(delta, AddOp{});
    if constexpr (T::kNarrow) {
      float most = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const u32x4_t y = __builtin_bit_cast(u32x4_t, gx[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2_t w = T::unpack(y[i]);
          most = fmaxf(most, fmaxf(fabsf(w[0]), fabsf(w[1])));
        }
      }
      grow = max(exponent(half32_reduce(most, MaxOp{})), exponent(delta) - 14);  // dout under 2^grow, delta under 2^14 of that
    }
    if (kg == 0 && h == 0 && row < rows) {
      float* st = a.delta + qh * a.q_tokens + at;
      st[0] = delta;
      const int64_t all = static_cast<int64_t>(a.k_heads) * a.group * a.q_tokens;
      st[all] = T::kNarrow ? lse2 - kUp : lse2;
      if (T::kNarrow) st[2 * all] = static_cast<float>(grow);
    }
    if (T::kNarrow) lse2 += static_cast<float>(grow);
  }
  f32x16_t dq[D / 32];
#pragma unroll
  for (int b = 0; b < D / 32; ++b) dq[b] = f32x16_t{};

  for (int t = 0; t < t1; ++t) {
    wait_copies();
    barrier();
    if (t + 1 < t1 && (!few || t + 1 >= S::kFew)) fetch(t + 1);
    const int key0 = t * S::kKeys + 32 * S::kBlocks * kg;
    const char HK_LDS* kt = lds + (t & 1) * S::kStage + 32 * S::kBlocks * kg * (2 * D);
    const char HK_LDS* vt = kt + S::kTile;
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n) {
      if (key0 + 32 * n > lim_hi) break;
      f32x16_t s, dp;
      products(kt + 32 * n * (2 * D), vt + 32 * n * (2 * D), key0 + 32 * n, s, dp);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sc, -lse2)) * (dp[i] - delta);
      if constexpr (T::kNarrow) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[i]));
        if (__any(top > kMost)) {  // of large values: the row's power of two moves, and dq with it
          top = half32_reduce(top, MaxOp{});
          const int up = top > kMost && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
          const float f = ldexpf(1.f, -up);
          grow += up, lse2 += static_cast<float>(up);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] *= f;
#pragma unroll
          for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[b][i] *= f;
        }
      }
      s16x8_t ds[2];
      pack_block<T>(s, ds);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int b = 0; b < D / 32; ++b) dq[b] = T::mfma(rd.cols(kt, 32 * n + 16 * e, b), ds[e], dq[b]);
    }
  }

  const float out = T::kNarrow ? ldexpf(a.scale, grow) : a.scale;
  if constexpr (KG > 1) {
    // the sums of the waves that have the same rows
    constexpr int R = S::kRows;
    float HK_LDS* ex = (float HK_LDS*)lds;
    wait_copies();
    barrier();
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t HK_LDS*>(ex + (kg * R + w0 - r0 + c) * S::kPitch + 32 * b + 8 * g + 4 * h) =
            f32x4_t{dq[b][4 * g] * out, dq[b][4 * g + 1] * out, dq[b][4 * g + 2] * out, dq[b][4 * g + 3] * out};
    __syncthreads();
    const int er = threadIdx.x / (2 * KG), e0 = threadIdx.x % (2 * KG);
    if (r0 + er >= rows) return;
    const int et = (r0 + er) / a.group, eh = kh * a.group + (r0 + er) - et * a.group;
    char* op = a.dq.p + (q.q0 + et) * a.dq.m + eh * a.dq.h;
#pragma unroll
    for (int u = 0; u < D / (8 * KG); ++u) {
      const int col = 8 * KG * u + 4 * e0;
      f32x4_t x = {};
#pragma unroll
      for (int g = 0; g < KG; ++g)
        x += *reinterpret_cast<const f32x4_t HK_LDS*>(ex + (g * R + er) * S::kPitch + col);
      if (col < a.d)
        *reinterpret_cast<u32x2_t*>(op + 2 * col) = u32x2_t{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
    }
    return;
  }
  if (row >= rows) return;
  store_row<T, D>(a.dq.p + (q.q0 + tok) * a.dq.m + qh * a.dq.h, h, a.d, dq, out);
}

// A wave takes 32 keys and, of every tile of 64 rows, all or (HALVES = 2, two waves a key block) 32 rows. Heads past 64
// elements have 128 accumulators of dK and dV a lane: K and V then stay in LDS, beside the rows' tiles, so that a lane's
// registers are few enough for two waves a SIMD. Halves are added through LDS at the end.
template <int D>
struct DkvShape {
  static constexpr int kKeys = 128;
  static constexpr int kRows = D == 128 ? 64 : 32;  // rows a tile
  static constexpr int kHalves = D == 128 ? 2 : 1, kThreads = 256 * kHalves;
  static constexpr int kTile = kRows * D * 2;
  static constexpr int kStage = 2 * kTile + 3 * 64 * 4;  // Q, dO, delta, lse, exponent (of 64 rows)
  static constexpr int kHeld = 2 * kKeys * D * 2;  // K, V
  static constexpr int kPitch = D + 4;
  static constexpr int kExchange = kHalves == 2 ? kKeys * kPitch * 4 : 0;
  static constexpr int kNorms = kHeld + 2 * kStage;  // fp16: of the keys' values
  static constexpr int kLds = kNorms + 4 * kKeys > kExchange ? kNorms + 4 * kKeys : kExchange;
};

__device__ __forceinline__ void copy4_to_lds(const void* sbase, int voff, unsigned lds_addr) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_addr));
}
__device__ __forceinline__ void copy4_to_lds(const void* addr, unsigned lds_addr) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, off" ::"v"(addr), "{m0}"(lds_addr));
}

template <class T, int D, bool SPLIT>
__global__ __launch_bounds__(DkvShape<D>::kThreads, D == 64 ? 3 : 2) void attn_packed_dkv(Args a) {
  using S = DkvShape<D>;
  constexpr int kWaves = S::kThreads / 64;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  char HK_LDS* const lds = (char HK_LDS*)lds_raw;

  Seq q;
  int share, kh;
  if (!find_item<false>(a, 1, S::kKeys, S::kHalves == 2 ? 1 : 3, q, share, kh)) return;
  // under the causal mask the first keys meet the most rows: they go first
  const int k0 = (q.tiles - 1 - q.tile) * S::kKeys;
  const int rows = q.mq * a.group, ahead = q.mk - q.mq;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int kb = wave & 3, half = S::kHalves == 2 ? wave >> 2 : 0;
  const int kw = k0 + 32 * kb, key = kw + c, kk = min(key, q.mk - 1);
  // key j is seen by queries from j - ahead on: rows from group times that on
  auto first_row = [&](int j) { return a.causal ? min(max(j - ahead, 0) * a.group, rows) : 0; };
  const int from = first_row(kk);
  const int from_lo = __builtin_amdgcn_readfirstlane(from), from_hi = __builtin_amdgcn_readlane(from, 31);

  int t0 = first_row(k0) / S::kRows, t1 = (rows + S::kRows - 1) / S::kRows;
  if (SPLIT) {
    const int per = (t1 - t0 + a.splits - 1) / a.splits;
    t0 += share * per;
    t1 = min(t1, t0 + per);
  }

  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds));
  constexpr int kChunks = D / 8, kCopyRows = 64 / kChunks, kCopies = S::kRows / (kWaves * kCopyRows);
  const int64_t heads = static_cast<int64_t>(a.k_heads) * a.group;
  // A wave's copies are 32 rows apart. Where groups divide that, whole tiles differ by scalars.
  static_assert(kWaves * kCopyRows == 32, "copies are 32 rows apart");
  const int lr = wave * kCopyRows + lane / kChunks;
  const int ch = 16 * min((lane % kChunks) ^ swz<D>(lr), a.d / 8 - 1);
  constexpr int kStats = T::kNarrow ? 3 : 2;
  int off_q = 0, off_g = 0, off_d = 0, per32 = 0;
  if (a.near) {
    per32 = 32 / a.group;
    const int tok = lr / a.group, hd = lr - tok * a.group;
    off_q = static_cast<int>(tok * a.q.m + hd * a.q.h) + ch;
    off_g = static_cast<int>(tok * a.dout.m + hd * a.dout.h) + ch;
    const int dt = lane / a.group;
    off_d = static_cast<int>(((lane - dt * a.group) * a.q_tokens + dt) * 4);
  }
  const char* const q0p = a.q.p + q.q0 * a.q.m + kh * a.group * a.q.h;
  const char* const g0p = a.dout.p + q.q0 * a.dout.m + kh * a.group * a.dout.h;
  const char* const d0p =
      reinterpret_cast<const char*>(a.delta + ((wave < kStats ? wave : 0) * heads + kh * a.group) * a.q_tokens + q.q0);
  auto fetch = [&](int t) {
    const unsigned to = lds0 + S::kHeld + (t & 1) * S::kStage;
    if (a.near && t * S::kRows + 64 <= rows) {
      const int64_t tok = static_cast<int64_t>(S::kRows / 32 * t) * per32;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        copy16_to_lds(q0p + (tok + i * per32) * a.q.m, off_q, to + 1024 * (wave + kWaves * i));
        copy16_to_lds(g0p + (tok + i * per32) * a.dout.m, off_g, to + S::kTile + 1024 * (wave + kWaves * i));
      }
      if (wave < kStats) copy4_to_lds(d0p + 4 * tok, off_d, to + 2 * S::kTile + 256 * wave);
      return;
    }
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = min(t * S::kRows + lr + 32 * i, rows - 1);
      const int tok = r / a.group, hd = r - tok * a.group;
      copy16_to_lds(q0p + tok * a.q.m + hd * a.q.h + ch, to + 1024 * (wave + kWaves * i));
      copy16_to_lds(g0p + tok * a.dout.m + hd * a.dout.h + ch, to + S::kTile + 1024 * (wave + kWaves * i));
    }
    if (wave < kStats) {
      const int r = min(t * S::kRows + lane, rows - 1);
      const int tok = r / a.group, hd = r - tok * a.group;
      copy4_to_lds(d0p + 4 * (hd * a.q_tokens + tok), to + 2 * S::kTile + 256 * wave);
    }
  };
  float HK_LDS* const norms = (float HK_LDS*)(lds + S::kNorms);
  {
    // columns behind the head's last element are zero: those of Q and dO are copies of others
    constexpr int kLoads = S::kKeys * kChunks / S::kThreads;
    u32x4_t x[kLoads] = {}, y[kLoads] = {};
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (threadIdx.x + i * S::kThreads) / kChunks, ch = threadIdx.x % kChunks;
      const int64_t tok = q.k0 + min(k0 + r, q.mk - 1);
      if (8 * ch < a.d) {
        x[i] = *reinterpret_cast<const u32x4_t*>(a.k.p + tok * a.k.m + kh * a.k.h + 16 * ch);
        y[i] = *reinterpret_cast<const u32x4_t*>(a.v.p + tok * a.v.m + kh * a.v.h + 16 * ch);
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (threadIdx.x + i * S::kThreads) / kChunks, ch = threadIdx.x % kChunks;
      *reinterpret_cast<u32x4_t HK_LDS*>(lds + at_chunk<D>(r, ch)) = x[i];
      *reinterpret_cast<u32x4_t HK_LDS*>(lds + S::kHeld / 2 + at_chunk<D>(r, ch)) = y[i];
      if constexpr (T::kNarrow) {
        // sum |v| of the key: kChunks lanes have it
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x2_t w = T::unpack(y[i][e]);
          sum += fabsf(w[0]) + fabsf(w[1]);
        }
        sum += detail::dpp<detail::kDppXor1>(sum);
        sum += detail::dpp<detail::kDppXor2>(sum);
        sum += detail::dpp<detail::kDppHalfMirror>(sum);
        if (kChunks == 16) sum += detail::dpp<detail::kDppMirror>(sum);
        if (ch == 0) norms[r] = sum;
      }
    }
  }
  if (t0 < t1) fetch(t0);

  const Reads<D> rd(lane);
  const char HK_LDS* const kt = lds + 32 * kb * (2 * D);
  auto k_of = [&](int i) { return rd.rows(kt, 0, i); };
  auto v_of = [&](int i) { return rd.rows(kt + S::kHeld / 2, 0, i); };
  const float sc = a.scale * kLog2e;
  const f32x16_t zero = zero_block();
  f32x16_t dk[D / 32], dv[D / 32];
#pragma unroll
  for (int b = 0; b < D / 32; ++b) dk[b] = dv[b] = f32x16_t{};
  float grow = kLeast;  // exponent of the dout that dk is formed for, and what it is more than that for large values:
  float more = 0.f;     // |dp| is under sum |v| times 2^grow, which is under 2^(14 + more) times that
  if constexpr (T::kNarrow) {
    wait_copies();
    barrier();
    more = static_cast<float>(max(exponent(norms[32 * kb + c]) - 14, 0));
  }

  for (int t = t0; t < t1; ++t) {
    wait_copies();
    barrier();
    if (t + 1 < t1) fetch(t + 1);
    const char HK_LDS* qt = lds + S::kHeld + (t & 1) * S::kStage;
    const char HK_LDS* gt = qt + S::kTile;
    const float HK_LDS* dl = (const float HK_LDS*)(gt + S::kTile);
    if constexpr (T::kNarrow) {
      const float g = wave_max(dl[128 + lane]);
      if (g > grow) {
        const float f = __builtin_amdgcn_exp2f(grow - g);
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) dk[b][i] *= f;
        grow = g;
      }
    }
    const float shrink = T::kNarrow ? __builtin_amdgcn_exp2f(-grow - more - kUp) : 1.f;
#pragma unroll
    for (int u = 0; u < S::kRows / 32 / S::kHalves; ++u) {
      const int n = S::kHalves == 2 ? half : u;
      const int r0 = t * S::kRows + 32 * n;
      if (r0 + 31 < from_lo) continue;  // none of these rows sees the wave's keys
      f32x16_t s = T::mfma(rd.rows(qt, 32 * n, 0), k_of(0), zero);
#pragma unroll
      for (int i = 1; i < D / 16; ++i) s = T::mfma(rd.rows(qt, 32 * n, i), k_of(i), s);
      f32x16_t dp = T::mfma(rd.rows(gt, 32 * n, 0), v_of(0), zero);
#pragma unroll
      for (int i = 1; i < D / 16; ++i) dp = T::mfma(rd.rows(gt, 32 * n, i), v_of(i), dp);
      if (r0 < from_hi || r0 + 32 > rows) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = r0 + 8 * (i >> 2) + 4 * h + (i & 3);
          if (r < from || r >= rows) s[i] = -INFINITY;
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t de = *reinterpret_cast<const f32x4_t HK_LDS*>(dl + 32 * n + 8 * g + 4 * h);
        const f32x4_t ls = *reinterpret_cast<const f32x4_t HK_LDS*>(dl + 64 + 32 * n + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[4 * g + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + e], sc, -ls[e]));
          dp[4 * g + e] -= de[e];
          if (T::kNarrow) dp[4 * g + e] *= shrink;
          dp[4 * g + e] *= s[4 * g + e];
        }
      }
      s16x8_t p[2], ds[2];
      pack_block<T>(s, p);
      pack_block<T>(dp, ds);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int b = 0; b < D / 32; ++b) dv[b] = T::mfma(rd.cols(gt, 32 * n + 16 * e, b), p[e], dv[b]);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int b = 0; b < D / 32; ++b) dk[b] = T::mfma(rd.cols(qt, 32 * n + 16 * e, b), ds[e], dk[b]);
    }
  }
  if constexpr (T::kNarrow) {
    const float f = __builtin_amdgcn_exp2f(grow + more);
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[b][i] *= f, dv[b][i] *= 1.f / (1 << kUp);
  }
  if constexpr (S::kHalves == 2) {
    // the second half's sums, first of dK, then of dV
    float HK_LDS* ex = (float HK_LDS*)lds + (32 * kb + c) * S::kPitch + 4 * h;
    auto add = [&](f32x16_t (&x)[D / 32]) {
      wait_copies();
      barrier();
      if (half == 1)
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4_t HK_LDS*>(ex + 32 * b + 8 * g) =
                f32x4_t{x[b][4 * g], x[b][4 * g + 1], x[b][4 * g + 2], x[b][4 * g + 3]};
      __syncthreads();
      if (half == 0)
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4_t y = *reinterpret_cast<const f32x4_t HK_LDS*>(ex + 32 * b + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[b][4 * g + e] += y[e];
          }
    };
    add(dk);
    add(dv);
    if (half == 1) return;
  }
  if (key >= q.mk) return;
  if constexpr (SPLIT) {
    float* p = a.part + ((static_cast<int64_t>(share) * a.k_heads + kh) * a.k_tokens + q.k0 + key) * (2 * D);
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * b + 8 * g + 4 * h;
        *reinterpret_cast<f32x4_t*>(p + at) =
            f32x4_t{dk[b][4 * g], dk[b][4 * g + 1], dk[b][4 * g + 2], dk[b][4 * g + 3]};
        *reinterpret_cast<f32x4_t*>(p + D + at) =
            f32x4_t{dv[b][4 * g], dv[b][4 * g + 1], dv[b][4 * g + 2], dv[b][4 * g + 3]};
      }
    return;
  }
  store_row<T, D>(a.dk.p + (q.k0 + key) * a.dk.m + kh * a.dk.h, h, a.d, dk, a.scale);
  store_row<T, D>(a.dv.p + (q.k0 + key) * a.dv.m + kh * a.dv.h, h, a.d, dv, 1.f);
}

// Sums the shares of dk and dv in order: D / 2 lanes a key and key head, four elements of both a lane.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_packed_dkv_join(Args a) {
  constexpr int kLanes = D / 2;
  const int64_t keys = a.k_tokens * a.k_heads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (i >= keys) return;
  const int kh = static_cast<int>(i / a.k_tokens);
  const int64_t tok = i - kh * a.k_tokens;
  if (tok < a.cu_k[0] || tok >= a.cu_k[a.n]) return;
  const int col = 4 * (threadIdx.x % kLanes);  // dk, then dv
  f32x4_t x = {};
  for (int s = 0; s < a.splits; ++s)
    x += *reinterpret_cast<const f32x4_t*>(a.part + (s * keys + i) * (2 * D) + col);
  const bool is_dk = col < D;
  const int at = is_dk ? col : col - D;
  if (at >= a.d) return;
  if (is_dk) x *= a.scale;
  const Tensor& t = is_dk ? a.dk : a.dv;
  *reinterpret_cast<u32x2_t*>(t.p + tok * t.m + kh * t.h + 2 * at) =
      u32x2_t{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
}

// ---- host --------------------------------------------------------------------------------------------------
namespace {

struct Plan {
  int kg, row_tiles, key_tiles, splits;
  int64_t part, stat;  // bytes
};
Plan plan(const hk_attn_packed_params* p) {
  const int group = p->q_heads / p->k_heads, cus = device_cu_count();
  const int64_t rows = p->q_tokens * group, wide = slots(p->q_tokens, p->num_seqs, group, 128) * p->k_heads;
  Plan r{};
  // as the forward; the same sequences: 64 rows 53.7 us, 128 72.6
  r.kg = rows < int64_t(96) * p->num_seqs || wide < cus ? 4 : wide < 2 * cus ? 2 : 1;
  r.row_tiles = static_cast<int>(slots(p->q_tokens, p->num_seqs, group, 128 / r.kg));
  r.key_tiles = static_cast<int>(slots(p->k_tokens, p->num_seqs, 1, 128));
  // Key tiles that leave CUs idle share their rows between workgroups, 256 rows each at least.
  const int64_t wgs = static_cast<int64_t>(r.key_tiles) * p->k_heads;
  const int64_t want = wgs < 2 * cus ? ceil_div(3 * cus, wgs) : 1;
  r.splits = static_cast<int>(clamp64(want, 1, clamp64(rows / p->num_seqs / 256, 1, 64)));
  if (r.splits > 1) r.part = r.splits * p->k_tokens * p->k_heads * (p->head_dim <= 64 ? 64 : 128) * 8;
  r.stat = ceil_div(12 * p->q_tokens * p->q_heads, 16) * 16;
  return r;
}

template <class T, int D>
hipError_t run(Args a, const Plan& r, hipStream_t stream) {
  if (a.q_tokens > 0) {
    a.tiles = r.row_tiles, a.splits = 1;
    const dim3 grid(static_cast<unsigned>(a.tiles) * a.k_heads);
    HK_RETURN_IF_ERROR(r.kg == 1 ? (launch<&attn_packed_dq<T, D, 1>, DqShape<D, 1>::kLds>(grid, a, stream))
                           : r.kg == 2 ? (launch<&attn_packed_dq<T, D, 2>, DqShape<D, 2>::kLds>(grid, a, stream))
                                       : (launch<&attn_packed_dq<T, D, 4>, DqShape<D, 4>::kLds>(grid, a, stream)));
  }
  if (a.k_tokens == 0) return hipSuccess;
  a.tiles = r.key_tiles, a.splits = r.splits;
  auto span = [&](const Tensor& t) { return 32 / a.group * t.m + a.group * t.h; };
  constexpr int64_t kNear = int64_t(1) << 30;
  a.near = 32 % a.group == 0 && span(a.q) < kNear && span(a.dout) < kNear && a.group * a.q_tokens < kNear / 4;
  const unsigned x = static_cast<unsigned>(a.tiles) * a.k_heads;
  if (r.splits == 1) return launch<&attn_packed_dkv<T, D, false>, DkvShape<D>::kLds, DkvShape<D>::kThreads>(dim3(x), a, stream);
  HK_RETURN_IF_ERROR((launch<&attn_packed_dkv<T, D, true>, DkvShape<D>::kLds, DkvShape<D>::kThreads>(dim3(x * r.splits), a, stream)));
  const int64_t keys = a.k_tokens * a.k_heads;
  return launch<&attn_packed_dkv_join<T, D>, 0>(dim3(static_cast<unsigned>(ceil_div(keys, 512 / D))), a, stream);
}
template <class T>
hipError_t by_width(const Args& a, const Plan& r, hipStream_t stream) {
  return a.d <= 64 ? run<T, 64>(a, r, stream) : run<T, 128>(a, r, stream);
}

}  // namespace
}  // namespace packed
}  // namespace hk

using namespace hk::packed;

extern "C" int64_t hk_attn_packed_workspace(const hk_attn_packed_params* p, int type, int backward) {
  if (check(p, type, backward != 0) != hipSuccess) return -1;
  if (!backward) return forward_workspace(p);
  if (p->num_seqs == 0 || p->q_tokens + p->k_tokens == 0) return 0;
  const Plan r = plan(p);
  return r.part + r.stat;
}

extern "C" hipError_t hk_attn_packed_backward(const hk_attn_packed_params* p, int type, void* ws,
                                              int64_t workspace_bytes, hipStream_t stream) {
  HK_RETURN_IF_ERROR(check(p, type, true));
  if (p->num_seqs == 0 || p->q_tokens + p->k_tokens == 0) return hipSuccess;
  HK_CHECK_ARG(outputs_apart(p, true));
  const Plan r = plan(p);
  HK_RETURN_IF_ERROR(workspace(r.part + r.stat, ws, workspace_bytes, stream, &ws));
  Args a = make_args(p);
  a.part = static_cast<float*>(ws);
  a.delta = reinterpret_cast<float*>(static_cast<char*>(ws) + r.part);
  return type == HK_TYPE_BF16 ? by_width<TypeBF16>(a, r, stream) : by_width<TypeF16>(a, r, stream);
}

// attn_packed_fwd.hip - attention over packed sequences, bf16 or fp16, causal or not, query heads in groups that
// share a key head: o = softmax(scale q k^T) v and the log-sum-exp of each row.
//
// A workgroup of 4 waves owns 128 rows (32 a wave) or, where there are few, 32 rows, whose keys its waves share
// (KG = 4). The scores are formed transposed, S^T = K Q^T: a lane holds one row's scores, so the running maximum is a
// reduction in registers and one exchange with lane + 32, and the exponentials are, as they lie, the operand of
// O^T += V^T P^T. P is rounded to 16 bits for that product (half a step of the type, as the inputs are; the sum that
// divides it is of the fp32 values); scores, maximum, sum and O are fp32.
// Tiles of keys and values go from memory to LDS past the registers, the next one while this one is used.
//
// Measured, bf16, causal: 8192 tokens, 16 heads on 4 of 128, 277 us (0.99 PFLOP/s, three quarters of the matrix product's
// rate; MFMA busy half of the time, the softmax's VALU work the rest: the waves of a SIMD overlap them only in part). 13
// documents, 8192 tokens, 12 heads of 64, 28 us (10 at that rate): the longest tile is a chain of 16 key tiles of 1.3 us.
// A token each over 1 to 4000 keys: the keys and values are the bound; shares 14.7 us (3.2 TB/s), join 3.9.
#include <algorithm>

#include "attn_packed.h"

namespace hk {
namespace packed {

constexpr float kLazy = 8.f;

template <int D, int KG>
struct FwdShape {
  static constexpr int kRows = 128 / KG;
  static constexpr int kKeys = KG == 4 ? 128 : 64;  // keys a tile
  static constexpr int kBlocks = kKeys / KG / 32;   // blocks of 32 keys a wave
  static constexpr int kTile = kKeys * D * 2;       // bytes
  static constexpr int kStage = 2 * kTile;
  static constexpr int kPitch = D + 4;  // floats a row of the exchange
  static constexpr int kExchange = KG == 1 ? 0 : 4 * 32 * (kPitch * 4 + 8);
  static constexpr int kPerCu = (KG == 4 ? 128 : 256) / D;  // workgroups that a CU holds
  static constexpr int kLds = 2 * kStage > kExchange ? 2 * kStage : kExchange;
};

// One tile of rows over all of its keys, or (SPLIT) over one share of them.
template <class T, int D, int KG, bool SPLIT>
__device__ __forceinline__ void attend(const Args& a, const Seq& q, int kh, int share, int shares,
                                       char HK_LDS* const lds) {
  using S = FwdShape<D, KG>;
  const int rows = q.mq * a.group, r0 = q.tile * S::kRows;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int kg = wave % KG, w0 = r0 + 32 * (wave / KG);
  const int row = w0 + c, rr = min(row, rows - 1);
  const int tok = rr / a.group, qh = kh * a.group + rr - tok * a.group;
  const int ahead = q.mk - q.mq;  // row of query i sees keys 0 .. i + ahead
  const int lim = a.causal ? tok + ahead : q.mk - 1;
  const int lim_lo = __builtin_amdgcn_readfirstlane(lim);  // rows rise, and with them the limits
  const int lim_hi = __builtin_amdgcn_readlane(lim, 31);

  const int last_tok = min(r0 + S::kRows, rows) - 1;
  const int end = a.causal ? min(q.mk, last_tok / a.group + ahead + 1) : q.mk;
  int t0 = 0, t1 = end > 0 ? (end + S::kKeys - 1) / S::kKeys : 0;
  if (SPLIT) {
    t0 = share * a.chunk;
    t1 = min(t1, t0 + a.chunk);
  }

  s16x8_t qx[D / 16];
  load_row<D>(a.q.p + (q.q0 + tok) * a.q.m + qh * a.q.h, h, a.d, qx);

  const KeyCopy<D, S::kKeys> copy_k(a.k, q, kh, wave, lane, a.d), copy_v(a.v, q, kh, wave, lane, a.d);
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds));
  auto fetch = [&](int t) {
    const unsigned to = lds0 + (t & 1) * S::kStage;
    copy_k(t, q.mk, wave, to);
    copy_v(t, q.mk, wave, to + S::kTile);
  };
  if (t0 < t1) fetch(t0);
  if constexpr (KG == 4) {
    // the compiler waits for the rows here, with the first tile, and not for the second one later
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(qx[i]));
    if (t0 + 1 < t1) fetch(t0 + 1);
  }

  const Reads<D> rd(lane);
  const float sc = a.scale * kLog2e;
  f32x16_t o[D / 32];
#pragma unroll
  for (int b = 0; b < D / 32; ++b) o[b] = f32x16_t{};
  const f32x16_t zero = zero_block();
  float m = -INFINITY, l = 0.f;  // in units of log 2

  for (int t = t0; t < t1; ++t) {
    if constexpr (KG == 4) {
      // Few workgroups, bound by memory: the tile after the next is fetched as soon as all waves are done with the last,
      // whether or not the next has landed (16 tokens over 1 to 4000 keys of 4 heads of 128, with the join: 21.2 -> 19.3 us).
      if (t > t0) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
        if (t + 1 < t1) fetch(t + 1);
      }
      if (t + 1 < t1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * KeyCopy<D, S::kKeys>::kCopies) : "memory");
      else wait_copies();
      barrier();  // this tile has landed
    } else {
      wait_copies();
      barrier();  // this tile has landed, and every wave is done with the one before it
      if (t + 1 < t1) fetch(t + 1);
    }
    const int key0 = t * S::kKeys + 32 * S::kBlocks * kg;
    if (key0 > lim_hi) continue;  // the wave's rows see none of these
    const char HK_LDS* kt = lds + (t & 1) * S::kStage + 32 * S::kBlocks * kg * (2 * D);
    const char HK_LDS* vt = kt + S::kTile;

    f32x16_t s[S::kBlocks];
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n) {
      s[n] = T::mfma(rd.rows(kt, 32 * n, 0), qx[0], zero);
#pragma unroll
      for (int i = 1; i < D / 16; ++i) s[n] = T::mfma(rd.rows(kt, 32 * n, i), qx[i], s[n]);
    }
    if (key0 + 32 * S::kBlocks - 1 > lim_lo) {
#pragma unroll
      for (int n = 0; n < S::kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * n + 8 * (i >> 2) + 4 * h + (i & 3) > lim) s[n][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
    top = half32_reduce(top, MaxOp{}) * sc;
    // The reference moves only where a score passes it by 2^8 or a row meets its first key: exponentials stay under
    // 2^8 and most tiles leave O alone.
    const bool move = top > m + kLazy || (m == -INFINITY && top > -INFINITY);
    if (__any(move)) {
      const float mn = move ? top : m;
      const float f = move ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
      l *= f;
#pragma unroll
      for (int b = 0; b < D / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= f;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], sc, -base));
        part[i & 3] += s[n][i];
      }
      s16x8_t p[2];
      pack_block<T>(s[n], p);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int b = 0; b < D / 32; ++b) o[b] = T::mfma(rd.cols(vt, 32 * n + 16 * e, b), p[e], o[b]);
    }
    l += (part[0] + part[1]) + (part[2] + part[3]);
  }
  l = half32_reduce(l, AddOp{});

  if constexpr (KG > 1) {
    // the parts of the waves that have the same rows
    constexpr int R = S::kRows;
    float HK_LDS* ex = (float HK_LDS*)lds;
    float HK_LDS* st = ex + 4 * 32 * S::kPitch;
    const int mine = kg * R + w0 - r0 + c;
    wait_copies();
    barrier();
    if (h == 0) st[2 * mine] = m, st[2 * mine + 1] = l;
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t HK_LDS*>(ex + mine * S::kPitch + 32 * b + 8 * g + 4 * h) =
            f32x4_t{o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
    __syncthreads();
    // 2 KG lanes a row, four elements of it at a time
    const int er = threadIdx.x / (2 * KG), e0 = threadIdx.x % (2 * KG);
    float em[KG], mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int g = 0; g < KG; ++g) em[g] = st[2 * (g * R + er)], mx = fmaxf(mx, em[g]);
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      em[g] = __builtin_amdgcn_exp2f(em[g] - ref);
      sum += em[g] * st[2 * (g * R + er) + 1];
    }
    if (r0 + er >= rows) return;
    const int et = (r0 + er) / a.group, eh = kh * a.group + (r0 + er) - et * a.group;
    const int64_t at = static_cast<int64_t>(share * a.k_heads + kh) * a.q_tokens * a.group +
                       q.q0 * a.group + r0 + er;
    const float f = SPLIT ? 1.f : sum > 0.f ? 1.f / sum : sum;  // a NaN stays one
    char* op = a.o.p + (q.q0 + et) * a.o.m + eh * a.o.h;
#pragma unroll
    for (int u = 0; u < D / (8 * KG); ++u) {
      const int col = 8 * KG * u + 4 * e0;
      f32x4_t x = {};
#pragma unroll
      for (int g = 0; g < KG; ++g)
        x += em[g] * *reinterpret_cast<const f32x4_t HK_LDS*>(ex + (g * R + er) * S::kPitch + col);
      if (SPLIT) *reinterpret_cast<f32x4_t*>(a.part + at * D + col) = x;
      else if (col < a.d)
        *reinterpret_cast<u32x2_t*>(op + 2 * col) = u32x2_t{T::pack(x[0] * f, x[1] * f), T::pack(x[2] * f, x[3] * f)};
    }
    if (e0 == 0) {
      if constexpr (SPLIT) {
        a.stat[at] = make_float2(mx, sum);
        if (share == 0) a.shares[at] = shares;
      } else if (a.lse) a.lse[eh * a.lse_stride + q.q0 + et] = (mx + __builtin_amdgcn_logf(sum)) * kLn2;
    }
    return;
  }
  if (row >= rows) return;
  store_row<T, D>(a.o.p + (q.q0 + tok) * a.o.m + qh * a.o.h, h, a.d, o, l > 0.f ? 1.f / l : l);
  if (h == 0 && a.lse) a.lse[qh * a.lse_stride + q.q0 + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <class T, int D, int KG>
__global__ __launch_bounds__(256, KG == 4 ? 1 : 2) void attn_packed_fwd(Args a) {
  using S = FwdShape<D, KG>;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  Seq q;
  int share, kh;
  if (!find_item<true>(a, a.group, S::kRows, S::kPerCu, q, share, kh)) return;
  attend<T, D, KG, false>(a, q, kh, 0, 1, (char HK_LDS*)lds_raw);
}

// The grid cannot know how many shares there are: workgroups take them in turn.
template <class T, int D>
__global__ __launch_bounds__(256, 1) void attn_packed_fwd_shares(Args a) {
  using S = FwdShape<D, 4>;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  Seq q;
  int share, shares, kh;
  for (int L = blockIdx.x; find_share(a, S::kRows, S::kKeys, L, q, share, shares, kh); L += gridDim.x) {
    attend<T, D, 4, true>(a, q, kh, share, shares, (char HK_LDS*)lds_raw);
    __syncthreads();  // the exchange is read
  }
}

// Joins the shares of each row's keys, one wave a row of one query head: a share's maximum and sum a lane, then the
// values of eight shares at a time.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_packed_join(Args a) {
  const int64_t rows = a.q_tokens * a.group;  // of one key head
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= rows * a.k_heads) return;
  const int kh = static_cast<int>(i / rows);
  const int64_t r = i - kh * rows, tok = r / a.group, all = rows * a.k_heads;
  if (tok < a.cu_q[0] || tok >= a.cu_q[a.n]) return;  // of no sequence
  const int qh = kh * a.group + static_cast<int>(r - tok * a.group);
  const int lane = threadIdx.x & 63, shares = min(max(a.shares[i], 1), a.most);
  float m = -INFINITY, l = 0.f;
  for (int s0 = 0; s0 < shares; s0 += 64)
    if (s0 + lane < shares) m = fmaxf(m, a.stat[(s0 + lane) * all + i].x);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  f32x2_t x = {};
  for (int s0 = 0; s0 < shares; s0 += 64) {
    float w = 0.f;
    if (s0 + lane < shares) {
      const float2 st = a.stat[(s0 + lane) * all + i];
      w = __builtin_amdgcn_exp2f(st.x - ref);
      l += w * st.y;
    }
    const int here = min(shares - s0, 64);
    for (int u0 = 0; u0 < here; u0 += 8) {
      f32x2_t p[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        p[u] = f32x2_t{};
        if (u0 + u < here) {
          const float* at = a.part + ((s0 + u0 + u) * all + i) * D;
          if (D == 128) p[u] = reinterpret_cast<const f32x2_t*>(at)[lane];
          else p[u][0] = at[lane];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), (u0 + u) & 63));
        if (u0 + u < here) x += f * p[u];
      }
    }
  }
  l = wave_sum(l);
  const float f = l > 0.f ? 1.f / l : l;
  char* op = a.o.p + tok * a.o.m + qh * a.o.h;
  if (D == 128) {
    if (2 * lane < a.d) reinterpret_cast<uint32_t*>(op)[lane] = T::pack(x[0] * f, x[1] * f);
  } else if (lane < a.d) {
    T::format::store(reinterpret_cast<uint16_t*>(op), lane, x[0] * f);
  }
  if (lane == 0 && a.lse) a.lse[qh * a.lse_stride + tok] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- host --------------------------------------------------------------------------------------------------
namespace {

struct Plan {
  int kg, tiles, chunk, shares;  // shares: at most, 1 where keys are not shared
  int64_t part, stat, count;     // bytes
};
// 128 rows a workgroup where a sequence fills them and every CU gets two of them; 64, whose keys two waves share, where
// it gets one (sequences of 2048, 1001 and 333, 16 heads on 4 of 128: 61.3 -> 52.2 us; with two or more 128 are as fast,
// 13 sequences of 12 heads of 64, or faster, 8192 of 16 heads of 128: 330 against 442); else 32, and where even those
// leave CUs idle their keys are cut into equal shares, as many in all as the card takes at once.
Plan plan(const hk_attn_packed_params* p) {
  const int group = p->q_heads / p->k_heads, cus = device_cu_count(), n = p->num_seqs;
  const int64_t rows = p->q_tokens * group, wide = slots(p->q_tokens, n, group, 128) * p->k_heads;
  Plan r{};
  r.shares = 1;
  if (rows >= int64_t(96) * n && wide >= cus) {
    r.kg = wide < 2 * cus ? 2 : 1;
    r.tiles = static_cast<int>(slots(p->q_tokens, n, group, 128 / r.kg));
    return r;
  }
  r.kg = 4;
  r.tiles = static_cast<int>(slots(p->q_tokens, n, group, 32));
  const int64_t wgs = static_cast<int64_t>(r.tiles) * p->k_heads;
  if (wgs < cus && n <= 64 && p->k_tokens >= int64_t(512) * n) {
    constexpr int kKeys = FwdShape<64, 4>::kKeys;
    static_assert(kKeys == FwdShape<128, 4>::kKeys, "shares go by one size of tile");
    const int at_once = p->head_dim <= 64 ? 2 * cus : cus;
    // key tiles of all row tiles, taken to be spread evenly over the sequences
    const int64_t work = ceil_div(p->k_tokens, kKeys) * ceil_div(rows, int64_t(32) * n) * p->k_heads;
    // a sequence's last share is a part of one: all of them have to be under way at once all the same
    const int64_t whole = std::max<int64_t>(at_once - wgs, at_once / 2);
    r.chunk = static_cast<int>(std::max<int64_t>(2, ceil_div(work, whole)));
    r.shares = static_cast<int>(ceil_div(p->k_tokens, int64_t(r.chunk) * kKeys));
    const int64_t all = p->q_tokens * p->q_heads, D = p->head_dim <= 64 ? 64 : 128;
    r.part = r.shares * all * D * 4, r.stat = r.shares * all * 8, r.count = ceil_div(all * 4, 16) * 16;
  }
  return r;
}

template <class T, int D>
hipError_t run(Args a, const Plan& r, hipStream_t stream) {
  const unsigned x = static_cast<unsigned>(a.tiles) * a.k_heads;
  if (r.kg == 1) return launch<&attn_packed_fwd<T, D, 1>, FwdShape<D, 1>::kLds>(dim3(x), a, stream);
  if (r.kg == 2) return launch<&attn_packed_fwd<T, D, 2>, FwdShape<D, 2>::kLds>(dim3(x), a, stream);
  if (r.shares == 1) return launch<&attn_packed_fwd<T, D, 4>, FwdShape<D, 4>::kLds>(dim3(x), a, stream);
  const unsigned most = x * static_cast<unsigned>(r.shares), grid = static_cast<unsigned>(FwdShape<D, 4>::kPerCu * a.cus);
  HK_RETURN_IF_ERROR((launch<&attn_packed_fwd_shares<T, D>, FwdShape<D, 4>::kLds>(dim3(std::min(most, grid)), a, stream)));
  const int64_t rows = a.q_tokens * a.group * a.k_heads;
  return launch<&attn_packed_join<T, D>, 0>(dim3(static_cast<unsigned>(ceil_div(rows, 4))), a, stream);
}
template <class T>
hipError_t by_width(const Args& a, const Plan& r, hipStream_t stream) {
  return a.d <= 64 ? run<T, 64>(a, r, stream) : run<T, 128>(a, r, stream);
}

}  // namespace
}  // namespace packed
}  // namespace hk

using namespace hk::packed;

int64_t hk::packed::forward_workspace(const hk_attn_packed_params* p) {
  if (p->num_seqs == 0 || p->q_tokens == 0) return 0;
  const Plan r = plan(p);
  return r.part + r.stat + r.count;
}

extern "C" hipError_t hk_attn_packed_forward(const hk_attn_packed_params* p, int type, void* ws,
                                             int64_t workspace_bytes, hipStream_t stream) {
  HK_RETURN_IF_ERROR(check(p, type, false));
  if (p->num_seqs == 0 || p->q_tokens == 0) return hipSuccess;
  HK_CHECK_ARG(outputs_apart(p, false));
  const Plan r = plan(p);
  HK_RETURN_IF_ERROR(workspace(r.part + r.stat + r.count, ws, workspace_bytes, stream, &ws));
  Args a = make_args(p);
  a.tiles = r.tiles, a.chunk = r.chunk, a.most = r.shares;
  a.part = static_cast<float*>(ws);
  a.stat = reinterpret_cast<float2*>(static_cast<char*>(ws) + r.part);
  a.shares = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + r.part + r.stat);
  return type == HK_TYPE_BF16 ? by_width<TypeBF16>(a, r, stream) : by_width<TypeF16>(a, r, stream);
}

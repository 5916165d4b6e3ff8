// adamw8.hip - multi-tensor AdamW step over fp32 parameters whose two moments are held in 8 bits.
//
// The update is AdamW's (adamw.hip); only the form of its states differs. Both moments of a tensor are
// cut into blocks of 256 elements with one fp32 scale each, and an element holds one code:
//   m = scale_m c |c| / 127^2, c = -127 .. 127        v = scale_v (c / 255)^4, c = 0 .. 255
// The steps between two values grow with the value, so that elements far below their block's largest
// keep some digits: m resolves 6e-5 of it, sqrt(v), which the update divides by, 1.5e-5. After the
// update, scale_m is the largest |m| of the block and scale_v the largest v, rounded to fp32, and each
// code the one whose value is nearest, the larger of two that are equally near. A v > 0 keeps code 1
// at least: a v that fell to 0 beside an m that did not would divide by eps alone.
//
// The moments are formed and compared with the borders between codes in fp64, so that the codes are
// those of the definition whatever the order of the operations (in fp32 about one code of 10^5 would
// fall on the other side of a border; where no code adds to it a moment is exact there, and so is the
// rounding of the scales, whose ties 16-bit gradients do meet). With um = scale_m / 127^2 and
// uv = scale_v / 255^4, the values are um c |c| and uv c^4, and the borders are
//   um (c^2 - c + 1/2)    and    uv ((c - 1)^4 + c^4) / 2 = uv (h^4 + 3/2 h^2 + 1/16), h = c - 1/2.
// The parameter itself is updated in fp32 from the moments
// before they are rounded to codes, with the hardware's square root and reciprocal (1 ulp each, of a
// step that is lr times smaller than the parameter's own scale); in fp64 where v is no normal fp32 number and
// eps does not hide it.
//
// Bound: HBM, 16 bytes a parameter with fp32 gradients (28 with states in 32 bits: 573 us for the same
// step). One wave takes a block: 4 consecutive elements a lane, 16-byte accesses of p and g at any
// alignment, 4-byte ones of the codes, the scale by a register butterfly over the wave. Elements behind the
// end of a tensor have codes of 0. A non-finite gradient or moment gives the block NaN scales, and so NaN
// moments from then on: 8 bits cannot hold it in its element alone.
#include <math.h>

#include <algorithm>
#include <iterator>
#include <utility>
#include <vector>

#include "hk_device.h"
#include "hk_host.h"
#include "hk_overlap.h"

namespace {

constexpr int kBlock = HK_ADAM8_BLOCK;
static_assert(kBlock == 4 * HK_WAVE, "a wave holds a block, 4 elements a lane");

constexpr double kUnitM = 127.0 * 127.0, kUnitV = 255.0 * 255.0 * 255.0 * 255.0;

// ---- access at any element alignment (gfx950 serves unaligned vectors) -----------------------------
typedef float f32x4a4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2a2_t __attribute__((ext_vector_type(2), aligned(2)));
// Pointers out of a table are generic to the compiler, whose flat accesses wait with the LDS's; these are
// in device memory.
#define HK_GLOBAL __attribute__((address_space(1)))

// Four elements of a tensor from i on, zeros behind its end n; FULL: all of the block's lie before it.
struct GradF32 {
  using T = float;
  template <bool FULL>
  __device__ static void load4(const float* g, int64_t i, int64_t n, float (&f)[4]) {
    if (FULL || i + 4 <= n) {
      const f32x4a4_t v = __builtin_nontemporal_load((const f32x4a4_t HK_GLOBAL*)(g + i));
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = i + e < n ? g[i + e] : 0.f;
    }
  }
};
template <float (*ToF32)(uint16_t)>
struct Grad16 {
  using T = uint16_t;
  template <bool FULL>
  __device__ static void load4(const uint16_t* g, int64_t i, int64_t n, float (&f)[4]) {
    if (FULL || i + 4 <= n) {
      const u32x2a2_t v = __builtin_nontemporal_load((const u32x2a2_t HK_GLOBAL*)(g + i));
      f[0] = ToF32(static_cast<uint16_t>(v[0])), f[1] = ToF32(static_cast<uint16_t>(v[0] >> 16));
      f[2] = ToF32(static_cast<uint16_t>(v[1])), f[3] = ToF32(static_cast<uint16_t>(v[1] >> 16));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = i + e < n ? ToF32(g[i + e]) : 0.f;
    }
  }
};
template <bool FULL>
__device__ __forceinline__ void store4(float* p, int64_t i, int64_t n, const float (&f)[4]) {
  if (FULL || i + 4 <= n) {
    __builtin_nontemporal_store(f32x4a4_t{f[0], f[1], f[2], f[3]}, (f32x4a4_t HK_GLOBAL*)(p + i));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) p[i + e] = f[e];
  }
}
template <bool FULL>
__device__ __forceinline__ void store4(uint16_t* p, int64_t i, int64_t n, const float (&f)[4]) {
  const uint32_t lo = hk::pack_bf16x2(f[0], f[1]), hi = hk::pack_bf16x2(f[2], f[3]);
  if (FULL || i + 4 <= n) {
    __builtin_nontemporal_store(u32x2a2_t{lo, hi}, (u32x2a2_t HK_GLOBAL*)(p + i));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) p[i + e] = static_cast<uint16_t>((e < 2 ? lo : hi) >> (16 * (e & 1)));
  }
}

// ---- codes -----------------------------------------------------------------------------------------
// The values of a word's four codes in units of um and uv: c |c|, and c^2, whose square it is.
__device__ __forceinline__ void units_m(uint32_t w, float (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float c = static_cast<float>(static_cast<int>(w << (24 - 8 * e)) >> 24);
    f[e] = c * __builtin_fabsf(c);
  }
}
__device__ __forceinline__ void root_units_v(uint32_t w, float (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float c = static_cast<float>((w >> (8 * e)) & 255u);
    f[e] = c * c;
  }
}

// Codes are found in fp32 from x = |m| / um (v / uv): c^2 - c + 1/2 <= x exactly when
//   c <= t = 1/2 + sqrt(x - 1/4), and h^4 + 3/2 h^2 + 1/16 <= x when c <= t = 1/2 + sqrt(sqrt(x + 1/2) - 3/4),
// so that the code is the whole part of t. x is off by a few parts in 10^7, t, at most 255, by less than
// 10^-4: nearer than that to a whole number, the border itself decides, in fp64. About one block in
// eleven has such an element; deciding all of them that way took VALU time that the loads did not
// hide (124.4 M parameters, fp32 and bf16 gradients: 375 and 366 us; so, and with 60 instructions fewer a
// block elsewhere, 298 and 277, 6.7 and 6.3 TB/s).
constexpr float kNear = 1e-4f;
__device__ __forceinline__ float bound_m(float x) {
  return 0.5f + __builtin_amdgcn_sqrtf(fmaxf(x - 0.25f, 0.0f));
}
__device__ __forceinline__ float bound_v(float x) {
  return 0.5f + __builtin_amdgcn_sqrtf(fmaxf(__builtin_amdgcn_sqrtf(x + 0.5f) - 0.75f, 0.0f));
}
// The same decided by the border below k, the whole number nearest to t (at least 1).
__device__ __forceinline__ float exact_m(float t, double a, double um) {
  const float k = __builtin_amdgcn_fmed3f(__builtin_rintf(t), 1.0f, 127.0f);
  const double border = __builtin_fmaf(k, k, 0.5f - k);  // exact: under 2^15, in halves
  return a < border * um ? k - 1.0f : k;
}
__device__ __forceinline__ float exact_v(float t, double v, double uv) {
  const float k = __builtin_amdgcn_fmed3f(__builtin_rintf(t), 1.0f, 255.0f), h = k - 0.5f;
  const double u = h * h;  // exact: 18 bits
  return v < __builtin_fma(u, u + 1.5, 0.0625) * uv ? k - 1.0f : k;
}

// The largest magnitude of a block's fp32 values, by their bits: a NaN is larger than an infinity, and that
// than every number. NaN where the largest is not finite.
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max_u32(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
                        0, static_cast<int>(v), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ float block_max(const float (&f)[4]) {
  uint32_t v = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) v = max_u32(v, __float_as_uint(f[e]) & 0x7fffffffu);
  using namespace hk::detail;
  v = max_dpp<kDppMirror>(max_dpp<kDppHalfMirror>(max_dpp<kDppXor2>(max_dpp<kDppXor1>(v))));
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max_u32(r[0], r[1]);
  const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = __builtin_amdgcn_readfirstlane(max_u32(h[0], h[1]));
  return v < 0x7f800000u ? __uint_as_float(v) : NAN;
}

// Encodes a lane's part of a block and gives its scales. mf and vf: the moments rounded to fp32.
__device__ __forceinline__ void encode_block(const double (&m)[4], const double (&v)[4],
                                             const float (&mf)[4], const float (&vf)[4],
                                             uint32_t& mw, uint32_t& vw, float& sm, float& sv) {
  // rounding to fp32 keeps the order: the largest of the rounded is the largest, rounded
  sm = block_max(mf);
  sv = block_max(vf);
  if (!(sm < INFINITY && sv < INFINITY)) sm = sv = NAN;
  // estimates; a scale of 0 has no element over 0
  const float im = sm > 0.f ? __builtin_amdgcn_rcpf(sm) * static_cast<float>(kUnitM) : 0.f;
  const float iv = sv > 0.f ? __builtin_amdgcn_rcpf(sv) * static_cast<float>(kUnitV) : 0.f;
  float cm[4], cv[4], far = 1.f;  // far: the least distance of a bound from a whole number
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float tm = bound_m(fabsf(mf[e]) * im), tv = bound_v(vf[e] * iv);
    far = fminf(far, fminf(fabsf(tm - __builtin_rintf(tm)), fabsf(tv - __builtin_rintf(tv))));
    cm[e] = __builtin_floorf(tm);
    cv[e] = __builtin_floorf(tv);
  }
  // Scales whose elements or whose reciprocals fp32 does not hold go the long way, too: from 2^126 = 8.5e37 on
  // the reciprocal is subnormal, and the instruction gives 0.
  if (__ballot(far < kNear) != 0 || sm < 1e-25f || sv < 1e-25f || sm > 1e37f || sv > 1e37f) {
    const double um = sm > 0.f ? sm * (1.0 / kUnitM) : 1.0, uv = sv > 0.f ? sv * (1.0 / kUnitV) : 1.0;
    const double jm = __builtin_amdgcn_rcp(um), jv = __builtin_amdgcn_rcp(uv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cm[e] = exact_m(bound_m(static_cast<float>(fabs(m[e]) * jm)), fabs(m[e]), um);
      cv[e] = exact_v(bound_v(static_cast<float>(v[e] * jv)), v[e], uv);
    }
  }
  uint32_t c[4];
  vw = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    c[e] = static_cast<uint32_t>(static_cast<int>(copysignf(cm[e], mf[e])));
    vw = __builtin_amdgcn_cvt_pk_u8_f32(v[e] > 0.0 ? fmaxf(cv[e], 1.0f) : 0.0f, e, vw);
  }
  // the low bytes of the four
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u);
  mw = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu) | lo;
}

// ---- the step --------------------------------------------------------------------------------------
struct TensorEntry {
  float* p;
  const void* g;
  uint16_t* copy;  // NULL: none
  int64_t numel;
  int64_t block0;  // the tensor's first block in the states
};
struct States {
  uint32_t* m;
  uint32_t* v;
  float* m_scale;
  float* v_scale;
};
struct Hyper {
  double beta1, beta2, rest1, rest2;  // rest: 1 - beta
  float root_ibc2, eps;               // sqrt(1 / bias correction 2)
  float lr1, decay;                   // lr / bias correction 1, lr * weight decay
  int small_eps;                      // eps < kSmallEps
};
// The hardware's square root takes a subnormal v for 0, and a v under those is 0 in fp32. Both roots are under
// 1.1e-19 (divided by bias correction 2's root, under 1e-17): nothing beside an eps from here on, but all of the
// denominator where eps is 0.
constexpr float kSmallEps = 1e-9f, kLeastNormal = 1.1754944e-38f;

// One block of tensor t: its elements from `start` on, block `blk` of the states.
template <class G, bool FULL>
__device__ __forceinline__ void step_block(const TensorEntry& t, const States& st, const Hyper& h,
                                           int64_t start, int64_t blk, int lane) {
  const int64_t i = start + 4 * lane, w = blk * HK_WAVE + lane;
  float p[4], gf[4];
  GradF32::load4<FULL>(t.p, i, t.numel, p);
  G::template load4<FULL>(static_cast<const typename G::T*>(t.g), i, t.numel, gf);
  uint32_t mc = st.m[w], vc = st.v[w];
  __builtin_amdgcn_sched_barrier(0);  // every load is issued before any of them is waited for
  if (!FULL) {  // whatever lies behind the end counts as 0
    const int64_t left = t.numel - i;
    const uint32_t keep = left >= 4 ? ~0u : left > 0 ? ~0u >> (32 - 8 * static_cast<int>(left)) : 0u;
    mc &= keep;
    vc &= keep;
  }
  const float sm = st.m_scale[blk], sv = st.v_scale[blk];
  const double bm = h.beta1 * (sm * (1.0 / kUnitM)), bv = h.beta2 * (sv * (1.0 / kUnitV));
  double m[4], v[4];
  float mf[4], vf[4], cm[4], cv[4];
  units_m(mc, cm);
  root_units_v(vc, cv);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double ge = gf[e], c2 = cv[e];
    m[e] = __builtin_fma(bm, static_cast<double>(cm[e]), h.rest1 * ge);
    v[e] = __builtin_fma(bv, c2 * c2, h.rest2 * (ge * ge));
    mf[e] = static_cast<float>(m[e]);
    vf[e] = static_cast<float>(v[e]);
    // p - lr wd p - lr (m / bc1) / (sqrt(v / bc2) + eps)
    const float denom = __builtin_fmaf(__builtin_amdgcn_sqrtf(vf[e]), h.root_ibc2, h.eps);
    const float rest = __builtin_fmaf(-h.decay, p[e], p[e]);
    p[e] = __builtin_fmaf(-h.lr1 * mf[e], __builtin_amdgcn_rcpf(denom), rest);
    if (h.small_eps && vf[e] < kLeastNormal && v[e] > 0.0)
      p[e] = static_cast<float>(rest - h.lr1 * m[e] / (sqrt(v[e]) * h.root_ibc2 + h.eps));
  }
  uint32_t mw, vw;
  float sm1, sv1;
  encode_block(m, v, mf, vf, mw, vw, sm1, sv1);
  store4<FULL>(t.p, i, t.numel, p);
  if (t.copy) store4<FULL>(t.copy, i, t.numel, p);
  st.m[w] = mw;
  st.v[w] = vw;
  if (lane == 0) {
    st.m_scale[blk] = sm1;
    st.v_scale[blk] = sv1;
  }
}

// tensor_of: the tensor of each block, from block `first` on. One block a workgroup of one wave: 124.4 M parameters,
// fp32 gradients, 300 us, 315 with two blocks, 329 with four.
template <class G>
__global__ __launch_bounds__(HK_WAVE) void adam8_step(const TensorEntry* __restrict__ tensors,
                                                      const int32_t* __restrict__ tensor_of,
                                                      States st, Hyper h, uint32_t first) {
  const int64_t blk = first + blockIdx.x;
  const TensorEntry t = tensors[tensor_of[blk]];
  const int64_t start = (blk - t.block0) * kBlock;
  if (start + kBlock <= t.numel) step_block<G, true>(t, st, h, start, blk, threadIdx.x);
  else step_block<G, false>(t, st, h, start, blk, threadIdx.x);
}

// ---- conversion ------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void adam8_quantize(const float* __restrict__ m,
                                                      const float* __restrict__ v, int64_t numel,
                                                      States st) {
  const int lane = threadIdx.x & 63;
  const int64_t blk = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (blk * kBlock >= numel) return;
  const int64_t i = blk * kBlock + 4 * lane;
  float mf[4], vf[4];
  GradF32::load4<false>(m, i, numel, mf);
  GradF32::load4<false>(v, i, numel, vf);
  double m64[4], v64[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    vf[e] = vf[e] < 0.f ? 0.f : vf[e];  // NaN stays
    m64[e] = mf[e];
    v64[e] = vf[e];
  }
  uint32_t mw, vw;
  float sm, sv;
  encode_block(m64, v64, mf, vf, mw, vw, sm, sv);
  st.m[blk * HK_WAVE + lane] = mw;
  st.v[blk * HK_WAVE + lane] = vw;
  if (lane == 0) {
    st.m_scale[blk] = sm;
    st.v_scale[blk] = sv;
  }
}

__global__ __launch_bounds__(256) void adam8_dequantize(const uint32_t* __restrict__ mc,
                                                        const uint32_t* __restrict__ vc,
                                                        const float* __restrict__ m_scale,
                                                        const float* __restrict__ v_scale,
                                                        int64_t numel, float* __restrict__ m,
                                                        float* __restrict__ v) {
  const int lane = threadIdx.x & 63;
  const int64_t blk = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (blk * kBlock >= numel) return;
  const int64_t i = blk * kBlock + 4 * lane;
  const uint32_t mw = mc[blk * HK_WAVE + lane], vw = vc[blk * HK_WAVE + lane];
  const double um = m_scale[blk] * (1.0 / kUnitM), uv = v_scale[blk] * (1.0 / kUnitV);
  float mf[4], vf[4], cm[4], cv[4];
  units_m(mw, cm);
  root_units_v(vw, cv);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double c2 = cv[e];
    mf[e] = static_cast<float>(cm[e] * um);
    vf[e] = static_cast<float>(c2 * c2 * uv);
  }
  store4<false>(m, i, numel, mf);
  store4<false>(v, i, numel, vf);
}

// Blocks of one launch: a dimension of a grid has under 2^32 threads, and more of them run as their number
// modulo 2^32, with no error.
constexpr int64_t kLaunchBlocks = int64_t{1} << 25;

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

struct hk_adam8_plan {
  TensorEntry* d_tensors = nullptr;
  int32_t* d_tensor_of = nullptr;
  int64_t num_blocks = 0;
  int grad_type = HK_TYPE_F32, device = 0;
  States st{};
};

extern "C" hipError_t hk_adam8_plan_create(int num_tensors, float* const* params,
                                           const void* const* grads, int grad_type,
                                           hk_bf16* const* copies, const int64_t* sizes,
                                           int8_t* m_codes, uint8_t* v_codes, float* m_scales,
                                           float* v_scales, hk_adam8_plan** plan_out) try {
  HK_CHECK_ARG(plan_out != nullptr);
  *plan_out = nullptr;
  HK_CHECK_ARG(num_tensors >= 0);
  HK_CHECK_ARG(grad_type >= HK_TYPE_F32 && grad_type <= HK_TYPE_F16);
  HK_CHECK_ARG(num_tensors == 0 || (params && grads && sizes));
  std::vector<TensorEntry> tensors(num_tensors);
  std::vector<int32_t> tensor_of;
  int64_t blocks = 0;
  const unsigned grad_align = grad_type == HK_TYPE_F32 ? 3u : 1u;
  for (int t = 0; t < num_tensors; ++t) {
    HK_CHECK_ARG(sizes[t] >= 0 && sizes[t] <= int64_t{INT32_MAX} * kBlock);
    uint16_t* copy = copies ? copies[t] : nullptr;
    HK_CHECK_ARG(sizes[t] == 0 || (params[t] && grads[t]));
    HK_CHECK_ARG(aligned4(params[t]) && (reinterpret_cast<uintptr_t>(grads[t]) & grad_align) == 0 &&
                 (reinterpret_cast<uintptr_t>(copy) & 1u) == 0);
    const int64_t nb = hk::ceil_div(sizes[t], kBlock);
    HK_CHECK_ARG(nb <= INT32_MAX - blocks);
    tensors[t] = TensorEntry{params[t], grads[t], copy, sizes[t], blocks};
    blocks += nb;
  }
  HK_CHECK_ARG(blocks == 0 || (m_codes && v_codes && m_scales && v_scales));
  HK_CHECK_ARG(aligned4(m_codes) && aligned4(v_codes) && aligned4(m_scales) && aligned4(v_scales));
  // what a step writes, each memory once: blocks of one step run in any order
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
  auto writes = [&](const void* q, int64_t bytes) {
    const auto a = reinterpret_cast<uintptr_t>(q);
    if (q && bytes > 0) written.emplace_back(a, a + bytes);
  };
  for (int t = 0; t < num_tensors; ++t) {
    writes(params[t], 4 * sizes[t]);
    if (copies) writes(copies[t], 2 * sizes[t]);
  }
  writes(m_codes, kBlock * blocks);
  writes(v_codes, kBlock * blocks);
  writes(m_scales, 4 * blocks);
  writes(v_scales, 4 * blocks);
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i) HK_CHECK_ARG(written[i - 1].second <= written[i].first);
  // nor a gradient on any of it, but on its own parameter element by element
  const int64_t grad_bytes = grad_type == HK_TYPE_F32 ? 4 : 2;
  for (int t = 0; t < num_tensors; ++t) {
    if (sizes[t] == 0 || (grad_bytes == 4 && grads[t] == params[t])) continue;
    const auto a = reinterpret_cast<uintptr_t>(grads[t]), end = a + grad_bytes * sizes[t];
    const auto next = std::lower_bound(written.begin(), written.end(), std::make_pair(end, uintptr_t{0}));
    HK_CHECK_ARG(next == written.begin() || std::prev(next)->second <= a);
  }
  tensor_of.reserve(blocks);
  for (int t = 0; t < num_tensors; ++t)
    tensor_of.insert(tensor_of.end(), hk::ceil_div(sizes[t], kBlock), t);
  hk_adam8_plan* plan = new hk_adam8_plan();
  plan->num_blocks = blocks;
  plan->grad_type = grad_type;
  plan->st = States{reinterpret_cast<uint32_t*>(m_codes), reinterpret_cast<uint32_t*>(v_codes),
                    m_scales, v_scales};
  hipError_t e = hipGetDevice(&plan->device);
  if (e == hipSuccess && blocks > 0) {
    e = hipMalloc(&plan->d_tensors, tensors.size() * sizeof(TensorEntry));
    if (e == hipSuccess)
      e = hipMemcpy(plan->d_tensors, tensors.data(), tensors.size() * sizeof(TensorEntry),
                    hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMalloc(&plan->d_tensor_of, tensor_of.size() * sizeof(int32_t));
    if (e == hipSuccess)
      e = hipMemcpy(plan->d_tensor_of, tensor_of.data(), tensor_of.size() * sizeof(int32_t),
                    hipMemcpyHostToDevice);
  }
  if (e != hipSuccess) {
    (void)hk_adam8_plan_destroy(plan);
    return e;
  }
  *plan_out = plan;
  return hipSuccess;
} catch (...) {
  return hipErrorOutOfMemory;  // the tables' host memory
}

extern "C" hipError_t hk_adam8_plan_step(const hk_adam8_plan* plan, float lr, float beta1,
                                         float beta2, float eps, float weight_decay,
                                         float bias_correction1, float bias_correction2,
                                         hipStream_t stream) {
  HK_CHECK_ARG(plan != nullptr);
  if (plan->num_blocks == 0) return hipSuccess;
  int device = 0;
  HK_RETURN_IF_ERROR(hipGetDevice(&device));
  HK_CHECK_ARG(device == plan->device);
  const Hyper h{beta1, beta2, 1.0 - beta1, 1.0 - beta2,
                static_cast<float>(1.0 / sqrt(static_cast<double>(bias_correction2))), eps,
                static_cast<float>(static_cast<double>(lr) / bias_correction1),
                static_cast<float>(static_cast<double>(lr) * weight_decay), eps < kSmallEps};
  auto* k = plan->grad_type == HK_TYPE_F32    ? adam8_step<GradF32>
            : plan->grad_type == HK_TYPE_BF16 ? adam8_step<Grad16<hk::bf16_to_f32>>
                                              : adam8_step<Grad16<hk::f16_to_f32>>;
  for (int64_t first = 0; first < plan->num_blocks; first += kLaunchBlocks) {
    const int64_t n = std::min(kLaunchBlocks, plan->num_blocks - first);
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(n)), dim3(HK_WAVE), 0, stream, plan->d_tensors,
                       plan->d_tensor_of, plan->st, h, static_cast<uint32_t>(first));
    HK_RETURN_IF_ERROR(hk::launch_status());
  }
  return hipSuccess;
}

extern "C" hipError_t hk_adam8_plan_destroy(hk_adam8_plan* plan) {
  if (!plan) return hipSuccess;
  hipError_t e = hipSuccess;
  if (plan->d_tensors) e = hipFree(plan->d_tensors);
  if (plan->d_tensor_of) {
    const hipError_t e2 = hipFree(plan->d_tensor_of);
    if (e == hipSuccess) e = e2;
  }
  delete plan;
  return e;
}

extern "C" int64_t hk_adam8_plan_num_blocks(const hk_adam8_plan* plan) {
  return plan ? plan->num_blocks : 0;
}

namespace {
// What a conversion works on; the checks that both have in common.
bool conversion_holds(const void* m_codes, const void* v_codes, const float* m_scales,
                      const float* v_scales, int64_t numel, const float* m, const float* v) {
  if (numel < 0 || numel > int64_t{INT32_MAX} * kBlock) return false;
  if (numel == 0) return true;
  for (const void* p : {m_codes, v_codes, static_cast<const void*>(m_scales),
                        static_cast<const void*>(v_scales), static_cast<const void*>(m),
                        static_cast<const void*>(v)})
    if (!p || !aligned4(p)) return false;
  // blocks are converted in any order: all six apart
  const int64_t blocks = hk::ceil_div(numel, kBlock);
  const hk::Rows part[6] = {hk::Rows(m_codes, kBlock, blocks), hk::Rows(v_codes, kBlock, blocks),
                            hk::Rows(m_scales, 4, blocks),     hk::Rows(v_scales, 4, blocks),
                            hk::Rows(m, 4, numel),             hk::Rows(v, 4, numel)};
  for (int i = 1; i < 6; ++i)
    for (int j = 0; j < i; ++j)
      if (hk::overlap(part[i], part[j])) return false;
  return true;
}
// Calls launch(first block, elements from there on, workgroups of four blocks) for each launch's blocks.
template <class Launch>
hipError_t by_launch(int64_t numel, Launch&& launch) {
  constexpr int64_t kElements = kLaunchBlocks * kBlock;
  for (int64_t at = 0; at < numel; at += kElements) {
    const int64_t n = std::min(kElements, numel - at);
    launch(at / kBlock, n, dim3(static_cast<unsigned>(hk::ceil_div(n, 4 * kBlock))));
    HK_RETURN_IF_ERROR(hk::launch_status());
  }
  return hipSuccess;
}
}  // namespace

extern "C" hipError_t hk_adam8_quantize(const float* m, const float* v, int64_t numel,
                                        int8_t* m_codes, uint8_t* v_codes, float* m_scales,
                                        float* v_scales, hipStream_t stream) {
  HK_CHECK_ARG(conversion_holds(m_codes, v_codes, m_scales, v_scales, numel, m, v));
  return by_launch(numel, [&](int64_t block, int64_t n, dim3 grid) {
    const int64_t i = block * kBlock;
    const States st{reinterpret_cast<uint32_t*>(m_codes + i), reinterpret_cast<uint32_t*>(v_codes + i),
                    m_scales + block, v_scales + block};
    hipLaunchKernelGGL(adam8_quantize, grid, dim3(256), 0, stream, m + i, v + i, n, st);
  });
}

extern "C" hipError_t hk_adam8_dequantize(const int8_t* m_codes, const uint8_t* v_codes,
                                          const float* m_scales, const float* v_scales,
                                          int64_t numel, float* m, float* v, hipStream_t stream) {
  HK_CHECK_ARG(conversion_holds(m_codes, v_codes, m_scales, v_scales, numel, m, v));
  return by_launch(numel, [&](int64_t block, int64_t n, dim3 grid) {
    const int64_t i = block * kBlock;
    hipLaunchKernelGGL(adam8_dequantize, grid, dim3(256), 0, stream,
                       reinterpret_cast<const uint32_t*>(m_codes + i),
                       reinterpret_cast<const uint32_t*>(v_codes + i), m_scales + block,
                       v_scales + block, n, m + i, v + i);
  });
}

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
// step that is lr times smaller than the parameter's own scale).
//
// One wave takes a block: 4 consecutive elements a lane, 16-byte accesses of p and g at any alignment,
// 4-byte ones of the codes, the scale by a register butterfly over the wave. Elements behind the end
// of a tensor have codes of 0. A non-finite gradient or moment gives the block NaN scales, and so NaN
// moments from then on: 8 bits cannot hold it in its element alone.
#include <vector>

#include "hk_device.h"
#include "hk_host.h"

namespace {

constexpr int kBlock = HK_ADAM8_BLOCK;
static_assert(kBlock == 4 * HK_WAVE, "a wave holds a block, 4 elements a lane");
constexpr int kBlocksPerWave = 2;

constexpr double kUnitM = 127.0 * 127.0, kUnitV = 255.0 * 255.0 * 255.0 * 255.0;

// ---- access at any element alignment (gfx950 serves unaligned vectors) -----------------------------
typedef float f32x4a4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2a2_t __attribute__((ext_vector_type(2), aligned(2)));

// Four elements of a tensor from i on, zeros behind its end n.
struct GradF32 {
  using T = float;
  __device__ static void load4(const float* g, int64_t i, int64_t n, float (&f)[4]) {
    if (i + 4 <= n) {
      const f32x4a4_t v = __builtin_nontemporal_load(reinterpret_cast<const f32x4a4_t*>(g + i));
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
  __device__ static void load4(const uint16_t* g, int64_t i, int64_t n, float (&f)[4]) {
    if (i + 4 <= n) {
      const u32x2a2_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x2a2_t*>(g + i));
      f[0] = ToF32(static_cast<uint16_t>(v[0])), f[1] = ToF32(static_cast<uint16_t>(v[0] >> 16));
      f[2] = ToF32(static_cast<uint16_t>(v[1])), f[3] = ToF32(static_cast<uint16_t>(v[1] >> 16));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = i + e < n ? ToF32(g[i + e]) : 0.f;
    }
  }
};
__device__ __forceinline__ void store4(float* p, int64_t i, int64_t n, const float (&f)[4]) {
  if (i + 4 <= n) {
    __builtin_nontemporal_store(f32x4a4_t{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4a4_t*>(p + i));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) p[i + e] = f[e];
  }
}
__device__ __forceinline__ void store4(uint16_t* p, int64_t i, int64_t n, const float (&f)[4]) {
  const uint32_t lo = hk::pack_bf16x2(f[0], f[1]), hi = hk::pack_bf16x2(f[2], f[3]);
  if (i + 4 <= n) {
    __builtin_nontemporal_store(u32x2a2_t{lo, hi}, reinterpret_cast<u32x2a2_t*>(p + i));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) p[i + e] = static_cast<uint16_t>((e < 2 ? lo : hi) >> (16 * (e & 1)));
  }
}

// ---- codes -----------------------------------------------------------------------------------------
__device__ __forceinline__ int code_m(uint32_t w, int e) { return static_cast<int>(w << (24 - 8 * e)) >> 24; }
__device__ __forceinline__ uint32_t code_v(uint32_t w, int e) { return (w >> (8 * e)) & 255u; }
// The code's value in units of um and uv.
__device__ __forceinline__ double units_m(int c) { return static_cast<double>(c * abs(c)); }
__device__ __forceinline__ double units_v(uint32_t c) {
  const uint32_t c2 = c * c;
  return static_cast<double>(c2 * c2);  // 255^4 < 2^32
}

// The code of a = |m| >= 0. With x = a / um, c^2 - c + 1/2 <= x exactly when c <= 1/2 + sqrt(x - 1/4):
// the whole number nearest to that bound, found in fp32, is the code or one more, which the border
// in fp64 decides. inv: about 1 / um, or 0 where um is 0.
__device__ __forceinline__ int encode_m(double a, double um, double inv) {
  const float x = static_cast<float>(a * inv);
  const float t = 0.5f + __builtin_amdgcn_sqrtf(fmaxf(x - 0.25f, 0.0f));
  const int k = static_cast<int>(__builtin_rintf(fminf(fmaxf(t, 1.0f), 127.0f)));
  const double border = static_cast<double>(k * (k - 1)) + 0.5;
  return k - (a < border * um || !(a > 0.0) ? 1 : 0);
}
// The code of v >= 0, the same way: h^4 + 3/2 h^2 + 1/16 <= x exactly when h^2 <= sqrt(x + 1/2) - 3/4.
__device__ __forceinline__ uint32_t encode_v(double v, double uv, double inv) {
  const float x = static_cast<float>(v * inv);
  const float t =
      0.5f + __builtin_amdgcn_sqrtf(fmaxf(__builtin_amdgcn_sqrtf(x + 0.5f) - 0.75f, 0.0f));
  const float k = __builtin_rintf(fminf(fmaxf(t, 1.0f), 255.0f));
  const double h = static_cast<double>(k) - 0.5, u = h * h;
  const double border = __builtin_fma(u, u + 1.5, 0.0625);
  const int c = static_cast<int>(k) - (v < border * uv ? 1 : 0);
  return v > 0.0 ? max(c, 1) : 0;
}

// Encodes a lane's part of a block and gives its scales. bad: a lane's moments are not finite.
__device__ __forceinline__ void encode_block(const double (&m)[4], const double (&v)[4], bool bad,
                                             uint32_t& mw, uint32_t& vw, float& sm, float& sv) {
  const double am = fmax(fmax(fabs(m[0]), fabs(m[1])), fmax(fabs(m[2]), fabs(m[3])));
  const double av = fmax(fmax(v[0], v[1]), fmax(v[2], v[3]));
  // rounding to fp32 keeps the order, so the largest can be rounded before the lanes are compared
  sm = hk::wave_max(static_cast<float>(am));
  sv = hk::wave_max(static_cast<float>(av));
  if (__ballot(bad) != 0 || !(sm < INFINITY) || !(sv < INFINITY)) sm = sv = NAN;
  const double um = sm * (1.0 / kUnitM), uv = sv * (1.0 / kUnitV);
  // estimates (v_rcp_f64); in fp64, where no scale that fp32 holds overflows
  const double im = sm > 0.f ? __builtin_amdgcn_rcp(um) : 0.0;
  const double iv = sv > 0.f ? __builtin_amdgcn_rcp(uv) : 0.0;
  mw = vw = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = encode_m(fabs(m[e]), um, im);
    mw |= static_cast<uint32_t>((m[e] < 0.0 ? -c : c) & 255) << (8 * e);
    vw |= encode_v(v[e], uv, iv) << (8 * e);
  }
}

// ---- the step --------------------------------------------------------------------------------------
struct TensorEntry {
  float* p;
  const void* g;
  uint16_t* copy;  // NULL: none
  int64_t numel;
  int64_t block0;  // the tensor's first block in the states
};
struct ChunkEntry {  // kBlocksPerWave blocks of a tensor
  int32_t tensor;
  int32_t chunk;
};
struct States {
  uint32_t* m;
  uint32_t* v;
  float* m_scale;
  float* v_scale;
};
struct Hyper {
  double beta1, beta2, rest1, rest2;  // rest: 1 - beta
  float ibc1, ibc2;                   // 1 / bias correction
  float lr, eps, wd;
};

template <class G>
__global__ __launch_bounds__(HK_WAVE) void adam8_step(const TensorEntry* __restrict__ tensors,
                                                      const ChunkEntry* __restrict__ chunks,
                                                      States st, Hyper h) {
  const ChunkEntry ce = chunks[blockIdx.x];
  const TensorEntry t = tensors[ce.tensor];
  const typename G::T* g = static_cast<const typename G::T*>(t.g);
  const int lane = threadIdx.x;
  const int64_t first = static_cast<int64_t>(ce.chunk) * kBlocksPerWave;
#pragma unroll
  for (int b = 0; b < kBlocksPerWave; ++b) {
    const int64_t i = (first + b) * kBlock + 4 * lane;
    if ((first + b) * kBlock >= t.numel) break;
    const int64_t blk = t.block0 + first + b, w = blk * HK_WAVE + lane;
    float p[4], gf[4];
    GradF32::load4(t.p, i, t.numel, p);
    G::load4(g, i, t.numel, gf);
    const uint32_t mc = st.m[w], vc = st.v[w];
    const float sm = st.m_scale[blk], sv = st.v_scale[blk];
    const double bm = h.beta1 * (sm * (1.0 / kUnitM)), bv = h.beta2 * (sv * (1.0 / kUnitV));
    double m[4], v[4];
    float zero = 0.f;  // NaN where a gradient is not finite
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = i + e < t.numel;
      const double ge = gf[e];
      m[e] = in ? __builtin_fma(bm, units_m(code_m(mc, e)), h.rest1 * ge) : 0.0;
      v[e] = in ? __builtin_fma(bv, units_v(code_v(vc, e)), h.rest2 * (ge * ge)) : 0.0;
      zero = __builtin_fmaf(gf[e], 0.f, zero);
      const float denom = __builtin_amdgcn_sqrtf(static_cast<float>(v[e]) * h.ibc2) + h.eps;
      const float update = static_cast<float>(m[e]) * h.ibc1 * __builtin_amdgcn_rcpf(denom);
      p[e] = p[e] - h.lr * (update + h.wd * p[e]);
    }
    uint32_t mw, vw;
    float sm1, sv1;
    encode_block(m, v, zero != 0.f || !(sm < INFINITY) || !(sv < INFINITY), mw, vw, sm1, sv1);
    store4(t.p, i, t.numel, p);
    if (t.copy) store4(t.copy, i, t.numel, p);
    st.m[w] = mw;
    st.v[w] = vw;
    if (lane == 0) {
      st.m_scale[blk] = sm1;
      st.v_scale[blk] = sv1;
    }
  }
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
  GradF32::load4(m, i, numel, mf);
  GradF32::load4(v, i, numel, vf);
  double m64[4], v64[4];
  float zero = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m64[e] = mf[e];
    v64[e] = fmaxf(vf[e], 0.f);
    zero = __builtin_fmaf(mf[e], 0.f, __builtin_fmaf(vf[e], 0.f, zero));
  }
  uint32_t mw, vw;
  float sm, sv;
  encode_block(m64, v64, zero != 0.f, mw, vw, sm, sv);
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
  float mf[4], vf[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    mf[e] = static_cast<float>(units_m(code_m(mw, e)) * um);
    vf[e] = static_cast<float>(units_v(code_v(vw, e)) * uv);
  }
  store4(m, i, numel, mf);
  store4(v, i, numel, vf);
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

struct hk_adam8_plan {
  TensorEntry* d_tensors = nullptr;
  ChunkEntry* d_chunks = nullptr;
  int64_t num_chunks = 0, num_blocks = 0;
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
  std::vector<ChunkEntry> chunks;
  int64_t blocks = 0;
  const unsigned grad_align = grad_type == HK_TYPE_F32 ? 3u : 1u;
  for (int t = 0; t < num_tensors; ++t) {
    HK_CHECK_ARG(sizes[t] >= 0);
    uint16_t* copy = copies ? copies[t] : nullptr;
    HK_CHECK_ARG(sizes[t] == 0 || (params[t] && grads[t]));
    HK_CHECK_ARG(aligned4(params[t]) && (reinterpret_cast<uintptr_t>(grads[t]) & grad_align) == 0 &&
                 (reinterpret_cast<uintptr_t>(copy) & 1u) == 0);
    const int64_t nb = hk::ceil_div(sizes[t], kBlock), nch = hk::ceil_div(nb, kBlocksPerWave);
    HK_CHECK_ARG(nch <= INT32_MAX - static_cast<int64_t>(chunks.size()));
    tensors[t] = TensorEntry{params[t], grads[t], copy, sizes[t], blocks};
    for (int64_t c = 0; c < nch; ++c) chunks.push_back(ChunkEntry{t, static_cast<int32_t>(c)});
    blocks += nb;
  }
  HK_CHECK_ARG(blocks == 0 || (m_codes && v_codes && m_scales && v_scales));
  HK_CHECK_ARG(aligned4(m_codes) && aligned4(v_codes) && aligned4(m_scales) && aligned4(v_scales));
  hk_adam8_plan* plan = new hk_adam8_plan();
  plan->num_chunks = static_cast<int64_t>(chunks.size());
  plan->num_blocks = blocks;
  plan->grad_type = grad_type;
  plan->st = States{reinterpret_cast<uint32_t*>(m_codes), reinterpret_cast<uint32_t*>(v_codes),
                    m_scales, v_scales};
  hipError_t e = hipGetDevice(&plan->device);
  if (e == hipSuccess && !chunks.empty()) {
    e = hipMalloc(&plan->d_tensors, tensors.size() * sizeof(TensorEntry));
    if (e == hipSuccess)
      e = hipMemcpy(plan->d_tensors, tensors.data(), tensors.size() * sizeof(TensorEntry),
                    hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMalloc(&plan->d_chunks, chunks.size() * sizeof(ChunkEntry));
    if (e == hipSuccess)
      e = hipMemcpy(plan->d_chunks, chunks.data(), chunks.size() * sizeof(ChunkEntry),
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
  if (plan->num_chunks == 0) return hipSuccess;
  int device = 0;
  HK_RETURN_IF_ERROR(hipGetDevice(&device));
  HK_CHECK_ARG(device == plan->device);
  const Hyper h{beta1, beta2, 1.0 - beta1, 1.0 - beta2, 1.0f / bias_correction1,
                1.0f / bias_correction2, lr, eps, weight_decay};
  auto* k = plan->grad_type == HK_TYPE_F32    ? adam8_step<GradF32>
            : plan->grad_type == HK_TYPE_BF16 ? adam8_step<Grad16<hk::bf16_to_f32>>
                                              : adam8_step<Grad16<hk::f16_to_f32>>;
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(plan->num_chunks)), dim3(HK_WAVE), 0, stream,
                     plan->d_tensors, plan->d_chunks, plan->st, h);
  return hk::launch_status();
}

extern "C" hipError_t hk_adam8_plan_destroy(hk_adam8_plan* plan) {
  if (!plan) return hipSuccess;
  hipError_t e = hipSuccess;
  if (plan->d_tensors) e = hipFree(plan->d_tensors);
  if (plan->d_chunks) {
    const hipError_t e2 = hipFree(plan->d_chunks);
    if (e == hipSuccess) e = e2;
  }
  delete plan;
  return e;
}

extern "C" int64_t hk_adam8_plan_num_blocks(const hk_adam8_plan* plan) {
  return plan ? plan->num_blocks : 0;
}

namespace {
// Workgroups of four blocks, or -1 where the arguments do not hold.
int64_t conversion_grid(const void* m_codes, const void* v_codes, const float* m_scales,
                        const float* v_scales, int64_t numel, const float* m, const float* v) {
  if (numel < 0) return -1;
  if (numel == 0) return 0;
  if (!m_codes || !v_codes || !m_scales || !v_scales || !m || !v) return -1;
  for (const void* p : {m_codes, v_codes, static_cast<const void*>(m_scales),
                        static_cast<const void*>(v_scales), static_cast<const void*>(m),
                        static_cast<const void*>(v)})
    if (!aligned4(p)) return -1;
  const int64_t grid = hk::ceil_div(hk::ceil_div(numel, kBlock), 4);
  return grid <= INT32_MAX ? grid : -1;
}
}  // namespace

extern "C" hipError_t hk_adam8_quantize(const float* m, const float* v, int64_t numel,
                                        int8_t* m_codes, uint8_t* v_codes, float* m_scales,
                                        float* v_scales, hipStream_t stream) {
  const int64_t grid = conversion_grid(m_codes, v_codes, m_scales, v_scales, numel, m, v);
  HK_CHECK_ARG(grid >= 0);
  if (grid == 0) return hipSuccess;
  const States st{reinterpret_cast<uint32_t*>(m_codes), reinterpret_cast<uint32_t*>(v_codes),
                  m_scales, v_scales};
  hipLaunchKernelGGL(adam8_quantize, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, m, v,
                     numel, st);
  return hk::launch_status();
}

extern "C" hipError_t hk_adam8_dequantize(const int8_t* m_codes, const uint8_t* v_codes,
                                          const float* m_scales, const float* v_scales,
                                          int64_t numel, float* m, float* v, hipStream_t stream) {
  const int64_t grid = conversion_grid(m_codes, v_codes, m_scales, v_scales, numel, m, v);
  HK_CHECK_ARG(grid >= 0);
  if (grid == 0) return hipSuccess;
  hipLaunchKernelGGL(adam8_dequantize, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream,
                     reinterpret_cast<const uint32_t*>(m_codes),
                     reinterpret_cast<const uint32_t*>(v_codes), m_scales, v_scales, numel, m, v);
  return hk::launch_status();
}

// qk_norm_rope.hip - RMS norm of each query and key head with the position rotation, in one pass.
//
// Per token and head, x its head_dim elements:
//   n = x r, r = (mean(x^2) + eps)^(-1/2),  z = n w,  y = z with pair i of its first rotary_dim elements
//   (z_i, z_{i + rotary_dim / 2}), or (z_2i, z_2i+1) where interleaved, turned by the angle of the
//   token's position: (a cos - b sin, b cos + a sin).
// Backward, from dy: g = dy turned back by the same angles, and
//   dw = sum over tokens and heads of g n,   dx = r (g w - n mean(g w n)).
// All arithmetic is fp32, with one rounding where an output has 16 bits. r is not kept between the
// passes: the backward pass reads x anyway and forms it again.
//
// Bound: HBM, each row read once and written once (the table's rows and w are shared by the heads of a
// token and come from the caches). A row is held by 2^k lanes, each with a unit of V pairs: the two
// vectors of V elements that its rotation combines sit in one lane, so the only exchange between
// lanes is the sum of squares (and of g w n), a register butterfly over the row's lanes. Vectors are
// 16 bytes of 16-bit elements where both parts of a row, the rotated one and the rest, are whole units of
// them; else 4 elements, at any element alignment, and a part that is not whole units ends with one that
// overlaps the unit before it.
// Rows go to lane groups token by token, heads innermost, so that the groups of a wave read the same
// table rows. Elements behind rotary_dim are units of two neighbouring vectors with an angle of zero. Stores
// are non-temporal (8 x 1024 tokens of 12 + 12 heads of 64, bf16 -> fp32: forward 16.3 -> 14.7 us,
// backward with dw 23.9 -> 22.5), loads are not (18.8 and 25.7: heads share their cache lines).
//
// The gradients of the two weight vectors are summed in registers over the rows of a lane group, over
// a workgroup through LDS, and over the workgroups by a second kernel, all in a fixed order.
#include <algorithm>

#include "hk_device.h"
#include "hk_host.h"
#include "hk_overlap.h"

namespace {

constexpr int kThreads = 256;      // forward
constexpr int kBackThreads = 512, kBackWaves = kBackThreads / HK_WAVE;
constexpr int kBackPerCu = 3;      // workgroups of the backward pass that a CU holds
constexpr int kMaxDim = 256;

// Vectors of V elements at any alignment of the element type.
template <typename S, int V>
__device__ __forceinline__ void load_vec(const S* p, S (&f)[V]) {
  __builtin_memcpy(f, p, V * sizeof(S));
}
// ONCE: device memory that this call does not read again.
template <bool ONCE, typename S, int V>
__device__ __forceinline__ void store_vec(S* p, const S (&f)[V]) {
  if constexpr (ONCE && V > 1) {
    typedef S vec_t __attribute__((ext_vector_type(V), aligned(sizeof(S))));
    vec_t v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = f[e];
    __builtin_nontemporal_store(v, reinterpret_cast<vec_t*>(p));
  } else {
    __builtin_memcpy(p, f, V * sizeof(S));
  }
}
template <class F, int V>
__device__ __forceinline__ void load_f32(const typename F::storage* p, float (&f)[V]) {
  typename F::storage s[V];
  load_vec(p, s);
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = F::load(s, e);
}
template <class F, int V, bool ONCE>
__device__ __forceinline__ void store_f32(typename F::storage* p, const float (&f)[V]) {
  typename F::storage s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) F::store(s, e, f[e]);
  store_vec<ONCE>(p, s);
}

struct Shape {
  int d, rot, half;           // half: rot / 2
  int rotated, units, lanes;  // rotated: units that are; lanes: of a row, a power of two
  bool interleaved;
};

// Where the two vectors of unit u lie in a row, and whether the second exists (a head of odd size,
// V == 1). OVERLAP: the last unit of the rotated part and that of the rest are moved back to whole
// vectors; their first elements are the unit's before them too, and only its (old).
template <int V, bool OVERLAP>
struct Unit {
  int a, b, angle;   // angle: first pair of the table row, -1: not rotated
  int old_a, old_b;  // elements of the two vectors that are another unit's
  bool on, pairs;    // pairs: neighbouring elements are rotated together
  __device__ Unit(const Shape& s, int u) {
    on = u < s.units;
    pairs = u < s.rotated && s.interleaved;
    angle = -1;
    old_a = old_b = 0;
    if (u < s.rotated) {
      angle = u * V;
      if (OVERLAP && angle + V > s.half) {
        old_a = old_b = angle + V - s.half;
        angle = s.half - V;
      }
      a = s.interleaved ? 2 * angle : angle;
      b = s.interleaved ? a + V : s.half + angle;
    } else {
      a = s.rot + 2 * (u - s.rotated) * V;
      if (OVERLAP && a + 2 * V > s.d) {
        const int old = a + 2 * V - s.d;
        old_a = min(V, old);
        old_b = old - old_a;
        a = s.d - 2 * V;
      }
      b = a + V;
    }
  }
  // v where element e of the first (second) vector is the unit's own, else 0
  __device__ float own_a(int e, float v) const { return OVERLAP && e < old_a ? 0.f : v; }
  __device__ float own_b(int e, float v) const { return OVERLAP && e < old_b ? 0.f : v; }
};

// x as the pairs (a[j], b[j]) of a unit.
template <class F, int V, bool O>
__device__ __forceinline__ void load_unit(const typename F::storage* row, const Unit<V, O>& u, int d,
                                          float (&a)[V], float (&b)[V]) {
  load_f32<F, V>(row + u.a, a);
  if (V > 1 || u.b < d) {
    load_f32<F, V>(row + u.b, b);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) b[e] = 0.f;
  }
  if (V > 1 && u.pairs) {
    float t[2 * V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = a[e], t[V + e] = b[e];
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] = t[2 * e], b[e] = t[2 * e + 1];
  }
}
template <class F, int V, bool ONCE = true, bool O>
__device__ __forceinline__ void store_unit(typename F::storage* row, const Unit<V, O>& u, int d,
                                           const float (&a)[V], const float (&b)[V]) {
  if (V > 1 && u.pairs) {
    float t[2 * V], lo[V], hi[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[2 * e] = a[e], t[2 * e + 1] = b[e];
#pragma unroll
    for (int e = 0; e < V; ++e) lo[e] = t[e], hi[e] = t[V + e];
    store_f32<F, V, ONCE>(row + u.a, lo);
    store_f32<F, V, ONCE>(row + u.b, hi);
  } else {
    store_f32<F, V, ONCE>(row + u.a, a);
    if (V > 1 || u.b < d) store_f32<F, V, ONCE>(row + u.b, b);
  }
}

// Sum over the `lanes` lanes of a row (a power of two, aligned groups).
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  using namespace hk::detail;
  if (lanes > 1) v += dpp<kDppXor1>(v);
  if (lanes > 2) v += dpp<kDppXor2>(v);
  if (lanes > 4) v += dpp<kDppHalfMirror>(v);
  if (lanes > 8) v += dpp<kDppMirror>(v);
  if (lanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lanes > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Rows whose mean of squares (eps added) fp32 does not hold well: their sums are formed again from x times a power of
// two, and r from those. Under 2^-80 squares begin to lose digits (elements are under 2^-36 then, times 2^88
// their squares lie between 2^-122 and 2^104); where the sum passes fp32, elements of up to 2^128 times 2^-70
// have sums up to 2^124. r itself is a normal number for rows of 2^-126 to 2^126, and x r is then formed as for
// every other row. The branch that asks is the wave's, and leaves what the rows hold in registers as it is (8 x 1024
// tokens of 12 + 12 heads, without it and with it: bf16 -> fp32 forward 13.9 and 13.2 us, backward 19.6 and 20.3;
// bf16 -> bf16 11.4 and 11.2, 15.1 and 14.9; x scaled in its registers instead, backward 20.7 and 15.9).
__device__ __forceinline__ bool in_range(float mean) { return mean >= 0x1p-80f && mean < INFINITY; }
__device__ __forceinline__ float row_scale(float mean) {
  return in_range(mean) ? 1.0f : mean < 1.0f ? 0x1p88f : 0x1p-70f;
}

// Queries or keys: a strided [B, heads, T, d] tensor and what belongs to it.
struct Side {
  const void* x;
  const void* w;   // NULL: 1
  const void* dy;  // backward
  void* out;       // forward: y, backward: dx
  float* part;     // backward: partial sums of dw, one row of d a workgroup (NULL: none asked for)
  int heads, rows, blocks;
  int64_t xB, xM, xH, yB, yM, yH, oB, oM, oH;  // strides of x, dy and out
};
struct Args {
  Side side[2];
  Shape s;
  const float* cos;
  const float* sin;
  int64_t table_stride, table_rows;
  const int64_t* positions;  // NULL: the token's index
  int64_t pos_stride;
  int T;
  int first;  // forward: the launch's first workgroup
  float eps, inv_d;
};

__device__ __forceinline__ int64_t position(const Args& g, int b, int t) {
  return g.positions ? g.positions[b * g.pos_stride + t] : t;
}
// The cosines and sines of a unit at a position; NaN where the table has no such one.
template <int V, bool O>
__device__ __forceinline__ void angles(const Args& g, const Unit<V, O>& u, int64_t pos, float (&c)[V],
                                       float (&s)[V]) {
  if (pos < 0 || pos >= g.table_rows) {
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = s[e] = NAN;
  } else if (u.angle >= 0) {
    load_vec(g.cos + pos * g.table_stride + u.angle, c);
    load_vec(g.sin + pos * g.table_stride + u.angle, s);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = 1.f, s[e] = 0.f;
  }
}

template <class F, int V, bool O>
__device__ __forceinline__ void weights(const void* w, const Unit<V, O>& u, int d, float (&a)[V],
                                        float (&b)[V]) {
  if (w && u.on) {
    load_unit<F, V>(static_cast<const typename F::storage*>(w), u, d, a, b);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] = b[e] = 1.f;
  }
}

// U: units a lane holds (more than one only where a row needs more than 64 of them, V == 1). O: OVERLAP.
template <class FI, class FO, int V, int U, bool O>
__global__ __launch_bounds__(kThreads) void qk_forward(Args g) {
  const int group = blockIdx.x + g.first, which = group >= g.side[0].blocks ? 1 : 0;
  const Side& sd = g.side[which];
  const int block = group - (which ? g.side[0].blocks : 0);
  const int per_block = kThreads / g.s.lanes;
  const int row = block * per_block + threadIdx.x / g.s.lanes;
  const int j = threadIdx.x & (g.s.lanes - 1);
  if (row >= sd.rows) return;  // whole lane groups: the butterflies below stay inside a group
  const int token = row / sd.heads, head = row - token * sd.heads;
  const int b = token / g.T, t = token - b * g.T;
  const auto* x = static_cast<const typename FI::storage*>(sd.x) + b * sd.xB + t * sd.xM + head * sd.xH;
  auto* y = static_cast<typename FO::storage*>(sd.out) + b * sd.oB + t * sd.oM + head * sd.oH;
  float xa[U][V], xb[U][V], sum = 0.f;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const Unit<V, O> u(g.s, j + k * HK_WAVE);
    if (!u.on) {
#pragma unroll
      for (int e = 0; e < V; ++e) xa[k][e] = xb[k][e] = 0.f;
      continue;
    }
    load_unit<FI, V>(x, u, g.s.d, xa[k], xb[k]);
#pragma unroll
    for (int e = 0; e < V; ++e)
      sum += u.own_a(e, xa[k][e] * xa[k][e]) + u.own_b(e, xb[k][e] * xb[k][e]);
  }
  const float mean = lanes_sum(sum, g.s.lanes) * g.inv_d + g.eps;
  float r = __builtin_amdgcn_rsqf(mean);
  if (__builtin_expect(__ballot(!in_range(mean)) != 0, 0)) {
    const float by = row_scale(mean);
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Unit<V, O> u(g.s, j + k * HK_WAVE);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float a = xa[k][e] * by, bb = xb[k][e] * by;
        sum += u.own_a(e, a * a) + u.own_b(e, bb * bb);
      }
    }
    r = __builtin_amdgcn_rsqf(lanes_sum(sum, g.s.lanes) * g.inv_d + g.eps * by * by) * by;
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const Unit<V, O> u(g.s, j + k * HK_WAVE);
    if (!u.on) continue;
    float wa[V], wb[V], c[V], s[V], ya[V], yb[V];
    weights<FI, V>(sd.w, u, g.s.d, wa, wb);
    angles(g, u, position(g, b, t), c, s);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = xa[k][e] * r * wa[e], bb = xb[k][e] * r * wb[e];
      ya[e] = a * c[e] - bb * s[e];
      yb[e] = bb * c[e] + a * s[e];
    }
    store_unit<FO, V>(y, u, g.s.d, ya, yb);
  }
}

template <class FI, class FO, int V, int U, bool O>
__global__ __launch_bounds__(kBackThreads, 6) void qk_backward(Args g) {
  __shared__ float lds[kBackWaves][kMaxDim];
  const int which = static_cast<int>(blockIdx.x) >= g.side[0].blocks ? 1 : 0;
  const Side& sd = g.side[which];
  const int block = blockIdx.x - (which ? g.side[0].blocks : 0);
  const int per_block = kBackThreads / g.s.lanes;
  const int j = threadIdx.x & (g.s.lanes - 1);
  float wa[U][V], wb[U][V], da[U][V], db[U][V];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    weights<FI, V>(sd.w, Unit<V, O>(g.s, j + k * HK_WAVE), g.s.d, wa[k], wb[k]);
#pragma unroll
    for (int e = 0; e < V; ++e) da[k][e] = db[k][e] = 0.f;
  }
  for (int row = block * per_block + threadIdx.x / g.s.lanes; row < sd.rows;
       row += sd.blocks * per_block) {
    const int token = row / sd.heads, head = row - token * sd.heads;
    const int b = token / g.T, t = token - b * g.T;
    const auto* x = static_cast<const typename FI::storage*>(sd.x) + b * sd.xB + t * sd.xM + head * sd.xH;
    const auto* dy = static_cast<const typename FO::storage*>(sd.dy) + b * sd.yB + t * sd.yM + head * sd.yH;
    auto* dx = static_cast<typename FI::storage*>(sd.out) + b * sd.oB + t * sd.oM + head * sd.oH;
    const int64_t pos = position(g, b, t);
    float xa[U][V], xb[U][V], ga[U][V], gb[U][V], sum = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Unit<V, O> u(g.s, j + k * HK_WAVE);
      if (!u.on) {
#pragma unroll
        for (int e = 0; e < V; ++e) xa[k][e] = xb[k][e] = ga[k][e] = gb[k][e] = 0.f;
        continue;
      }
      float c[V], s[V], ya[V], yb[V];
      load_unit<FI, V>(x, u, g.s.d, xa[k], xb[k]);
      load_unit<FO, V>(dy, u, g.s.d, ya, yb);
      angles(g, u, pos, c, s);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        ga[k][e] = ya[e] * c[e] + yb[e] * s[e];
        gb[k][e] = yb[e] * c[e] - ya[e] * s[e];
        sum += u.own_a(e, xa[k][e] * xa[k][e]) + u.own_b(e, xb[k][e] * xb[k][e]);
        dot += u.own_a(e, ga[k][e] * wa[k][e] * xa[k][e]) + u.own_b(e, gb[k][e] * wb[k][e] * xb[k][e]);
      }
    }
    const float mean = lanes_sum(sum, g.s.lanes) * g.inv_d + g.eps;
    float r = __builtin_amdgcn_rsqf(mean);
    // mean(g w n) = r mean(g w x)
    float m = lanes_sum(dot, g.s.lanes) * g.inv_d * r;
    if (__builtin_expect(__ballot(!in_range(mean)) != 0, 0)) {
      const float by = row_scale(mean);
      sum = dot = 0.f;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const Unit<V, O> u(g.s, j + k * HK_WAVE);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float a = xa[k][e] * by, bb = xb[k][e] * by;
          sum += u.own_a(e, a * a) + u.own_b(e, bb * bb);
          dot += u.own_a(e, ga[k][e] * wa[k][e] * a) + u.own_b(e, gb[k][e] * wb[k][e] * bb);
        }
      }
      r = __builtin_amdgcn_rsqf(lanes_sum(sum, g.s.lanes) * g.inv_d + g.eps * by * by);
      m = lanes_sum(dot, g.s.lanes) * g.inv_d * r;
      r *= by;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Unit<V, O> u(g.s, j + k * HK_WAVE);
      float oa[V], ob[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float na = xa[k][e] * r, nb = xb[k][e] * r;
        da[k][e] += ga[k][e] * na;
        db[k][e] += gb[k][e] * nb;
        oa[e] = r * (ga[k][e] * wa[k][e] - na * m);
        ob[e] = r * (gb[k][e] * wb[k][e] - nb * m);
      }
      if (u.on) store_unit<FI, V>(dx, u, g.s.d, oa, ob);
    }
  }
  if (!sd.part) return;
  // the row groups of a wave, then the waves of the workgroup, in a fixed order
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const Unit<V, O> u(g.s, j + k * HK_WAVE);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      for (int step = g.s.lanes; step < HK_WAVE; step *= 2) {
        da[k][e] += __shfl_xor(da[k][e], step);
        db[k][e] += __shfl_xor(db[k][e], step);
      }
    }
    if (u.on && (threadIdx.x & 63) < g.s.lanes) {
      store_unit<hk::F32, V, false>(lds[threadIdx.x / HK_WAVE], u, g.s.d, da[k], db[k]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < g.s.d; i += kBackThreads) {
    float v = lds[0][i];
#pragma unroll
    for (int k = 1; k < kBackWaves; ++k) v += lds[k][i];
    sd.part[static_cast<int64_t>(block) * g.s.d + i] = v;
  }
}

// dw[i] (+)= the sum over n rows of part[n][d]; blockIdx.y: queries, keys. Each workgroup sums 16
// columns, its 64 row groups take every 64th row.
struct Weights {
  const float* part[2];
  float* dw[2];
  int n[2];
};
__global__ __launch_bounds__(1024) void qk_weight_sums(Weights a, int d, int accumulate) {
  __shared__ float lds[16][17];
  const int which = blockIdx.y, tx = threadIdx.x & 15, col = blockIdx.x * 16 + tx;
  const int grp = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  if (!a.dw[which]) return;
  float v = 0.f;
  if (col < d) {
    const float* p = a.part[which] + col;
    const int n = a.n[which];
    for (int i0 = grp; i0 < n; i0 += 512) {  // eight loads in flight
      float f[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = i0 + 64 * u < n ? p[static_cast<int64_t>(i0 + 64 * u) * d] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) v += f[u];
    }
  }
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  if ((threadIdx.x & 63) < 16) lds[wave][tx] = v;
  __syncthreads();
  if (threadIdx.x < 16 && col < d) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][tx];
    a.dw[which][col] = accumulate ? a.dw[which][col] + s : s;
  }
}

// ---- host ------------------------------------------------------------------------------------------
size_t elem_size(int type) { return type == HK_TYPE_F32 ? 4 : 2; }
bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

hipError_t check(const hk_qk_norm_rope_params* p, int type, bool backward) {
  HK_CHECK_ARG(p != nullptr && type >= HK_TYPE_F32 && type <= HK_TYPE_F16);
  HK_CHECK_ARG(p->B >= 0 && p->T >= 0 && p->q_heads >= 0 && p->k_heads >= 0);
  HK_CHECK_ARG(p->head_dim >= 1 && p->head_dim <= kMaxDim);
  HK_CHECK_ARG(p->rotary_dim >= 0 && p->rotary_dim <= p->head_dim && p->rotary_dim % 2 == 0);
  const int64_t tokens = static_cast<int64_t>(p->B) * p->T;
  HK_CHECK_ARG(tokens <= INT32_MAX / 2 && tokens * p->q_heads <= INT32_MAX / 2 &&
               tokens * p->k_heads <= INT32_MAX / 2);
  const size_t ei = elem_size(type), eo = p->f32_io ? 4 : ei;
  if (tokens == 0) return hipSuccess;
  if (p->rotary_dim > 0) {
    HK_CHECK_ARG(p->cos && p->sin && aligned_to(p->cos, 4) && aligned_to(p->sin, 4));
    HK_CHECK_ARG(p->table_rows >= 0 && p->table_stride >= p->rotary_dim / 2);
    HK_CHECK_ARG(p->positions != nullptr || p->T <= p->table_rows);
    HK_CHECK_ARG(aligned_to(p->positions, 8));
  }
  const void* x[2] = {p->q, p->k};
  const void* w[2] = {p->q_weight, p->k_weight};
  const void* y[2] = {backward ? p->dq_out : p->q_out, backward ? p->dk_out : p->k_out};
  const void* dx[2] = {p->dq, p->dk};
  const int heads[2] = {p->q_heads, p->k_heads};
  for (int i = 0; i < 2; ++i) {
    if (heads[i] == 0) continue;
    HK_CHECK_ARG(x[i] && y[i] && aligned_to(x[i], ei) && aligned_to(w[i], ei) && aligned_to(y[i], eo));
    HK_CHECK_ARG(!backward || (dx[i] && aligned_to(dx[i], ei)));
  }
  HK_CHECK_ARG(!backward || (aligned_to(p->dq_weight, 4) && aligned_to(p->dk_weight, 4)));
  return hipSuccess;
}

// Whether what a call writes lies apart: no two rows of it, nor one and what the call reads, share memory, but for
// an output that is its own side's input (in the backward pass, or the gradient of its output) row by row.
bool outputs_apart(const hk_qk_norm_rope_params* p, int type, bool backward) {
  const int64_t ei = elem_size(type), eo = p->f32_io ? 4 : ei, d = p->head_dim;
  auto tensor = [&](const void* t, int heads, int64_t elem, int64_t sB, int64_t sM, int64_t sH) {
    return hk::Rows(t, elem, d).along(p->B, elem * sB).along(heads, elem * sH).along(p->T, elem * sM);
  };
  const hk::Rows x[2] = {tensor(p->q, p->q_heads, ei, p->q_strideB, p->q_strideM, p->q_strideH),
                         tensor(p->k, p->k_heads, ei, p->k_strideB, p->k_strideM, p->k_strideH)};
  const hk::Rows y[2] = {  // the outputs, or their gradients
      tensor(backward ? p->dq_out : p->q_out, p->q_heads, eo, p->qo_strideB, p->qo_strideM, p->qo_strideH),
      tensor(backward ? p->dk_out : p->k_out, p->k_heads, eo, p->ko_strideB, p->ko_strideM, p->ko_strideH)};
  hk::Rows out[4] = {y[0], y[1], hk::Rows(nullptr, 4, d), hk::Rows(nullptr, 4, d)};
  if (backward) {
    out[0] = tensor(p->dq, p->q_heads, ei, p->dq_strideB, p->dq_strideM, p->dq_strideH);
    out[1] = tensor(p->dk, p->k_heads, ei, p->dk_strideB, p->dk_strideM, p->dk_strideH);
    if (p->q_heads > 0) out[2] = hk::Rows(p->dq_weight, 4, d);
    if (p->k_heads > 0) out[3] = hk::Rows(p->dk_weight, 4, d);
  }
  const int64_t half = p->rotary_dim / 2;
  const hk::Rows shared[5] = {
      hk::Rows(p->q_heads > 0 ? p->q_weight : nullptr, ei, d),
      hk::Rows(p->k_heads > 0 ? p->k_weight : nullptr, ei, d),
      hk::Rows(half > 0 ? p->cos : nullptr, 4, half).along(p->table_rows, 4 * p->table_stride),
      hk::Rows(half > 0 ? p->sin : nullptr, 4, half).along(p->table_rows, 4 * p->table_stride),
      hk::Rows(half > 0 ? p->positions : nullptr, 8, p->T).along(p->B, 8 * p->pos_strideB)};
  for (int i = 0; i < 4; ++i) {
    if (i < 2 && hk::overlaps_itself(out[i])) return false;
    for (int j = 0; j < i; ++j)
      if (hk::overlap(out[i], out[j])) return false;
    for (int j = 0; j < 2; ++j) {
      if (i == j ? hk::overlap_unless_same(out[i], x[j]) : hk::overlap(out[i], x[j])) return false;
      if (backward && (i == j ? hk::overlap_unless_same(out[i], y[j]) : hk::overlap(out[i], y[j]))) return false;
    }
    for (const hk::Rows& s : shared)
      if (hk::overlap(out[i], s)) return false;
  }
  return true;
}

// Pairs a unit holds: whole vectors of both halves of the rotated part and of what lies behind it. 8 (16-byte
// vectors of 16-bit elements) where a row is only read and written in 16 bits; 4 where outputs are fp32
// (stores through the caches, forward, 8 x 1024 tokens of 12 + 12 heads of 64, bf16 -> fp32: 17.5 and
// 16.2 us; bf16 -> bf16 the other way: 11.7 and 12.6; stored past them, as here, fp32 13.2 with 4, bf16 11.2 with
// 8), and in the backward pass, which holds weights and their gradients beside the row (110 registers a lane
// with 8: 25.4 us with dw, with 4 and three workgroups a CU 23.9; 16 + 4 heads of 128, fp16: 46.3 and 36.8).
// Parts that are no whole vectors of 4 keep them where they are long enough for the last unit to be moved
// back (8 x 1024 tokens, forward: 12 + 12 bf16 heads of 64 with 20 rotated 31.7 us one by one, 21.3 so; 8 + 8 of
// 90, all rotated, 41.2 and 16.5; fp16 of 96 with 50 rotated 43.6 and 17.4; backward 36.5, 49.1 and 51.5
// against 27.0, 21.3 and 22.9; an element-wise tail on each unit instead: 44.4, 31.5, 34.3 forward).
int units_of(int d, int rot, int v) { return (rot / 2 + v - 1) / v + (d - rot + 2 * v - 1) / (2 * v); }
bool whole_units(int d, int rot, int v) { return d % (2 * v) == 0 && rot % (2 * v) == 0; }
int unit_pairs(int type, int d, int rot, bool wide) {
  if (type != HK_TYPE_F32 && wide && whole_units(d, rot, 8)) return 8;
  for (int v = 4; v > 1; v /= 2)
    if ((rot == 0 || rot >= 2 * v) && (d == rot || d - rot >= 2 * v) && units_of(d, rot, v) <= HK_WAVE)
      return v;
  return 1;
}

Args make_args(const hk_qk_norm_rope_params* p, int v, bool backward) {
  Args g{};
  const int d = p->head_dim, rot = p->rotary_dim;
  g.s = Shape{d, rot, rot / 2, (rot / 2 + v - 1) / v, units_of(d, rot, v), 1, p->interleaved};
  while (g.s.lanes < g.s.units && g.s.lanes < HK_WAVE) g.s.lanes *= 2;
  g.cos = p->cos, g.sin = p->sin;
  g.table_stride = p->table_stride;
  // without a rotation no position is out of the table
  g.table_rows = p->rotary_dim > 0 ? p->table_rows : INT64_MAX;
  g.positions = p->rotary_dim > 0 ? p->positions : nullptr;
  g.pos_stride = p->pos_strideB;
  g.T = p->T;
  g.eps = p->eps;
  g.inv_d = 1.0f / static_cast<float>(p->head_dim);
  const int tokens = p->B * p->T;
  Side& q = g.side[0];
  q.x = p->q, q.w = p->q_weight, q.dy = p->dq_out, q.out = backward ? p->dq : p->q_out;
  q.heads = p->q_heads, q.rows = tokens * p->q_heads;
  q.xB = p->q_strideB, q.xM = p->q_strideM, q.xH = p->q_strideH;
  q.yB = p->qo_strideB, q.yM = p->qo_strideM, q.yH = p->qo_strideH;
  q.oB = backward ? p->dq_strideB : q.yB, q.oM = backward ? p->dq_strideM : q.yM;
  q.oH = backward ? p->dq_strideH : q.yH;
  Side& k = g.side[1];
  k.x = p->k, k.w = p->k_weight, k.dy = p->dk_out, k.out = backward ? p->dk : p->k_out;
  k.heads = p->k_heads, k.rows = tokens * p->k_heads;
  k.xB = p->k_strideB, k.xM = p->k_strideM, k.xH = p->k_strideH;
  k.yB = p->ko_strideB, k.yM = p->ko_strideM, k.yH = p->ko_strideH;
  k.oB = backward ? p->dk_strideB : k.yB, k.oM = backward ? p->dk_strideM : k.yM;
  k.oH = backward ? p->dk_strideH : k.yH;
  const int64_t per_block = (backward ? kBackThreads : kThreads) / g.s.lanes;
  // Backward: one round of workgroups, each of which leaves one row of partial sums, and as many rows for
  // each of their lane groups as that takes.
  int64_t passes = 1;
  if (backward)
    passes = hk::ceil_div(static_cast<int64_t>(q.rows) + k.rows,
                          per_block * kBackPerCu * hk::device_cu_count());
  for (Side& s : g.side)
    s.blocks = static_cast<int>(hk::ceil_div(s.rows, per_block * (passes > 0 ? passes : 1)));
  return g;
}

template <class FI, class FO, int V, int U, bool O>
hipError_t launch(const Args& args, bool backward, hipStream_t stream) {
  Args g = args;
  const int blocks = g.side[0].blocks + g.side[1].blocks;
  if (backward) {
    if constexpr (V == 8) return hipErrorInvalidValue;  // unit_pairs
    else hipLaunchKernelGGL((qk_backward<FI, FO, V, U, O>), dim3(blocks), dim3(kBackThreads), 0, stream, g);
    return hk::launch_status();
  }
  // a dimension of a grid has under 2^32 threads, and more of them run as their number modulo 2^32
  constexpr int kMost = 1 << 23;
  for (; g.first < blocks; g.first += kMost) {
    hipLaunchKernelGGL((qk_forward<FI, FO, V, U, O>), dim3(std::min(kMost, blocks - g.first)), dim3(kThreads),
                       0, stream, g);
    HK_RETURN_IF_ERROR(hk::launch_status());
  }
  return hipSuccess;
}
template <class FI, class FO>
hipError_t by_unit(const Args& g, int v, bool backward, hipStream_t stream) {
  if constexpr (FI::kPerVec == 8 && FO::kPerVec == 8)
    if (v == 8) return launch<FI, FO, 8, 1, false>(g, backward, stream);
  if (v == 4)
    return whole_units(g.s.d, g.s.rot, 4) ? launch<FI, FO, 4, 1, false>(g, backward, stream)
                                          : launch<FI, FO, 4, 1, true>(g, backward, stream);
  if (v == 2) return launch<FI, FO, 2, 1, true>(g, backward, stream);
  return g.s.units > HK_WAVE ? launch<FI, FO, 1, 2, false>(g, backward, stream)
                             : launch<FI, FO, 1, 1, false>(g, backward, stream);
}
hipError_t by_type(const Args& g, int type, bool f32_io, int v, bool backward, hipStream_t stream) {
  using namespace hk;
  if (type == HK_TYPE_F32) return by_unit<F32, F32>(g, v, backward, stream);
  if (type == HK_TYPE_BF16)
    return f32_io ? by_unit<BF16, F32>(g, v, backward, stream) : by_unit<BF16, BF16>(g, v, backward, stream);
  return f32_io ? by_unit<F16, F32>(g, v, backward, stream) : by_unit<F16, F16>(g, v, backward, stream);
}

size_t partial_bytes(const Args& g) {
  return static_cast<size_t>(g.side[0].blocks + g.side[1].blocks) * g.s.d * sizeof(float);
}

}  // namespace

extern "C" hipError_t hk_qk_norm_rope_forward(const hk_qk_norm_rope_params* p, int type,
                                              hipStream_t stream) {
  HK_RETURN_IF_ERROR(check(p, type, false));
  const int v = unit_pairs(type, p->head_dim, p->rotary_dim, !p->f32_io);
  const Args g = make_args(p, v, false);
  if (g.side[0].rows + g.side[1].rows == 0) return hipSuccess;
  HK_CHECK_ARG(outputs_apart(p, type, false));
  return by_type(g, type, p->f32_io, v, false, stream);
}

extern "C" int64_t hk_qk_norm_rope_workspace(const hk_qk_norm_rope_params* p, int type) {
  if (check(p, type, true) != hipSuccess) return -1;
  if (!p->dq_weight && !p->dk_weight) return 0;
  return static_cast<int64_t>(
      partial_bytes(make_args(p, unit_pairs(type, p->head_dim, p->rotary_dim, false), true)));
}

extern "C" hipError_t hk_qk_norm_rope_backward(const hk_qk_norm_rope_params* p, int type,
                                               void* workspace, int64_t workspace_bytes,
                                               hipStream_t stream) {
  HK_RETURN_IF_ERROR(check(p, type, true));
  HK_CHECK_ARG(outputs_apart(p, type, true));
  const int v = unit_pairs(type, p->head_dim, p->rotary_dim, false);
  Args g = make_args(p, v, true);
  Weights w{{nullptr, nullptr},
            {p->q_heads ? p->dq_weight : nullptr, p->k_heads ? p->dk_weight : nullptr},
            {g.side[0].blocks, g.side[1].blocks}};
  const bool sums = w.dw[0] || w.dw[1];
  if (sums && g.side[0].rows + g.side[1].rows > 0) {
    const size_t bytes = partial_bytes(g);
    void* ws = workspace;
    if (ws) {
      HK_CHECK_ARG(workspace_bytes >= static_cast<int64_t>(bytes) && aligned_to(ws, 4));
    } else {
      // a graph would keep the stream's workspace, which other graphs and eager calls write too
      if (hk::stream_capturing(stream)) return hipErrorStreamCaptureUnsupported;
      HK_RETURN_IF_ERROR(hk::device_workspace(bytes, stream, &ws));
    }
    float* part = static_cast<float*>(ws);
    for (int i = 0; i < 2; ++i) {
      if (w.dw[i]) w.part[i] = g.side[i].part = part;
      part += static_cast<int64_t>(g.side[i].blocks) * g.s.d;
    }
  }
  if (g.side[0].rows + g.side[1].rows > 0)
    HK_RETURN_IF_ERROR(by_type(g, type, p->f32_io, v, true, stream));
  if (!sums || (p->accumulate && g.side[0].rows + g.side[1].rows == 0)) return hipSuccess;
  // without rows the sums are zero
  hipLaunchKernelGGL(qk_weight_sums, dim3(static_cast<unsigned>((g.s.d + 15) / 16), 2), dim3(1024), 0,
                     stream, w, g.s.d, p->accumulate ? 1 : 0);
  return hk::launch_status();
}

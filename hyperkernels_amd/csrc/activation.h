// activation.h - activation functions and their derivatives in fp32.
#pragma once

#include "hk_device.h"

namespace hk {

// With u = c (x + a x^3) (c = sqrt(2/pi), a = 0.044715, the Hendrycks & Gimpel tanh fit):
// (1 + tanh(u)) / 2 = sigmoid(2u) = 1 / (1 + 2^(-2 log2(e) u)): no cancellation for u << 0,
// where 1 + tanh(u) formed from a rounded tanh loses most of its digits. The exponent is
// -2 log2(e) u = x (k1 + k2 x^2) with the constants folded (float64-rounded once):
//   k1 = -2 log2(e) c, k2 = k1 a.
// 2^t overflow (x << 0) gives s = 0 and underflow (x >> 0) gives s = 1, the correct limits.
// v_exp_f32 is the hardware 2^t (about 1 ulp) and v_rcp_f32 the hardware reciprocal (1 ulp):
// s carries a few ulp of relative error everywhere.
constexpr float kK1 = -2.302208198144325f;   // -2 log2(e) sqrt(2/pi)
constexpr float kK2 = -0.1029432395800235f;  // kK1 * 0.044715
constexpr float kC = 0.7978845608028654f;    // sqrt(2/pi)
constexpr float kC3a = 0.10703222440890f;    // 3 * 0.044715 * sqrt(2/pi)

__device__ __forceinline__ float sigmoid_2u(float x, float x2) {
  const float t = x * __builtin_fmaf(kK2, x2, kK1);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}

// GELU(x) = 0.5 x (1 + tanh(u)) = x s
__device__ __forceinline__ float gelu_fwd(float x) { return x * sigmoid_2u(x, x * x); }

// GELU'(x) = 0.5 (1 + th) + 0.5 x (1 - th^2) du = s + 2 x du s (1 - s), with s as above,
// 1 - th^2 = (1 - th)(1 + th) = 4 s (1 - s) and du = c (1 + 3 a x^2).
__device__ __forceinline__ float gelu_grad(float x) {
  const float x2 = x * x;
  const float s = sigmoid_2u(x, x2);
  const float two_x_du = 2.0f * x * __builtin_fmaf(kC3a, x2, kC);
  return __builtin_fmaf(two_x_du, __builtin_fmaf(-s, s, s), s);
}

// An activation HK_ACT_* as a call's kernels evaluate it, the same for all of its elements. GELU and SiLU
// are both x s with s = 1 / (1 + e^-q), q = x (c1 + c3 x^2): one code for the two, with the constants
// of t = -log2(e) q = x (k1 + k2 x^2) and of q'. Derivative: s + x q' s (1 - s). SiLU's cubic terms are 0;
// 10^-30 in their place, which x^2 under 10^19 cannot raise to the last bit of k1, keeps an infinite
// x^2 from meeting a 0.
struct Activation {
  int kind;       // HK_ACT_*
  float k1, k2;   // of t
  float d1, d3;   // q' = d1 + d3 x^2
};
__host__ __device__ __forceinline__ Activation make_activation(int kind) {
  if (kind == HK_ACT_GELU) return Activation{kind, kK1, kK2, 2.0f * kC, 2.0f * kC3a};
  return Activation{kind, -1.442695040888963f, -1e-30f, 1.0f, 1e-30f};  // SiLU
}
// 2^t overflows to s = 0 and underflows to s = 1, the right limits. ReLU keeps a NaN.
template <int N>
__device__ __forceinline__ void activate(const Activation& f, float (&x)[N]) {
  if (f.kind >= HK_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float t = x[e] * __builtin_fmaf(f.k2, x[e] * x[e], f.k1);
      x[e] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
    }
  } else if (f.kind == HK_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = x[e] < 0.0f ? 0.0f : x[e];
  }
}
// d *= the derivative at x (ReLU: 0 at 0).
template <int N>
__device__ __forceinline__ void scale_by_grad(const Activation& f, const float (&x)[N], float (&d)[N]) {
  if (f.kind >= HK_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x2 = x[e] * x[e];
      const float s = __builtin_amdgcn_rcpf(
          1.0f + __builtin_amdgcn_exp2f(x[e] * __builtin_fmaf(f.k2, x2, f.k1)));
      // s (1 - s) is 0 long before x q' overflows; a NaN in x is one in s
      const float xq = __builtin_amdgcn_fmed3f(x[e] * __builtin_fmaf(f.d3, x2, f.d1), -1e30f, 1e30f);
      d[e] *= __builtin_fmaf(xq, __builtin_fmaf(-s, s, s), s);
    }
  } else if (f.kind == HK_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float s = x[e] > 0.0f ? 1.0f : 0.0f;
      d[e] *= x[e] == x[e] ? s : x[e];
    }
  }
}

}  // namespace hk

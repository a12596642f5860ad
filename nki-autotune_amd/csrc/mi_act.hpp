// mi_act.hpp -- the activations of the epilogue products and their slopes,
// fp32, for the hardware's exp2 and reciprocal (1 ulp each).
//
//   relu       max(x, 0)
//   gelu       x P(x), P(x) = erfc(-x / sqrt 2) / 2
//   gelu_tanh  x / (1 + exp(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3)  (= x (1 + tanh u) / 2)
//   silu       x / (1 + exp(-x))
//
// An epilogue runs on VALUs while the matrix cores wait, so each is a dozen
// instructions.  erfc goes by exp(-x^2/2) q(t), t = 1 / (1 + 0.36 |x|), with q
// of degree 7 fitted here to erfc(z) exp(z^2) / 2 at z = |x| / sqrt 2 for the
// least relative error over |x| <= 14 (9e-7; past it the result is under
// 1e-43): relative, so the left tail keeps its digits, where 1 + erf loses
// them all.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mi_kernels.h"

namespace mi {

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

constexpr float kGeluK = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float kGeluC = 0.044715f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

// P(x), and exp(-x^2 / 2) beside it.
__device__ __forceinline__ float normal_cdf(float x, float& bell) {
  const float z = __builtin_fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, z, 1.0f));
  float q = 0.047065752f;
  q = __builtin_fmaf(q, t, -0.179797258f);
  q = __builtin_fmaf(q, t, 0.180998617f);
  q = __builtin_fmaf(q, t, 0.0265183863f);
  q = __builtin_fmaf(q, t, 0.139730653f);
  q = __builtin_fmaf(q, t, 0.141770359f);
  q = __builtin_fmaf(q, t, 0.143713195f);
  bell = exp_fast(-0.5f * x * x);
  const float h = bell * (q * t);
  return x >= 0.0f ? 1.0f - h : h;
}

__device__ __forceinline__ float sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == MI_ACT_RELU) return x < 0.0f ? 0.0f : x;
  if constexpr (ACT == MI_ACT_GELU) {
    float bell;
    return x * normal_cdf(x, bell);
  }
  if constexpr (ACT == MI_ACT_GELU_TANH) return x * sigmoid_fast(2.0f * kGeluK * x * (1.0f + kGeluC * x * x));
  if constexpr (ACT == MI_ACT_SILU) return x * sigmoid_fast(x);
  return x;
}

// d act / dx.  In the far tails the slope's second term is a product of a 0
// and a large number: it counts as 0.
template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
  if constexpr (ACT == MI_ACT_RELU) return x > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == MI_ACT_GELU) {
    float bell;
    const float p = normal_cdf(x, bell);
    return p + (bell == 0.0f ? 0.0f : x * bell * kInvSqrt2Pi);
  }
  if constexpr (ACT == MI_ACT_GELU_TANH || ACT == MI_ACT_SILU) {
    const float u = ACT == MI_ACT_SILU ? x : 2.0f * kGeluK * x * (1.0f + kGeluC * x * x);
    const float du = ACT == MI_ACT_SILU ? 1.0f : 2.0f * kGeluK * (1.0f + 3.0f * kGeluC * x * x);
    const float s = sigmoid_fast(u), ds = s * (1.0f - s);
    return s + (ds == 0.0f ? 0.0f : x * ds * du);
  }
  return 1.0f;
}

// f(integral_constant<ACT>) for the run-time `act`: a wave-uniform branch.
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case MI_ACT_RELU: f(std::integral_constant<int, MI_ACT_RELU>{}); break;
    case MI_ACT_GELU: f(std::integral_constant<int, MI_ACT_GELU>{}); break;
    case MI_ACT_GELU_TANH: f(std::integral_constant<int, MI_ACT_GELU_TANH>{}); break;
    case MI_ACT_SILU: f(std::integral_constant<int, MI_ACT_SILU>{}); break;
    default: f(std::integral_constant<int, MI_ACT_NONE>{}); break;
  }
}

}  // namespace mi

// Arithmetic of the gated linear recurrence's gates, shared by its kernels.
//
//   r = sigmoid(gate), i = sigmoid(input_gate)
//   with decay:  log2 a = k r, k = -decay_scale softplus(decay) log2 e;  beta^2 = 1 - a^2
//   without:     a = r, beta = 1 - r
//
// exp2, reciprocal and square root are the hardware's (1 ulp); everything is fp32.
#pragma once

#include "ops_common.h"

namespace ccv1d {
namespace ops {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
}

// k of a channel: log2 a = k * r.
__device__ __forceinline__ float decay_rate(float decay, float scale) {
  const float sp = decay > 20.0f ? decay : log1pf(expf(decay));
  return -scale * sp * kLog2e;
}

// d softplus / softplus: what turns the sum of dL/d(log a) log a into the gradient of decay. Tends
// to 1 as decay falls, where softplus itself underflows.
__device__ __forceinline__ float decay_ratio(float decay) {
  if (decay < -20.0f) return 1.0f;
  const float sp = decay > 20.0f ? decay : log1pf(expf(decay));
  return 1.0f / ((1.0f + expf(-decay)) * sp);
}

// 1 - a^2 from log2 a: below 0.35 of -2 ln a the difference cancels, and the series of
// -expm1(y), y = 2 ln a, is used instead (its next term is 2e-8 of the result there).
__device__ __forceinline__ float one_minus_square(float log2a, float a) {
  const float y = log2a * (2.0f * kLn2);
  float p = fmaf(y, 1.0f / 5040.0f, 1.0f / 720.0f);
  p = fmaf(y, p, 1.0f / 120.0f);
  p = fmaf(y, p, 1.0f / 24.0f);
  p = fmaf(y, p, 1.0f / 6.0f);
  p = fmaf(y, p, 0.5f);
  p = fmaf(y, p, 1.0f);
  return y > -0.35f ? -y * p : fmaf(-a, a, 1.0f);
}

// Without decay: a = sigmoid(g), beta = 1 - a without cancellation. Past 2^126 the exponential is
// held there (a stays a normal number and beta is 1); a NaN passes.
__device__ __forceinline__ void plain_gate(float g, float& a, float& beta) {
  const float z = -kLog2e * g;
  const float e = __builtin_amdgcn_exp2f(z > 126.0f ? 126.0f : z);
  a = __builtin_amdgcn_rcpf(1.0f + e);
  beta = e * a;
}

}  // namespace ops
}  // namespace ccv1d

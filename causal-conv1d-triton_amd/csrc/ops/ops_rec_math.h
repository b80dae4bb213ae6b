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
constexpr float kLog2eLow = 1.92596299112661746887e-8f;  // log2 e - kLog2e
constexpr float kLn2 = 0.69314718055994530942f;

// exp(-z) = 2^t, t = -z log2 e. The rounding of t, |t| 2^-24, is a relative error of the result that
// grows with |z|. For fp32 inputs its residue is added back (4 operations, and twice the bytes per
// element to hide them); for 16-bit ones it lies far below the rounding of what is stored. t is held
// at 126, so that 1 / (1 + 2^t) stays a normal number; a NaN passes.
template <typename T>
__device__ __forceinline__ float exp_minus(float z) {
  float t = -kLog2e * z;
  if constexpr (sizeof(T) == 4) {
    const float rest = fmaf(z, -kLog2eLow, fmaf(z, -kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t > 126.0f ? 126.0f : t);
    return t > 126.0f ? e : fmaf(e, kLn2 * rest, e);
  }
  return __builtin_amdgcn_exp2f(t > 126.0f ? 126.0f : t);
}

// s = sigmoid(z), and 1 - s without cancellation.
template <typename T>
__device__ __forceinline__ void sigmoid_pair(float z, float& s, float& rest) {
  const float e = exp_minus<T>(z);
  s = __builtin_amdgcn_rcpf(1.0f + e);
  rest = e * s;
}

template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + exp_minus<T>(z));
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

// The factor of the state before a row and that of the row's own i * x.
template <typename T, bool DECAY>
__device__ __forceinline__ void forget(float k, float gate, float& a, float& beta) {
  if constexpr (DECAY) {
    const float l = k * sigmoid<T>(gate);
    a = __builtin_amdgcn_exp2f(l);
    beta = __builtin_amdgcn_sqrtf(one_minus_square(l, a));
  } else {
    sigmoid_pair<T>(gate, a, beta);
  }
}

}  // namespace ops
}  // namespace ccv1d

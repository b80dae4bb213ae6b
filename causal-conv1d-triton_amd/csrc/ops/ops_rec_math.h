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
// element to hide them). For 16-bit ones it is left in: a sigmoid takes at most |z| 2^-24 of itself from it,
// and that only far below zero, where it is small; so it lies far below the rounding of what is stored in 16
// bits, and is of the size of fp32's own in the fp32 results (states, the gradients of decay and states). t is held
// at 126, so that 1 / (1 + 2^t) stays a normal number. Past 2^-126 and 2^126 the residue, which is no
// number for an infinite t, is left out; a NaN passes through it.
template <typename T>
__device__ __forceinline__ float exp_minus(float z) {
  float t = -kLog2e * z;
  if constexpr (sizeof(T) == 4) {
    const float rest = fmaf(z, -kLog2eLow, fmaf(z, -kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(fminf(t, 126.0f));
    return fabsf(t) > 126.0f ? e : fmaf(e, kLn2 * rest, e);
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

// The same where 1 - s is only used as a factor of s, so that it need not be right once s is zero: an
// operation less. e is held below infinity in it, which would make no number of that zero.
template <typename T>
__device__ __forceinline__ void sigmoid_and_rest(float z, float& s, float& rest) {
  if constexpr (sizeof(T) == 4) return sigmoid_pair<T>(z, s, rest);
  const float e = __builtin_amdgcn_exp2f(-kLog2e * z);
  s = __builtin_amdgcn_rcpf(1.0f + e);
  rest = fminf(e, 8.507059e37f) * s;  // 2^126
}

// The same where a NaN need not pass (a factor beside it carries it): one operation less in 16 bits.
template <typename T>
__device__ __forceinline__ void sigmoid_pair_of_number(float z, float& s, float& rest) {
  if constexpr (sizeof(T) == 4) return sigmoid_pair<T>(z, s, rest);
  const float e = __builtin_amdgcn_exp2f(fminf(-kLog2e * z, 126.0f));
  s = __builtin_amdgcn_rcpf(1.0f + e);
  rest = e * s;
}

// sigmoid(z) alone, where 2^t may pass the largest number and the result reach zero.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_rcpf(1.0f + exp_minus<T>(z));
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
}

// k of a channel: log2 a = k * r. softplus = log(1 + e), e = exp(decay): for e below 0.1, where a decay
// that lets a channel remember lies, its series (the next term is 2e-8 of it), else the library's.
__device__ __forceinline__ float decay_rate(float decay, float scale) {
  const float e = exp_minus<float>(-decay);
  float sp = fmaf(e, 1.0f / 7.0f, -1.0f / 6.0f);
  sp = fmaf(e, sp, 1.0f / 5.0f);
  sp = fmaf(e, sp, -1.0f / 4.0f);
  sp = fmaf(e, sp, 1.0f / 3.0f);
  sp = fmaf(e, sp, -1.0f / 2.0f);
  sp = fmaf(e * e, sp, e);
  if (!(decay < -2.3f)) sp = decay > 20.0f ? decay : log1pf(expf(decay));
  return -scale * sp * kLog2e;
}

// d softplus / softplus: what turns the sum of dL/d(log a) log a into the gradient of decay. Tends
// to 1 as decay falls, where softplus itself underflows.
__device__ __forceinline__ float decay_ratio(float decay) {
  if (decay < -20.0f) return 1.0f;
  const float sp = decay > 20.0f ? decay : log1pf(expf(decay));
  return 1.0f / ((1.0f + expf(-decay)) * sp);
}

// 1 - a^2 = 2 a sinh(-ln a) from log2 a, without the difference's cancellation: sinh's series, to the
// 11th power, up to |ln a| = 1 (the next term is 3e-8 of it), beyond which 1 - a^2 itself is exact
// enough. A slow channel, |ln a| <= 1/4 even at an open gate (which its decay alone decides), does
// with the 5th power (5e-8). Where all channels of a wave are slow the rest is left out (SLOW); where
// not, a slow channel's higher powers count zero times, so that its values do not depend on its
// neighbours.
__device__ __forceinline__ bool slow_channel(float k) { return k >= -0.25f * kLog2e; }

constexpr float sinh_coefficient(double factorial, int power) {
  double v = -2.0 / factorial;
  for (int i = 0; i < power; ++i) v *= 0.69314718055994530942;
  return (float)v;
}

// 0 for a slow channel, which leaves the higher powers out; else 1.
__device__ __forceinline__ float sinh_tail(float k) { return slow_channel(k) ? 0.0f : 1.0f; }

template <bool SLOW>
__device__ __forceinline__ float one_minus_square(float tail, float log2a, float a) {
  const float l2 = log2a * log2a;
  float p = sinh_coefficient(120.0, 5);
  if constexpr (!SLOW) {
    float t = fmaf(l2, sinh_coefficient(39916800.0, 11), sinh_coefficient(362880.0, 9));
    t = fmaf(l2, t, sinh_coefficient(5040.0, 7));
    p = fmaf(l2 * tail, t, p);
  }
  p = fmaf(l2, p, sinh_coefficient(6.0, 3));
  p = fmaf(l2, p, sinh_coefficient(1.0, 1));
  p = log2a * a * p;
  if constexpr (SLOW) return p;
  return log2a < -kLog2e ? fmaf(-a, a, 1.0f) : p;
}

// The factor of the state before a row and that of the row's own i * x.
template <typename T, bool DECAY, bool SLOW>
__device__ __forceinline__ void forget(float k, float tail, float gate, float& a, float& beta) {
  if constexpr (DECAY) {
    const float l = k * sigmoid<T>(gate);
    a = __builtin_amdgcn_exp2f(l);
    beta = __builtin_amdgcn_sqrtf(one_minus_square<SLOW>(tail, l, a));
  } else {
    sigmoid_pair<T>(gate, a, beta);
  }
}

}  // namespace ops
}  // namespace ccv1d

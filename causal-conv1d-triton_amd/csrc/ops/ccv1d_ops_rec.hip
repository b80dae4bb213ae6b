// The gated linear recurrence: one lane walks one channel of one sequence.
#include "ops_rec_math.h"

namespace ccv1d {
namespace ops {

namespace {

// One row's forward: the factor of the state before it and its own contribution.
template <bool DECAY>
__device__ __forceinline__ void coefficients(float k, float gate, float& r, float& log2a, float& a,
                                             float& beta) {
  if constexpr (DECAY) {
    r = sigmoid(gate);
    log2a = k * r;
    a = __builtin_amdgcn_exp2f(log2a);
    beta = __builtin_amdgcn_sqrtf(one_minus_square(log2a, a));
  } else {
    plain_gate(gate, a, beta);
    r = a;
    log2a = 0.0f;
  }
}

struct Row {
  bool pad, first;  // padding; the state starts anew
};

__device__ __forceinline__ Row row_of(const int32_t* seq, int64_t t) {
  Row w{false, false};
  if (seq) {
    const int32_t id = seq[t];
    w.pad = id < 0;
    w.first = t > 0 && seq[t - 1] != id;
  }
  return w;
}

template <typename T, bool DECAY>
__global__ __launch_bounds__(64) void rec_fwd_kernel(ccv1d_rec_args p) {
  const int64_t nc = (p.dim + 63) / 64;
  const int64_t b = blockIdx.x / nc, d = (blockIdx.x % nc) * 64 + threadIdx.x;
  if (d >= p.dim) return;
  const T* x = static_cast<const T*>(p.x) + b * p.x_stride_b + d;
  const T* g = static_cast<const T*>(p.gate) + b * p.gate_stride_b + d;
  const T* ig = p.input_gate ? static_cast<const T*>(p.input_gate) + b * p.input_gate_stride_b + d
                             : nullptr;
  const int32_t* seq = p.seq_idx ? p.seq_idx + b * p.seqlen : nullptr;
  T* out = static_cast<T*>(p.out) + b * p.seqlen * p.dim + d;
  const int64_t ns = (p.seqlen + CCV1D_REC_SAVED_ROWS - 1) / CCV1D_REC_SAVED_ROWS;
  float* saved = p.saved ? p.saved + b * ns * p.dim + d : nullptr;
  const float k = DECAY ? decay_rate(p.decay[d], p.decay_scale) : 0.0f;
  float h = p.initial_states ? p.initial_states[b * p.dim + d] : 0.0f;
  for (int64_t t = 0; t < p.seqlen; ++t) {
    if (saved && t % CCV1D_REC_SAVED_ROWS == 0) saved[t / CCV1D_REC_SAVED_ROWS * p.dim] = h;
    float r, l, a, beta;
    coefficients<DECAY>(k, to_f32(g[t * p.gate_stride_t]), r, l, a, beta);
    float u = beta * to_f32(x[t * p.x_stride_t]);
    if (ig) u *= sigmoid(to_f32(ig[t * p.input_gate_stride_t]));
    const Row w = row_of(seq, t);
    h = w.pad ? 0.0f : w.first ? u : fmaf(a, h, u);
    out[t * p.dim] = static_cast<T>(h);
  }
  if (p.final_states) p.final_states[b * p.dim + d] = h;
}

template <typename T, bool DECAY>
__global__ __launch_bounds__(64) void rec_bwd_kernel(ccv1d_rec_args p) {
  const int64_t nc = (p.dim + 63) / 64;
  const int64_t b = blockIdx.x / nc, d = (blockIdx.x % nc) * 64 + threadIdx.x;
  if (d >= p.dim) return;
  const T* x = static_cast<const T*>(p.x) + b * p.x_stride_b + d;
  const T* g = static_cast<const T*>(p.gate) + b * p.gate_stride_b + d;
  const T* ig = p.input_gate ? static_cast<const T*>(p.input_gate) + b * p.input_gate_stride_b + d
                             : nullptr;
  const T* dy = static_cast<const T*>(p.dout) + b * p.dout_stride_b + d;
  const int32_t* seq = p.seq_idx ? p.seq_idx + b * p.seqlen : nullptr;
  const int64_t base = b * p.seqlen * p.dim + d;
  T* dx = static_cast<T*>(p.dx) + base;
  T* dg = static_cast<T*>(p.dgate) + base;
  T* dig = ig ? static_cast<T*>(p.dinput_gate) + base : nullptr;
  float* before = static_cast<float*>(p.workspace) + base;  // the state in front of each row
  const float k = DECAY ? decay_rate(p.decay[d], p.decay_scale) : 0.0f;
  float h = p.initial_states ? p.initial_states[b * p.dim + d] : 0.0f;
  for (int64_t t = 0; t < p.seqlen; ++t) {
    float r, l, a, beta;
    coefficients<DECAY>(k, to_f32(g[t * p.gate_stride_t]), r, l, a, beta);
    float u = beta * to_f32(x[t * p.x_stride_t]);
    if (ig) u *= sigmoid(to_f32(ig[t * p.input_gate_stride_t]));
    const Row w = row_of(seq, t);
    const float hp = w.pad || w.first ? 0.0f : h;
    before[t * p.dim] = hp;
    h = w.pad ? 0.0f : fmaf(a, hp, u);
  }
  float c = p.dfinal_states ? p.dfinal_states[b * p.dim + d] : 0.0f;  // what reaches row t's state
  float dk = 0.0f;
  for (int64_t t = p.seqlen - 1; t >= 0; --t) {
    const Row w = row_of(seq, t);
    if (w.pad) {
      c = 0.0f;
      dx[t * p.dim] = static_cast<T>(0.0f);
      dg[t * p.dim] = static_cast<T>(0.0f);
      if (dig) dig[t * p.dim] = static_cast<T>(0.0f);
      continue;
    }
    float r, l, a, beta;
    coefficients<DECAY>(k, to_f32(g[t * p.gate_stride_t]), r, l, a, beta);
    const float xv = to_f32(x[t * p.x_stride_t]), hp = before[t * p.dim];
    const float i = ig ? sigmoid(to_f32(ig[t * p.input_gate_stride_t])) : 1.0f;
    const float dh = to_f32(dy[t * p.dout_stride_t]) + c;
    dx[t * p.dim] = static_cast<T>(dh * beta * i);
    if (dig) dig[t * p.dim] = static_cast<T>(dh * beta * xv * i * (1.0f - i));
    if constexpr (DECAY) {
      const float la = l * kLn2, over = beta > 0.0f ? la / beta : 0.0f;
      const float q = dh * (la * a * hp - i * xv * a * a * over);
      dg[t * p.dim] = static_cast<T>(q * (1.0f - r));
      dk += q;
    } else {
      dg[t * p.dim] = static_cast<T>(dh * (hp - i * xv) * a * beta);
    }
    c = w.first ? 0.0f : a * dh;
  }
  if (p.dinitial_states) p.dinitial_states[b * p.dim + d] = c;
  if constexpr (DECAY) {
    static_cast<float*>(p.workspace)[p.batch * p.seqlen * p.dim + b * p.dim + d] = dk;
  }
}

__global__ __launch_bounds__(64) void rec_reduce_kernel(const float* part, int64_t rows, int64_t dim,
                                                        const float* decay, float* ddecay) {
  const int64_t d = blockIdx.x * 64 + threadIdx.x;
  if (d >= dim) return;
  float s = 0.0f;
  for (int64_t i = 0; i < rows; ++i) s += part[i * dim + d];
  ddecay[d] = s * decay_ratio(decay[d]);
}

template <typename T, bool DECAY>
__global__ __launch_bounds__(64) void rec_update_kernel(ccv1d_rec_update_args p) {
  const int64_t nc = (p.dim + 63) / 64;
  const int64_t row = blockIdx.x / nc, d = (blockIdx.x % nc) * 64 + threadIdx.x;
  if (d >= p.dim) return;
  const int64_t slot = p.state_indices ? p.state_indices[row] : row;
  float h = 0.0f;
  if (slot >= 0 && slot < p.slots) {
    float r, l, a, beta;
    const float k = DECAY ? decay_rate(p.decay[d], p.decay_scale) : 0.0f;
    coefficients<DECAY>(k, to_f32(static_cast<const T*>(p.gate)[row * p.gate_stride + d]), r, l, a, beta);
    float u = beta * to_f32(static_cast<const T*>(p.x)[row * p.x_stride + d]);
    if (p.input_gate)
      u *= sigmoid(to_f32(static_cast<const T*>(p.input_gate)[row * p.input_gate_stride + d]));
    float* st = p.state + slot * p.state_stride + d;
    h = fmaf(a, *st, u);
    *st = h;
  }
  static_cast<T*>(p.out)[row * p.dim + d] = static_cast<T>(h);
}

template <typename T>
hipError_t fwd_t(const ccv1d_rec_args& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.batch * ((a.dim + 63) / 64)));
  if (a.decay) rec_fwd_kernel<T, true><<<grid, 64, 0, s>>>(a);
  else rec_fwd_kernel<T, false><<<grid, 64, 0, s>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t bwd_t(const ccv1d_rec_args& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.batch * ((a.dim + 63) / 64)));
  if (a.decay) rec_bwd_kernel<T, true><<<grid, 64, 0, s>>>(a);
  else rec_bwd_kernel<T, false><<<grid, 64, 0, s>>>(a);
  if (a.decay)
    rec_reduce_kernel<<<(unsigned)((a.dim + 63) / 64), 64, 0, s>>>(
        static_cast<const float*>(a.workspace) + a.batch * a.seqlen * a.dim, a.batch, a.dim, a.decay,
        a.ddecay);
  return hipGetLastError();
}

template <typename T>
hipError_t update_t(const ccv1d_rec_update_args& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * ((a.dim + 63) / 64)));
  if (a.decay) rec_update_kernel<T, true><<<grid, 64, 0, s>>>(a);
  else rec_update_kernel<T, false><<<grid, 64, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

size_t rec_workspace(int64_t B, int64_t T, int64_t D, bool backward) {
  return backward ? (size_t)(B * T * D + B * D) * 4 : 0;
}

hipError_t rec_fwd(const ccv1d_rec_args& a, hipStream_t s) {
  switch (a.dtype) {
    case CCV1D_BF16: return fwd_t<__bf16>(a, s);
    case CCV1D_F16: return fwd_t<_Float16>(a, s);
    default: return fwd_t<float>(a, s);
  }
}

hipError_t rec_bwd(const ccv1d_rec_args& a, hipStream_t s) {
  switch (a.dtype) {
    case CCV1D_BF16: return bwd_t<__bf16>(a, s);
    case CCV1D_F16: return bwd_t<_Float16>(a, s);
    default: return bwd_t<float>(a, s);
  }
}

hipError_t rec_update(const ccv1d_rec_update_args& a, hipStream_t s) {
  switch (a.dtype) {
    case CCV1D_BF16: return update_t<__bf16>(a, s);
    case CCV1D_F16: return update_t<_Float16>(a, s);
    default: return update_t<float>(a, s);
  }
}

}  // namespace ops
}  // namespace ccv1d

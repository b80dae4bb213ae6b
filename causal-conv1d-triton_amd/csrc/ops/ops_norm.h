// Norms around a block (ccv1d_layer.h has the formulas), forward and backward.
//
// A row lies in the registers of 16 to 512 lanes, 8 elements a lane and step, so that each tensor is read once and
// written once per direction; its sums go through the wave and, for rows of several waves, LDS. Bound by memory:
// forward at 32768 rows of 4096 in bf16 with all parts 265 us (5.1 TB/s, a copy's rate), at 16384 rows of 2048 with an
// fp32 stream 78 us (5.2 TB/s), backward there 178 (3.5 TB/s; VALUs 40 % busy, rows one after another: a row requested ahead
// 196, three waves a SIMD 206), weights' sums 7.
// Backward, with h1 = x inv1, h2 = r inv2, t2 = w2 dy, inv = 1 / sqrt(mean(.^2) + eps):
//
//   dr += inv2 (t2 - h2 mean(h2 t2)),  dresidual = dr,  dm = s dr,  dn = dm act(gate),  t1 = w1 dn
//   dgate = dm n act'(gate),  dx = inv1 (t1 - h1 mean(h1 t1))
//   dw2 = sum dy h2,  ds = sum dr m,  dw1 = sum dn h1    over all rows
//
// Every row's r is made again from x, the gate and the residual stream, unrounded, as the forward had it. A
// workgroup adds the weights' gradients of its rows in registers and leaves one line of each; a second
// kernel (ccv1d_ops_norm.hip) adds the lines in order.
#pragma once

#include "ops_norm_launch.h"

namespace ccv1d {
namespace ops {

constexpr int kVec = 8;       // elements a lane and step
// log2 e in two parts, and ln 2.
constexpr float kLog2eNorm = 1.44269504088896340736f;
constexpr float kLog2eRest = (float)(1.44269504088896340736 - (double)kLog2eNorm);
constexpr float kLn2Norm = 0.693147180559945309417f;

// Eight elements from an address that is aligned to one.
template <typename T>
struct Vec {
  typedef T type __attribute__((ext_vector_type(kVec)));
};

template <typename T>
struct Held {  // as loaded
  typename Vec<T>::type v;
  __device__ __forceinline__ float operator[](int i) const { return to_f32(v[i]); }
};

// The first n of them (8 and more: all; none: nothing is read), zero for the others. WHOLE: rows are whole
// eights, so that n is 8 or none, and what lies past a row's end is zero throughout without being asked for: at
// 16384 rows of 2048 (both norms, fp32 stream) the backward takes 178 us, with the questions 192.
template <bool WHOLE, typename T>
__device__ __forceinline__ Held<T> load8(const T* p, int n) {
  Held<T> h;
  if constexpr (WHOLE) {
    h.v = typename Vec<T>::type{};
    if (n > 0) __builtin_memcpy(&h.v, p, sizeof h.v);
  } else if (n >= kVec) {
    __builtin_memcpy(&h.v, p, sizeof h.v);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) h.v[i] = i < n ? p[i] : (T)0.0f;
  }
  return h;
}

template <bool WHOLE, typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[kVec], int n) {
  typename Vec<T>::type v;
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = (T)x[i];
  if (WHOLE ? n > 0 : n >= kVec) {
    __builtin_memcpy(p, &v, sizeof v);
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < n) p[i] = v[i];
  }
}

// Eight elements of a weight, whose type is known at run time.
template <bool WHOLE>
__device__ __forceinline__ void load_weight(const void* p, int type, int64_t at, int n, float (&w)[kVec]) {
  auto from = [&](auto* q) {
    const auto h = load8<WHOLE>(q + at, n);
#pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] = h[i];
  };
  if (type == CCV1D_F32) from(static_cast<const float*>(p));
  else if (type == CCV1D_F16) from(static_cast<const _Float16*>(p));
  else from(static_cast<const __bf16*>(p));
}

// act(z) and act'(z). The hardware's exp2 and reciprocal, 1 ulp each; exp(-z) past fp32's range is infinity, and the
// sigmoid zero. What the rounding of -z log2 e leaves, up to 2^-18 for z = -80, comes as a factor 1 + rest ln 2; where
// that product is beyond fp32's exponents, infinite or NaN, there is none.
__device__ __forceinline__ float sigmoid_of(float z) {
  const float t = -kLog2eNorm * z;
  const float rest = fmaf(-kLog2eRest, z, fmaf(-kLog2eNorm, z, -t));
  return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(t), fabsf(t) < 256.0f ? fmaf(rest, kLn2Norm, 1.0f) : 1.0f, 1.0f));
}
__device__ __forceinline__ float act_of(float z, int act) {
  if (act == CCV1D_NORM_IDENTITY) return z;
  const float s = sigmoid_of(z);
  return act == CCV1D_NORM_SIGMOID ? s : z * s;
}
__device__ __forceinline__ float slope_of(float z, int act) {
  if (act == CCV1D_NORM_IDENTITY) return 1.0f;
  const float s = sigmoid_of(z), rest = sigmoid_of(-z);
  return act == CCV1D_NORM_SIGMOID ? s * rest : s * fmaf(z, rest, 1.0f);
}

// The sums of N numbers over the LANES lanes of a row. Rows of several waves meet in LDS, in two places in
// turn (`turn` counts the calls), so that one barrier a sum is enough.
template <int LANES, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], float (&lds)[2][8][N], int turn) {
  constexpr int IN_WAVE = LANES < 64 ? LANES : 64;
#pragma unroll
  for (int d = 1; d < IN_WAVE; d *= 2)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor(x[i], d);
  if constexpr (LANES > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) lds[turn & 1][w][i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = 0.0f;
#pragma unroll
      for (int n = 0; n < LANES / 64; ++n) x[i] += lds[turn & 1][n][i];
    }
  }
}

__device__ __forceinline__ float inverse(float sum, float by_dim, float eps) {
  return 1.0f / sqrtf(fmaf(sum, by_dim, eps));
}

template <int LANES>
constexpr int kThreads = LANES < 256 ? 256 : LANES;

// Where a lane's elements lie: row, step i at column(i).
template <int LANES>
__device__ __forceinline__ int column(int i) {
  return (i * LANES + (threadIdx.x & (LANES - 1))) * kVec;
}

template <typename T, typename R, int LANES, int STEPS, bool WHOLE>
__global__ __launch_bounds__(kThreads<LANES>) void norm_fwd_kernel(NormParams p) {
  const ccv1d_norm_args& a = p.a;
  __shared__ float lds[2][8][1];
  const int64_t row = (int64_t)blockIdx.x * (kThreads<LANES> / LANES) + threadIdx.x / LANES;
  if (row >= p.rows) return;  // all lanes of a row, and of a workgroup where rows have several waves
  const int64_t outer = row / a.inner, inner = row - outer * a.inner;
  const int dim = (int)a.dim;
  const T* xp = static_cast<const T*>(a.x) + outer * a.x_stride_o + inner * a.x_stride_i;
  const T* gp = static_cast<const T*>(a.gate) + outer * a.gate_stride_o + inner * a.gate_stride_i;
  const R* rp = static_cast<const R*>(a.residual) + outer * a.residual_stride_o + inner * a.residual_stride_i;
  Held<T> x[STEPS], z[STEPS];
  Held<R> res[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int d = column<LANES>(i), n = dim - d;
    x[i] = load8<WHOLE>(xp + d, n);
    if (a.gate) z[i] = load8<WHOLE>(gp + d, n);
    if (a.residual) res[i] = load8<WHOLE>(rp + d, n);
  }
  float inv[1] = {1.0f};
  if (a.post_weight) {
    inv[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) inv[0] = fmaf(x[i][e], x[i][e], inv[0]);
    row_sums<LANES, 1>(inv, lds, 0);
    inv[0] = inverse(inv[0], p.by_dim, a.eps);
  }
  float r[STEPS][kVec], sum[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int d = column<LANES>(i), n = dim - d;
    float w[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) r[i][e] = x[i][e] * inv[0];
    if (a.post_weight) {
      load_weight<WHOLE>(a.post_weight, a.post_dtype, d, n, w);
#pragma unroll
      for (int e = 0; e < kVec; ++e) r[i][e] *= w[e];
    }
    if (a.gate)
#pragma unroll
      for (int e = 0; e < kVec; ++e) r[i][e] *= act_of(z[i][e], a.activation);
#pragma unroll
    for (int e = 0; e < kVec; ++e) r[i][e] *= a.scale;
    if (a.scale_weight) {
      load_weight<WHOLE>(a.scale_weight, a.scale_dtype, d, n, w);
#pragma unroll
      for (int e = 0; e < kVec; ++e) r[i][e] *= w[e];
    }
    if (a.residual)
#pragma unroll
      for (int e = 0; e < kVec; ++e) r[i][e] += res[i][e];
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (!WHOLE && e >= n) r[i][e] = 0.0f;  // past the row's end act(0) and an infinite inv make no number
      sum[0] = fmaf(r[i][e], r[i][e], sum[0]);
    }
    if (a.r) store8<WHOLE>(static_cast<R*>(a.r) + row * dim + d, r[i], n);
  }
  if (!a.pre_weight) return;
  row_sums<LANES, 1>(sum, lds, 1);
  const float inv2 = inverse(sum[0], p.by_dim, a.eps);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int d = column<LANES>(i), n = dim - d;
    float w[kVec];
    load_weight<WHOLE>(a.pre_weight, a.pre_dtype, d, n, w);
#pragma unroll
    for (int e = 0; e < kVec; ++e) r[i][e] *= inv2 * w[e];
    store8<WHOLE>(static_cast<T*>(a.y) + row * dim + d, r[i], n);
  }
}

// POST, PRE: whether there is a norm of the block's output, and of the sum; without either there is nothing to do.
template <typename T, typename R, int LANES, int STEPS, bool POST, bool PRE, bool WHOLE>
__global__ __launch_bounds__(kThreads<LANES>) void norm_bwd_kernel(NormParams p) {
  constexpr int AT_ONCE = kThreads<LANES> / LANES;
  const ccv1d_norm_args& a = p.a;
  __shared__ float lds1[2][8][1], lds2[2][8][2];
  __shared__ float parts[LANES < 256 ? 256 * kVec : 1];
  const int dim = (int)a.dim;
  float d1[STEPS][kVec] = {}, d2[STEPS][kVec] = {}, dsc[STEPS][kVec] = {};
  struct Row {
    Held<T> x[STEPS], z[STEPS], dy[STEPS];
    Held<R> res[STEPS], dr[STEPS];
  } now;
  auto load = [&](Row& r, int64_t first) {
    const int64_t row = first + threadIdx.x / LANES;
    const bool in = row < p.rows;
    const int64_t outer = in ? row / a.inner : 0, inner = in ? row - outer * a.inner : 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int d = column<LANES>(i), n = in ? dim - d : 0;
      r.x[i] = load8<WHOLE>(static_cast<const T*>(a.x) + outer * a.x_stride_o + inner * a.x_stride_i + d, n);
      if (a.gate) r.z[i] = load8<WHOLE>(static_cast<const T*>(a.gate) + outer * a.gate_stride_o + inner * a.gate_stride_i + d, n);
      if (PRE && a.residual)
        r.res[i] =
            load8<WHOLE>(static_cast<const R*>(a.residual) + outer * a.residual_stride_o + inner * a.residual_stride_i + d, n);
      if (a.dr) r.dr[i] = load8<WHOLE>(static_cast<const R*>(a.dr) + outer * a.dr_stride_o + inner * a.dr_stride_i + d, n);
      if (PRE && a.dy) r.dy[i] = load8<WHOLE>(static_cast<const T*>(a.dy) + outer * a.dy_stride_o + inner * a.dy_stride_i + d, n);
    }
  };
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * AT_ONCE; first < p.rows; first += (int64_t)gridDim.x * AT_ONCE, ++turn) {
    const int64_t row = first + threadIdx.x / LANES;
    // The weights stay in registers from row to row, but of two steps a lane are read again for each row: 48
    // registers, which would spill.
    int shift = 0;
    if constexpr (STEPS > 1) asm volatile("" : "+v"(shift));
    const bool in = row < p.rows;  // of all lanes of a row
    load(now, first);
    const Held<T>(&x)[STEPS] = now.x, (&z)[STEPS] = now.z, (&dy)[STEPS] = now.dy;
    const Held<R>(&res)[STEPS] = now.res, (&dr)[STEPS] = now.dr;
    float inv1 = 1.0f;
    if constexpr (POST) {
      float s[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) s[0] = fmaf(x[i][e], x[i][e], s[0]);
      row_sums<LANES, 1>(s, lds1, 2 * turn);
      inv1 = in ? inverse(s[0], p.by_dim, a.eps) : 0.0f;  // of no row, with eps 0, it would be infinite
    }
    // dr of all, in fp32, and m where a gradient needs it again
    float g[STEPS][kVec];
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) g[i][e] = a.dr ? dr[i][e] : 0.0f;
    auto block_output = [&](int i, float (&m)[kVec]) {  // m
      const int d = column<LANES>(i) + shift, n = dim - d;
      float w[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) m[e] = x[i][e] * inv1;
      if constexpr (POST) {
        load_weight<WHOLE>(a.post_weight, a.post_dtype, d, n, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) m[e] *= w[e];
      }
      if (a.gate)
#pragma unroll
        for (int e = 0; e < kVec; ++e) m[e] *= act_of(z[i][e], a.activation);
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (!WHOLE && (e >= n || !in)) m[e] = 0.0f;
    };
    auto scales = [&](int i, float (&w)[kVec]) {
      const int d = column<LANES>(i) + shift;
      if (a.scale_weight) load_weight<WHOLE>(a.scale_weight, a.scale_dtype, d, dim - d, w);
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = a.scale_weight ? w[e] * a.scale : a.scale;
    };
    if (PRE && a.dy) {
      float r[STEPS][kVec], s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int d = column<LANES>(i) + shift, n = dim - d;
        float sc[kVec], w[kVec];
        block_output(i, r[i]);
        scales(i, sc);
        load_weight<WHOLE>(a.pre_weight, a.pre_dtype, d, n, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          r[i][e] *= sc[e];
          if (a.residual) r[i][e] += res[i][e];
          if (!WHOLE && (e >= n || !in)) r[i][e] = 0.0f;
          s[0] = fmaf(r[i][e], r[i][e], s[0]);
          s[1] = fmaf(r[i][e], w[e] * dy[i][e], s[1]);
        }
      }
      row_sums<LANES, 2>(s, lds2, turn);
      const float inv2 = in ? inverse(s[0], p.by_dim, a.eps) : 0.0f, mean = s[1] * p.by_dim * inv2;  // of h2 t2
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int d = column<LANES>(i) + shift, n = dim - d;
        float w[kVec];
        load_weight<WHOLE>(a.pre_weight, a.pre_dtype, d, n, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float h = WHOLE || (in && e < n) ? r[i][e] * inv2 : 0.0f;
          d2[i][e] = fmaf(dy[i][e], h, d2[i][e]);
          g[i][e] = fmaf(inv2, w[e] * dy[i][e] - h * mean, g[i][e]);
        }
      }
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int d = column<LANES>(i) + shift, n = in ? dim - d : 0;
      if (a.dresidual) store8<WHOLE>(static_cast<R*>(a.dresidual) + row * dim + d, g[i], n);
      float sc[kVec];
      if (a.scale_weight) {
        float m[kVec];
        block_output(i, m);
#pragma unroll
        for (int e = 0; e < kVec; ++e) dsc[i][e] = fmaf(g[i][e] * a.scale, m[e], dsc[i][e]);
      }
      scales(i, sc);
#pragma unroll
      for (int e = 0; e < kVec; ++e) g[i][e] = WHOLE || n > e ? g[i][e] * sc[e] : 0.0f;  // dm
      float w[kVec];
      if constexpr (POST) load_weight<WHOLE>(a.post_weight, a.post_dtype, d, dim - d, w);
      if (a.gate) {
        float dz[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float nn = POST ? x[i][e] * inv1 * w[e] : x[i][e];
          dz[e] = g[i][e] * nn * slope_of(z[i][e], a.activation);
          g[i][e] = WHOLE || n > e ? g[i][e] * act_of(z[i][e], a.activation) : 0.0f;  // dn
        }
        store8<WHOLE>(static_cast<T*>(a.dgate) + row * dim + d, dz, n);
      }
      if constexpr (POST) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float h = WHOLE || n > e ? x[i][e] * inv1 : 0.0f;
          d1[i][e] = fmaf(g[i][e], h, d1[i][e]);
          g[i][e] = WHOLE || n > e ? g[i][e] * w[e] : 0.0f;  // t1
          s[0] = fmaf(g[i][e], h, s[0]);
        }
      }
    }
    if constexpr (POST) row_sums<LANES, 1>(s, lds1, 2 * turn + 1);
    const float mean = s[0] * p.by_dim;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int d = column<LANES>(i) + shift, n = in ? dim - d : 0;
      if constexpr (POST)
#pragma unroll
        for (int e = 0; e < kVec; ++e) g[i][e] = inv1 * (g[i][e] - x[i][e] * inv1 * mean);
      store8<WHOLE>(static_cast<T*>(a.dx) + row * dim + d, g[i], n);
    }
  }
  // The workgroup's lines: the rows at once of a narrow row are added in order.
  auto leave = [&](int which, float (&v)[STEPS][kVec]) {
    float* line = p.lines + ((int64_t)blockIdx.x * 3 + which) * dim;
    if constexpr (LANES < 256) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < STEPS; ++i)  // STEPS is 1
#pragma unroll
        for (int e = 0; e < kVec; ++e) parts[threadIdx.x * kVec + e] = v[i][e];
      __syncthreads();
      for (int d = threadIdx.x; d < dim; d += 256) {
        float s = 0.0f;
        for (int n = 0; n < AT_ONCE; ++n) s += parts[n * LANES * kVec + d];
        line[d] = s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int d = column<LANES>(i);
        store8<WHOLE>(line + d, v[i], dim - d);
      }
    }
  };
  if constexpr (POST) leave(0, d1);
  if (a.scale_weight) leave(1, dsc);
  if constexpr (PRE) leave(2, d2);
}

template <typename T, typename R, int LANES, int STEPS, bool WHOLE>
hipError_t norm_launch(const NormParams& p, bool backward, hipStream_t s) {
  constexpr int AT_ONCE = kThreads<LANES> / LANES;
  if (!backward)
    return start(&norm_fwd_kernel<T, R, LANES, STEPS, WHOLE>, (p.rows + AT_ONCE - 1) / AT_ONCE, kThreads<LANES>, s, p);
  auto* kernel = !p.a.pre_weight    ? &norm_bwd_kernel<T, R, LANES, STEPS, true, false, WHOLE>
                 : !p.a.post_weight ? &norm_bwd_kernel<T, R, LANES, STEPS, false, true, WHOLE>
                                    : &norm_bwd_kernel<T, R, LANES, STEPS, true, true, WHOLE>;
  return start(kernel, norm_lines(p.a), kThreads<LANES>, s, p);
}

template <typename T, typename R, int LANES, int STEPS>
hipError_t norm_size(const NormParams& p, bool backward, hipStream_t s) {
  return p.a.dim % kVec == 0 ? norm_launch<T, R, LANES, STEPS, true>(p, backward, s)
                             : norm_launch<T, R, LANES, STEPS, false>(p, backward, s);
}

template <typename T, typename R>
hipError_t norm_types(const NormParams& p, bool backward, hipStream_t s) {
  const int64_t d = p.a.dim;
  if (d <= 16 * kVec) return norm_size<T, R, 16, 1>(p, backward, s);
  if (d <= 64 * kVec) return norm_size<T, R, 64, 1>(p, backward, s);
  if (d <= 256 * kVec) return norm_size<T, R, 256, 1>(p, backward, s);
  if (d <= 512 * kVec) return norm_size<T, R, 512, 1>(p, backward, s);
  return norm_size<T, R, 512, 2>(p, backward, s);
}

}  // namespace ops
}  // namespace ccv1d

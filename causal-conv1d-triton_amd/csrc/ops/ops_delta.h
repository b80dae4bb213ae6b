// Kernels of the gated delta rule over whole sequences (ccv1d_layer.h has the recurrence).
//
// A chunk is 64 rows. With G_i the running sum of the log-decays from the chunk's start, D_ij = exp(G_i - G_j)
// for j <= i (zero between rows of different sequences), S0 the state in front of the chunk and S1 behind it:
//
//   A_ij = beta_i D_ij k_i.k_j (j < i),   T = (I + A)^-1,   P_ij = scale D_ij q_i.k_j (j <= i)
//   R = beta (V - e^G K S0),   U = T R,   O = scale e^G Q S0 + P U,   S1 = e^G_C S0 + K^T (e^(G_C - G) U)
//
// and backwards, given dO and dS1:
//
//   dU = P^T dO + e^(G_C - G) K dS1,   dR = T^T dU,   dV = beta dR
//   dS0 = e^G_C dS1 + scale Q^T (e^G dO) - K^T (beta e^G dR)
//   z_i = e^G_i S0 dR_i + sum_{j<i} D_ij (dR_i.U_j) k_j,   dq_i = scale (e^G_i S0 dO_i + sum_{j<=i} D_ij (dO_i.U_j) k_j)
//   c_j = e^(G_C - G_j) dS1 U_j + sum_{i>=j} scale D_ij (dO_i.U_j) q_i - sum_{i>j} beta_i D_ij (dR_i.U_j) k_i
//   dk_i = c_i - beta_i z_i,   dbeta_i = dR_i.V_i - k_i.z_i
//   dG_i = q_i.dq_i - beta_i k_i.z_i - k_i.c_i,   dG_C += sum_j k_j.(first part of c_j) + e^G_C <dS1, S0>
//   dg_t = sum_{i >= t, the same sequence} dG_i
//
// What needs no state (T, P, the operands' layouts) is made for all chunks at once (delta_prep_kernel), the
// chain of states runs over the chunks, 16 value columns a workgroup (delta_fwd_kernel, delta_bwd_kernel), and
// the gradients that need no chain are again made for all chunks at once (delta_grad_kernel).
//
// Products run on the bf16 matrix cores (16x16x32), fp32 operands as sums of bf16 pieces: cut after 8 bits each, three
// pieces are the fp32 number itself, and the products of pieces i + j <= 2 leave out 2^-22 of the largest term.
// bf16 inputs are one piece, fp16 inputs two (11 bits), fp32 three. Nothing that reaches a state or a gradient is
// rounded to fewer than fp32's bits; what reaches an output in 16 bits alone (P and U in P U, S0 in Q S0) keeps
// two pieces, 2^-15 or better. By the rates of the instructions (16x16x32 in 16 bits 16 cycles, 16x16x4 in fp32
// 32) three pieces against a bf16 input take 3/16 of fp32's time, against three pieces 6/16.
//
// Layout: "fragment" is the operand of one such instruction, 16 rows (A) or columns (B) by 32 of the summed index,
// 8 elements for each of 64 lanes: lane l has row l % 16 and, of the sum, 4 (l / 16) + 0..3 and 16 + 4 (l / 16) + 0..3.
// The order of a sum is free as long as both operands have the same, and by this one a product's result (lane l has
// column l % 16, rows 4 (l / 16) + 0..3) is half of the B fragment of the next product in the lane that holds it. So
// states, X, R, U and their gradients go from product to product without changing lanes, and what other
// waves need of them passes LDS in 8-byte pieces at the same lane.
#pragma once

#include "ops_delta_launch.h"

namespace ccv1d {
namespace ops {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int kC = CCV1D_DELTA_CHUNK;
constexpr double kLog2eDouble = 1.4426950408889634074;

template <typename T>
constexpr int kPieces = std::is_same_v<T, __bf16> ? 1 : std::is_same_v<T, _Float16> ? 2 : 3;
// Pieces and limit of what reaches an output of type T alone.
template <typename T>
constexpr int kOutPieces = sizeof(T) == 4 ? 3 : 2;

// A barrier for LDS alone: loads from memory that are on their way stay on it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The upper halves of two words: two fp32 numbers cut to bf16.
__device__ __forceinline__ uint32_t cut_pair(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float cut(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  const uint32_t lo = __builtin_bit_cast(uint16_t, (__bf16)a), hi = __builtin_bit_cast(uint16_t, (__bf16)b);
  return lo | hi << 16;
}

// Two numbers as N words of bf16 pieces.
template <int N>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&o)[N]) {
  if constexpr (N == 1) {
    o[0] = round_pair(a, b);
  } else {
    o[0] = cut_pair(a, b);
    a -= cut(a), b -= cut(b);
    if constexpr (N == 2) {
      o[1] = round_pair(a, b);
    } else {
      o[1] = cut_pair(a, b);
      o[2] = cut_pair(a - cut(a), b - cut(b));
    }
  }
}

template <int N>
__device__ __forceinline__ void split8(f4 x, f4 y, u4 (&o)[N]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t w[N];
    const f4 v = p < 2 ? x : y;
    split2<N>(v[2 * (p & 1)], v[2 * (p & 1) + 1], w);
#pragma unroll
    for (int n = 0; n < N; ++n) o[n][p] = w[n];
  }
}

// Half a fragment.
template <int N>
__device__ __forceinline__ void split4(f4 x, u2 (&o)[N]) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    uint32_t w[N];
    split2<N>(x[2 * p], x[2 * p + 1], w);
#pragma unroll
    for (int n = 0; n < N; ++n) o[n][p] = w[n];
  }
}

__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// c + a b over the pieces i + j <= LIM, small terms first.
template <int LIM, int NA, int NB>
__device__ __forceinline__ f4 mac(const u4 (&a)[NA], const u4 (&b)[NB], f4 c) {
#pragma unroll
  for (int sum = LIM; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = sum - i;
      if (j >= 0 && j < NB) c = mfma(a[i], b[j], c);
    }
  return c;
}

template <int N>
__device__ __forceinline__ void load_frag(const u4* p, u4 (&o)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) o[n] = p[n * 64];
}

// Writes the half `half` of a fragment whose pieces lie 64 units apart; p is the lane's unit.
template <int N>
__device__ __forceinline__ void store_half(u4* p, int half, const u2 (&v)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) reinterpret_cast<u2*>(p + n * 64)[half] = v[n];
}

// Four elements from an address that is aligned to one.
template <typename T>
__device__ __forceinline__ f4 load4(const T* p) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 v;
  __builtin_memcpy(&v, p, sizeof v);
  return f4{to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3])};
}

template <typename T>
__device__ __forceinline__ f4 load4(const T* p, int64_t n) {  // the first n of them, zero for the others
  if (n >= 4) return load4(p);
  f4 r = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) r[i] = to_f32(p[i]);
  return r;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f4 v, int64_t n) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  if (n >= 4) {
    const v4 w = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    __builtin_memcpy(p, &w, sizeof w);
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = (T)v[i];
}

// An element of a tensor whose type is known at run time.
__device__ __forceinline__ float load_as(const void* p, int64_t at, int dtype) {
  if (dtype == CCV1D_F32) return static_cast<const float*>(p)[at];
  if (dtype == CCV1D_F16) return (float)static_cast<const _Float16*>(p)[at];
  return (float)static_cast<const __bf16*>(p)[at];
}
__device__ __forceinline__ void store_as(void* p, int64_t at, int dtype, float v) {
  if (dtype == CCV1D_F32) static_cast<float*>(p)[at] = v;
  else if (dtype == CCV1D_F16) static_cast<_Float16*>(p)[at] = (_Float16)v;
  else static_cast<__bf16*>(p)[at] = (__bf16)v;
}

// A fragment's eight elements of a row of T at `p` (its first four) and `p + 16`.
template <typename T>
__device__ __forceinline__ void frag_of(const T* p, u4 (&o)[kPieces<T>]) {
  if constexpr (kPieces<T> == 1) {
    const u2 a = *reinterpret_cast<const u2*>(p), b = *reinterpret_cast<const u2*>(p + 16);
    o[0] = u4{a[0], a[1], b[0], b[1]};
  } else {
    split8<kPieces<T>>(load4(p), load4(p + 16), o);
  }
}

// Element e of a fragment, from its pieces.
template <int N>
__device__ __forceinline__ float piece_sum(const u4 (&f)[N], int e) {
  float s = 0.0f;
#pragma unroll
  for (int n = N - 1; n >= 0; --n) {
    const uint32_t w = f[n][e >> 1];
    s += __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  }
  return s;
}

// The triangle of 16x16 tiles, in fragments of two tiles of the sum: lower has row tiles m with the sum's
// pairs s <= m / 2, upper row tiles n with s >= n / 2; six fragments each.
__device__ __forceinline__ int lower_frag(int m, int s) { return m < 2 ? m : 2 * m - 2 + s; }
__device__ __forceinline__ int upper_frag(int n, int s) { return n < 2 ? 2 * n + s : n + 2; }
constexpr int kTri = 6;

// What a chunk's rows have, per head: [0] e^G where the carried state reaches the row, [1] e^(G_C - G) where the
// row reaches the chunk's end, [2] beta, [3] one for a row that is there and no padding, [4][0] e^G_C where
// the carried state reaches the end; zero elsewhere.
constexpr int kRowFields = 5;

struct ChunkRows {
  double sum;   // G log2 e, from the row's sequence's start in the chunk
  int run;      // resets in the chunk up to the row
  bool live, reset;
  float beta;
};

// Row `lane` of chunk c. A row that starts a sequence, padding, and a decay that is zero in fp32 reset the state: its
// log-decay, which multiplies nothing, counts as zero, so that no sequence's sums meet another's.
__device__ __forceinline__ ChunkRows chunk_row(const ccv1d_delta_args& a, int64_t b, int64_t c, int64_t h, int lane) {
  ChunkRows r;
  const int64_t t = c * kC + lane;
  const bool in = t < a.seqlen;
  r.live = in, r.reset = false;
  if (a.seq_idx && in) {
    const int64_t at = b * a.seqlen + t;
    int64_t id, before;
    if (a.seq_idx_64) {
      const int64_t* s = static_cast<const int64_t*>(a.seq_idx);
      id = s[at], before = t ? s[at - 1] : id;
    } else {
      const int32_t* s = static_cast<const int32_t*>(a.seq_idx);
      id = s[at], before = t ? s[at - 1] : id;
    }
    r.live = id >= 0;
    r.reset = id < 0 || id != before;
  }
  float g = 0.0f;
  r.beta = 0.0f;
  if (r.live) {
    g = load_as(a.log_decay, b * a.log_decay_stride_b + t * a.log_decay_stride_t + h * a.log_decay_stride_h,
                a.log_decay_dtype);
    r.beta = load_as(a.beta, b * a.beta_stride_b + t * a.beta_stride_t + h * a.beta_stride_h, a.beta_dtype);
  }
  if (g < -104.0f) r.reset = true;
  const uint64_t resets = __ballot(r.reset);
  r.run = __popcll(resets & (~uint64_t(0) >> (63 - lane)));
  double s = r.reset ? 0.0 : (double)g * kLog2eDouble;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_up(s, d);
    const int run = __shfl_up(r.run, d);
    if (lane >= d && run == r.run) s += o;
  }
  r.sum = s;
  return r;
}

__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f((float)x); }

struct ChunkShared {
  double sum[kC];
  int run[kC];
  float beta[kC];
  int live[kC];
};

// A wave makes a chunk's rows and leaves them in LDS and, in the workspace, what the chain needs of them.
__device__ __forceinline__ ChunkRows share_rows(const ccv1d_delta_args& a, int64_t b, int64_t c, int64_t h, int lane,
                                                ChunkShared& sh, float* rows) {
  const ChunkRows r = chunk_row(a, b, c, h, lane);
  sh.sum[lane] = r.sum, sh.run[lane] = r.run, sh.beta[lane] = r.beta, sh.live[lane] = r.live;
  if (rows) {
    const double end = __shfl(r.sum, 63);
    const int last = __shfl(r.run, 63);
    rows[lane] = r.live && r.run == 0 ? exp2_of(r.sum) : 0.0f;
    rows[kC + lane] = r.live && r.run == last ? exp2_of(end - r.sum) : 0.0f;
    rows[2 * kC + lane] = r.beta;
    rows[3 * kC + lane] = r.live ? 1.0f : 0.0f;
    rows[4 * kC + lane] = lane == 0 && last == 0 ? exp2_of(end) : 0.0f;
  }
  return r;
}

// A chunk's rows of q or k into LDS, zero where there is none, past the last element, and in padding.
template <typename T, int DK, int LD, int THREADS>
__device__ __forceinline__ void load_rows(T* to, const T* from, int64_t stride_t, int64_t dk, int64_t t0, int64_t seqlen,
                                          const int* live) {
  typedef T v4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < kC * DK / 4 / THREADS; ++i) {
    const int u = i * THREADS + threadIdx.x, row = u / (DK / 4), d = u % (DK / 4) * 4;
    v4 v = {};
    if (t0 + row < seqlen && live[row]) {
      const T* p = from + (t0 + row) * stride_t + d;
      if (d + 4 <= dk) {
        __builtin_memcpy(&v, p, sizeof v);
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (d + e < dk) v[e] = p[e];
      }
    }
    *reinterpret_cast<v4*>(to + row * LD + d) = v;
  }
}

// All chunks: the operands of the chains as fragments, T and P (forward) or their transposes (backward).
// Bound by memory: reads q and k, writes them three (four) times as fragments and 30 KiB a head's chunk.
template <typename T, int DK, bool BWD>
__global__ __launch_bounds__(256) void delta_prep_kernel(DeltaParams p) {
  constexpr int NI = kPieces<T>, KS = DK / 32, LD = DK + 16 / sizeof(T), LA = 68;
  constexpr int NP = BWD ? 3 : kOutPieces<T>;
  __shared__ T kl[kC * LD], ql[kC * LD];
  __shared__ float al[kC * LA], td[4 * 16 * 20];
  __shared__ ChunkShared sh;
  const ccv1d_delta_args& a = p.a;
  const int lane = threadIdx.x & 63, m = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int64_t kc = blockIdx.x;  // (batch, key head, chunk)
  const int64_t c = kc % p.chunks, bk = kc / p.chunks, b = bk / a.key_heads, kh = bk - b * a.key_heads;
  const int64_t t0 = c * kC;
  if (m == 0) share_rows(a, b, c, kh * p.group, lane, sh, nullptr);
  lds_barrier();
  load_rows<T, DK, LD, 256>(kl, static_cast<const T*>(a.k) + b * a.k_stride_b + kh * a.k_stride_h, a.k_stride_t,
                            a.key_dim, t0, a.seqlen, sh.live);
  load_rows<T, DK, LD, 256>(ql, static_cast<const T*>(a.q) + b * a.q_stride_b + kh * a.q_stride_h, a.q_stride_t,
                            a.key_dim, t0, a.seqlen, sh.live);
  lds_barrier();

  // Tiles (n, m) of k.k and q.k, n <= m: keys j of tile n as rows and i of tile m as columns, backward the other
  // way round, so that a lane's results are halves of P's (P^T's) fragments.
  f4 kk[4] = {}, qk[4] = {};
  u4* kf = p.kf + kc * (4 * KS * NI * 64);
  u4* qf = p.qf + kc * (4 * KS * NI * 64);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    u4 km[NI], qm[NI];
    frag_of(kl + (16 * m + col) * LD + 32 * s + 4 * g, km);
    frag_of(ql + (16 * m + col) * LD + 32 * s + 4 * g, qm);
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      kf[((m * KS + s) * NI + n) * 64 + lane] = km[n];
      qf[((m * KS + s) * NI + n) * 64 + lane] = qm[n];
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n <= m) {
        u4 kn[NI];
        frag_of(kl + (16 * n + col) * LD + 32 * s + 4 * g, kn);
        kk[n] = BWD ? mac<2>(km, kn, kk[n]) : mac<2>(kn, km, kk[n]);
        qk[n] = BWD ? mac<2>(qm, kn, qk[n]) : mac<2>(kn, qm, qk[n]);
      }
  }
  // Transposed: a lane has one element of 8 rows.
#pragma unroll
  for (int i = 0; i < DK / 16 / 4; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int t = m + 4 * i;
      auto column = [&](const T* from, u4* to) {
        u4 f[NI];
        f4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = to_f32(from[(32 * s + 4 * g + e) * LD + 16 * t + col]);
          y[e] = to_f32(from[(32 * s + 16 + 4 * g + e) * LD + 16 * t + col]);
        }
        split8<NI>(x, y, f);
#pragma unroll
        for (int n = 0; n < NI; ++n) to[((t * 2 + s) * NI + n) * 64 + lane] = f[n];
      };
      column(kl, p.kt + kc * (DK / 16 * 2 * NI * 64));
      if constexpr (BWD) column(ql, p.qt + kc * (DK / 16 * 2 * NI * 64));
    }

  for (int64_t h = kh * p.group; h < (kh + 1) * p.group; ++h) {
    const int64_t hc = (b * a.heads + h) * p.chunks + c;
    u4* tf = p.tf + hc * (kTri * 3 * 64);
    u4* pf = p.pf + hc * (kTri * NP * 64);
    lds_barrier();
    if (m == 0) share_rows(a, b, c, h, lane, sh, p.rows + hc * (kRowFields * kC));
    lds_barrier();
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n > m + 1) continue;
      // tile (n, m): of the lane's four results, i and j
      f4 pv = {0, 0, 0, 0};
      if (n <= m) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 16 * m + (BWD ? 4 * g + e : col), j = 16 * n + (BWD ? col : 4 * g + e);
          const bool seen = j <= i && sh.run[i] == sh.run[j];
          const float d = seen ? exp2_of(sh.sum[i] - sh.sum[j]) : 0.0f;
          al[i * LA + j] = seen && j < i ? sh.beta[i] * d * kk[n][e] : 0.0f;
          pv[e] = seen ? a.scale * d * qk[n][e] : 0.0f;
        }
      } else if (m & 1) {
        continue;  // no half of a fragment that is read
      }
      u2 w[NP];
      split4<NP>(pv, w);
      if constexpr (BWD) {
        // rows j of tile n, sum over i of tile m; the tile m of a pair in front of n's is zero
        store_half<NP>(pf + upper_frag(n, m / 2) * (NP * 64) + lane, m & 1, w);
      } else {
        store_half<NP>(pf + lower_frag(m, n / 2) * (NP * 64) + lane, n & 1, w);
      }
    }
    lds_barrier();
    // T's tiles on the diagonal, a column a lane, by substitution.
    if (m == 0) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == col ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = fmaf(-al[(16 * g + i) * LA + 16 * g + j], x[j], s);
        x[i] = s;
        td[(g * 16 + i) * 20 + col] = s;
      }
    }
    lds_barrier();
    // The tiles below: T_im = -T_ii sum_{k=m}^{i-1} A_ik T_km, column of tiles m a wave, in fp32.
    f4 tc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < m) continue;
      if (i == m) {
#pragma unroll
        for (int e = 0; e < 4; ++e) tc[i][e] = td[(i * 16 + 4 * g + e) * 20 + col];
        continue;
      }
      f4 acc = {0, 0, 0, 0}, out = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < i; ++k)
        if (k >= m) {
          const f4 av = *reinterpret_cast<const f4*>(&al[(16 * i + col) * LA + 16 * k + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(av[e], tc[k][e], acc, 0, 0, 0);
        }
      const f4 tv = *reinterpret_cast<const f4*>(&td[(i * 16 + col) * 20 + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) out = __builtin_amdgcn_mfma_f32_16x16x4f32(tv[e], -acc[e], out, 0, 0, 0);
      tc[i] = out;
    }
    if constexpr (BWD) {
      // T^T: rows j of tile m, sum over i: as they are
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < m && !((m & 1) && i == m - 1)) continue;
        u2 w[3];
        split4<3>(i < m ? f4{0, 0, 0, 0} : tc[i], w);
        store_half<3>(tf + upper_frag(m, i / 2) * (3 * 64) + lane, i & 1, w);
      }
    } else {
      lds_barrier();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= m)
#pragma unroll
          for (int e = 0; e < 4; ++e) al[(16 * i + 4 * g + e) * LA + 16 * m + col] = tc[i][e];
      lds_barrier();
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m / 2) {
          const f4 x = *reinterpret_cast<const f4*>(&al[(16 * m + col) * LA + 32 * s + 4 * g]);
          f4 y = {0, 0, 0, 0};
          if (2 * s + 1 <= m) y = *reinterpret_cast<const f4*>(&al[(16 * m + col) * LA + 32 * s + 16 + 4 * g]);
          u4 f[3];
          split8<3>(x, y, f);
#pragma unroll
          for (int n = 0; n < 3; ++n) tf[(lower_frag(m, s) * 3 + n) * 64 + lane] = f[n];
        }
    }
  }
}

// Which head and which 16 value columns a workgroup of a chain has: workgroups go to the XCDs in turn, and all
// columns of a head to one, whose L2 then holds the head's fragments once.
struct ChainPlace {
  int64_t head;  // batch * heads + head
  int64_t dv0;
  bool any;
};
__device__ __forceinline__ ChainPlace chain_place(const DeltaParams& p) {
  const int64_t xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  ChainPlace r;
  r.head = xcd + 8 * (slot / p.tiles);
  r.dv0 = slot % p.tiles * 16;
  r.any = r.head < p.a.batch * p.a.heads;
  return r;
}

// Waves of a chain: 32 of the keys' elements each, 64 for the largest heads, whose operands need the registers.
template <int DK>
constexpr int kChainWaves = DK / 32 < 4 ? DK / 32 : 4;

// Whether a chain requests the next chunk's operands of k and q while it works on this one's: not for the largest
// heads in fp32, whose operands alone are 300 registers.
template <typename T, int DK>
constexpr bool kLoadAhead = !(sizeof(T) == 4 && DK == 256);

// The tiles of 16 rows that a wave has of the products between rows: four over the waves.
template <int NW>
struct RowTiles {
  static constexpr int kN = 4 / NW;
  static __device__ __forceinline__ int at(int wave, int q) { return NW == 2 && q ? 3 - wave : wave; }
};

// The chain of states forward. A workgroup has 16 value columns of a head, a wave 32 or 64 of the keys'
// elements of their states (in the accumulators' layout), and 16 or 32 of a chunk's rows.
// Bound by latency: three products after one another a chunk, each behind a barrier.
template <typename T, int DK, bool SAVE>
__global__ __launch_bounds__(kChainWaves<DK> * 64) void delta_fwd_kernel(DeltaParams p) {
  constexpr int NI = kPieces<T>, KS = DK / 32, NW = kChainWaves<DK>, KB = KS / NW, MT = RowTiles<NW>::kN;
  constexpr int NO = kOutPieces<T>, LO = NO - 1;
  constexpr bool AHEAD = kLoadAhead<T, DK>;
  __shared__ f4 red[2][NW][4][64];
  __shared__ u4 rb[2][3][64], ub[2][3][64], uo[2][NO][64];
  const ccv1d_delta_args& a = p.a;
  const ChainPlace at = chain_place(p);
  if (!at.any) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int64_t b = at.head / a.heads, h = at.head - b * a.heads, kh = h / p.group;
  const int64_t dv = at.dv0 + col;
  const bool column = dv < a.value_dim;
  const int64_t N = p.chunks, kc0 = (b * a.key_heads + kh) * N, hc0 = at.head * N;

  u4 kf[KB][4][NI], qf[KB][4][NI], kt[2 * KB][2][NI], tf[MT][2][3], pf[MT][2][NO];
  float v[MT][4];
  f4 into[MT], rest[MT], beta[MT], live[MT];
  float whole = 0.0f;
  auto load_kq = [&](int64_t c) {
#pragma unroll
    for (int i = 0; i < KB; ++i)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int64_t o = (kc0 + c) * (4 * KS * NI * 64) + (m * KS + w * KB + i) * (NI * 64) + lane;
        load_frag(p.kf + o, kf[i][m]);
        load_frag(p.qf + o, qf[i][m]);
      }
  };
  auto load_kt = [&](int64_t c) {
    whole = p.rows[(hc0 + c) * (kRowFields * kC) + 4 * kC];
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        load_frag(p.kt + (kc0 + c) * (DK / 16 * 2 * NI * 64) + ((2 * KB * w + t) * 2 + s) * (NI * 64) + lane, kt[t][s]);
  };
  auto load_rows_of = [&](int64_t c) {  // of the wave's row tiles, T and V
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      const float* rows = p.rows + (hc0 + c) * (kRowFields * kC) + 16 * m + 4 * g;
      into[q] = *reinterpret_cast<const f4*>(rows);
      rest[q] = *reinterpret_cast<const f4*>(rows + kC);
      beta[q] = *reinterpret_cast<const f4*>(rows + 2 * kC);
      live[q] = *reinterpret_cast<const f4*>(rows + 3 * kC);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m / 2) load_frag(p.tf + (hc0 + c) * (kTri * 3 * 64) + lower_frag(m, s) * (3 * 64) + lane, tf[q][s]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = c * kC + 16 * m + 4 * g + e;
        v[q][e] = column && t < a.seqlen
                      ? to_f32(static_cast<const T*>(a.v)[b * a.v_stride_b + t * a.v_stride_t + h * a.v_stride_h + dv])
                      : 0.0f;
      }
    }
  };
  auto load_p = [&](int64_t c) {
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m / 2) load_frag(p.pf + (hc0 + c) * (kTri * NO * 64) + lower_frag(m, s) * (NO * 64) + lane, pf[q][s]);
    }
  };

  f4 state[2 * KB];
#pragma unroll
  for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t d = 32 * KB * w + 16 * t + 4 * g + e;
      state[t][e] = a.initial_states && column && d < a.key_dim
                        ? a.initial_states[(at.head * a.key_dim + d) * a.value_dim + dv]
                        : 0.0f;
    }
  if constexpr (AHEAD) {
    load_kq(0);
    load_kt(0);
  }
  load_rows_of(0);
  load_p(0);
  for (int64_t c = 0; c < N; ++c) {
    const int64_t next = c + 1 < N ? c + 1 : c;
    if constexpr (SAVE) {
      float* to = p.s0 + (hc0 + c) * ((int64_t)DK * p.dvp) + at.dv0 + col;
#pragma unroll
      for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[(32 * KB * w + 16 * t + 4 * g + e) * p.dvp] = state[t][e];
    }
    {
      if constexpr (!AHEAD) load_kq(c);
      f4 x[4] = {}, y[4] = {};
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        u4 sb[3], so[NO];
        split8<3>(state[2 * i], state[2 * i + 1], sb);
#pragma unroll
        for (int n = 0; n < NO; ++n) so[n] = sb[n];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          x[m] = mac<2>(kf[i][m], sb, x[m]);
          y[m] = mac<LO>(qf[i][m], so, y[m]);
        }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) red[0][w][m][lane] = x[m], red[1][w][m][lane] = y[m];
    }
    if constexpr (AHEAD) load_kq(next);
    lds_barrier();
    f4 o[MT], now_live[MT];
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      f4 x = red[0][0][m][lane], y = red[1][0][m][lane];
#pragma unroll
      for (int n = 1; n < NW; ++n) x += red[0][n][m][lane], y += red[1][n][m][lane];
      f4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool carried = into[q][e] != 0.0f;  // not a product with zero: the state may hold no number
        const float ve = live[q][e] != 0.0f ? v[q][e] : 0.0f;
        r[e] = beta[q][e] * (ve - (carried ? into[q][e] * x[e] : 0.0f));
        o[q][e] = carried ? a.scale * into[q][e] * y[e] : 0.0f;
      }
      u2 half[3];
      split4<3>(r, half);
      store_half<3>(&rb[m / 2][0][lane], m & 1, half);
    }
    lds_barrier();
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      f4 u = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m / 2) {
          u4 r[3];
          load_frag(&rb[s][0][lane], r);
          u = mac<2>(tf[q][s], r, u);
        }
      if constexpr (SAVE) {
        float* to = p.u + (hc0 + c) * (kC * p.dvp) + at.dv0 + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[(16 * m + 4 * g + e) * p.dvp] = u[e];
      }
      u2 half[3], out[NO];
      split4<NO>(u, out);
      store_half<NO>(&uo[m / 2][0][lane], m & 1, out);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = rest[q][e] != 0.0f ? rest[q][e] * u[e] : 0.0f;
      split4<3>(u, half);
      store_half<3>(&ub[m / 2][0][lane], m & 1, half);
      now_live[q] = live[q];
    }
    load_rows_of(next);
    if constexpr (!AHEAD) load_kt(c);
    lds_barrier();
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) state[t][e] = whole != 0.0f ? whole * state[t][e] : 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u4 u[3];
        load_frag(&ub[s][0][lane], u);
        state[t] = mac<2>(kt[t][s], u, state[t]);
      }
    }
    if constexpr (AHEAD) load_kt(next);
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m / 2) {
          u4 u[NO];
          load_frag(&uo[s][0][lane], u);
          o[q] = mac<LO>(pf[q][s], u, o[q]);
        }
      T* out = static_cast<T*>(a.out);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = c * kC + 16 * m + 4 * g + e;
        if (column && t < a.seqlen)
          out[((b * a.seqlen + t) * a.heads + h) * a.value_dim + dv] = (T)(now_live[q][e] != 0.0f ? o[q][e] : 0.0f);
      }
    }
    load_p(next);
  }
  if (a.final_states && column)
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t d = 32 * KB * w + 16 * t + 4 * g + e;
        if (d < a.key_dim) a.final_states[(at.head * a.key_dim + d) * a.value_dim + dv] = state[t][e];
      }
}

// The chain of the states' gradients, from the last chunk to the first; divided like the forward's. Leaves dS1 of
// every chunk and dR, and writes dV.
template <typename T, int DK>
__global__ __launch_bounds__(kChainWaves<DK> * 64) void delta_bwd_kernel(DeltaParams p) {
  constexpr int NI = kPieces<T>, KS = DK / 32, NW = kChainWaves<DK>, KB = KS / NW, MT = RowTiles<NW>::kN;
  constexpr bool AHEAD = kLoadAhead<T, DK>;
  __shared__ f4 red[NW][4][64];
  __shared__ u4 ob[2][NI][64], oq[2][3][64], ub[2][3][64], rb[2][3][64];
  const ccv1d_delta_args& a = p.a;
  const ChainPlace at = chain_place(p);
  if (!at.any) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int64_t b = at.head / a.heads, h = at.head - b * a.heads, kh = h / p.group;
  const int64_t dv = at.dv0 + col;
  const bool column = dv < a.value_dim;
  const int64_t N = p.chunks, kc0 = (b * a.key_heads + kh) * N, hc0 = at.head * N;

  u4 kf[KB][4][NI], kt[2 * KB][2][NI], qt[2 * KB][2][NI], tf[MT][2][3], pf[MT][2][3];
  float dy[MT][4];
  f4 into[MT], rest[MT], beta[MT];
  float whole = 0.0f;
  auto load_k = [&](int64_t c) {
#pragma unroll
    for (int i = 0; i < KB; ++i)
#pragma unroll
      for (int m = 0; m < 4; ++m)
        load_frag(p.kf + (kc0 + c) * (4 * KS * NI * 64) + (m * KS + w * KB + i) * (NI * 64) + lane, kf[i][m]);
  };
  auto load_t = [&](int64_t c) {
    whole = p.rows[(hc0 + c) * (kRowFields * kC) + 4 * kC];
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int64_t o = (kc0 + c) * (DK / 16 * 2 * NI * 64) + ((2 * KB * w + t) * 2 + s) * (NI * 64) + lane;
        load_frag(p.kt + o, kt[t][s]);
        load_frag(p.qt + o, qt[t][s]);
      }
  };
  auto load_dy = [&](int64_t c) {
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      const float* rows = p.rows + (hc0 + c) * (kRowFields * kC) + 16 * m + 4 * g;
      into[q] = *reinterpret_cast<const f4*>(rows);
      const f4 live = *reinterpret_cast<const f4*>(rows + 3 * kC);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = c * kC + 16 * m + 4 * g + e;
        dy[q][e] = column && t < a.seqlen && live[e] != 0.0f
                       ? to_f32(static_cast<const T*>(
                             a.dout)[b * a.dout_stride_b + t * a.dout_stride_t + h * a.dout_stride_h + dv])
                       : 0.0f;
      }
    }
  };
  auto load_p = [&](int64_t c) {
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      rest[q] = *reinterpret_cast<const f4*>(p.rows + (hc0 + c) * (kRowFields * kC) + kC + 16 * m + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= m / 2) load_frag(p.pf + (hc0 + c) * (kTri * 3 * 64) + upper_frag(m, s) * (3 * 64) + lane, pf[q][s]);
    }
  };
  auto load_tri = [&](int64_t c) {
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      beta[q] = *reinterpret_cast<const f4*>(p.rows + (hc0 + c) * (kRowFields * kC) + 2 * kC + 16 * m + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= m / 2) load_frag(p.tf + (hc0 + c) * (kTri * 3 * 64) + upper_frag(m, s) * (3 * 64) + lane, tf[q][s]);
    }
  };

  f4 ds[2 * KB];
#pragma unroll
  for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t d = 32 * KB * w + 16 * t + 4 * g + e;
      ds[t][e] = a.dfinal_states && column && d < a.key_dim
                     ? a.dfinal_states[(at.head * a.key_dim + d) * a.value_dim + dv]
                     : 0.0f;
    }
  if constexpr (AHEAD) {
    load_k(N - 1);
    load_t(N - 1);
  }
  load_dy(N - 1);
  load_p(N - 1);
  load_tri(N - 1);
  for (int64_t c = N - 1; c >= 0; --c) {
    const int64_t next = c ? c - 1 : 0;
    {
      float* to = p.ds + (hc0 + c) * ((int64_t)DK * p.dvp) + at.dv0 + col;
#pragma unroll
      for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[(32 * KB * w + 16 * t + 4 * g + e) * p.dvp] = ds[t][e];
      if constexpr (!AHEAD) load_k(c);
      f4 x[4] = {};
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        u4 sb[3];
        split8<3>(ds[2 * i], ds[2 * i + 1], sb);
#pragma unroll
        for (int m = 0; m < 4; ++m) x[m] = mac<2>(kf[i][m], sb, x[m]);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) red[w][m][lane] = x[m];
    }
    if constexpr (AHEAD) load_k(next);
    f4 now_into[MT];
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      const f4 d = {dy[q][0], dy[q][1], dy[q][2], dy[q][3]};
      f4 s;
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = a.scale * into[q][e] * d[e];
      u2 half[NI], third[3];
      split4<NI>(d, half);
      store_half<NI>(&ob[m / 2][0][lane], m & 1, half);
      split4<3>(s, third);
      store_half<3>(&oq[m / 2][0][lane], m & 1, third);
      now_into[q] = into[q];
    }
    load_dy(next);
    lds_barrier();
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      f4 y = red[0][m][lane];
#pragma unroll
      for (int n = 1; n < NW; ++n) y += red[n][m][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = rest[q][e] != 0.0f ? rest[q][e] * y[e] : 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= m / 2) {
          u4 o[NI];
          load_frag(&ob[s][0][lane], o);
          y = mac<2>(pf[q][s], o, y);
        }
      u2 half[3];
      split4<3>(y, half);
      store_half<3>(&ub[m / 2][0][lane], m & 1, half);
    }
    load_p(next);
    lds_barrier();
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int m = RowTiles<NW>::at(w, q);
      f4 r = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= m / 2) {
          u4 u[3];
          load_frag(&ub[s][0][lane], u);
          r = mac<2>(tf[q][s], u, r);
        }
      float* to = p.dr + (hc0 + c) * (kC * p.dvp) + at.dv0 + col;
      T* out = static_cast<T*>(a.dv);
      u2 half[3];
      f4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = c * kC + 16 * m + 4 * g + e;
        to[(16 * m + 4 * g + e) * p.dvp] = r[e];
        if (column && t < a.seqlen)
          out[((b * a.seqlen + t) * a.heads + h) * a.value_dim + dv] =
              (T)(beta[q][e] != 0.0f ? beta[q][e] * r[e] : 0.0f);
        x[e] = now_into[q][e] != 0.0f ? -beta[q][e] * now_into[q][e] * r[e] : 0.0f;
      }
      split4<3>(x, half);
      store_half<3>(&rb[m / 2][0][lane], m & 1, half);
    }
    load_tri(next);
    if constexpr (!AHEAD) load_t(c);
    lds_barrier();
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) ds[t][e] = whole != 0.0f ? whole * ds[t][e] : 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u4 x[3];
        load_frag(&oq[s][0][lane], x);
        ds[t] = mac<2>(qt[t][s], x, ds[t]);
        load_frag(&rb[s][0][lane], x);
        ds[t] = mac<2>(kt[t][s], x, ds[t]);
      }
    }
    if constexpr (AHEAD) load_t(next);
    lds_barrier();  // ob and oq are written again before the next barrier
  }
  if (a.dinitial_states && column)
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t d = 32 * KB * w + 16 * t + 4 * g + e;
        if (d < a.key_dim) a.dinitial_states[(at.head * a.key_dim + d) * a.value_dim + dv] = ds[t][e];
      }
}

// All chunks: dq, dk and, as sums over the keys' elements, what dbeta and dlog_decay need, from S0, U, dS1 and dR. A
// workgroup has a chunk of a key head, up to 128 of the keys' elements, and goes through the heads that share
// the key, so that their gradients are added in fp32 and in order. A wave has 16 of the elements as rows and the
// chunk's rows as columns. (In fp16 and fp32 64 elements, for the registers of one wave per SIMD.)
template <typename T, int DK>
constexpr int kGradWaves = DK < 128 || kPieces<T> > 1 ? 4 : 8;
template <typename T, int DK>
constexpr int kGradParts = DK / 16 / kGradWaves<T, DK>;

// What a row's gates' gradients are made of: k.z, q.dq - k.c, dR.V; and of its chunk, what the end's sum has.
struct GateSums {
  float kz, other, rv, end;
};
constexpr int kGateFields = 4;

// dbeta and dlog_decay of row `lane` of a head's chunk, in a wave.
__device__ __forceinline__ void finish_gates(const ccv1d_delta_args& a, int64_t b, int64_t c, int64_t h, int lane,
                                             const GateSums& x) {
  const ChunkRows r = chunk_row(a, b, c, h, lane);
  double s = (double)x.other - (double)r.beta * (double)x.kz + (lane == 63 ? (double)x.end : 0.0);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_down(s, d);
    const int run = __shfl_down(r.run, d);
    if (lane + d < 64 && run == r.run) s += o;
  }
  const int64_t t = c * kC + lane, o = (b * a.seqlen + t) * a.heads + h;
  if (t < a.seqlen) {
    store_as(a.dlog_decay, o, a.log_decay_dtype, r.live && !r.reset ? (float)s : 0.0f);
    store_as(a.dbeta, o, a.beta_dtype, r.live ? x.rv - x.kz : 0.0f);
  }
}

// The same where the keys' elements lie in several workgroups; a wave has a head's chunk.
template <int PARTS>
__global__ __launch_bounds__(256) void delta_gates_kernel(DeltaParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t hc = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (hc >= p.a.batch * p.a.heads * p.chunks) return;
  const int64_t head = hc / p.chunks, b = head / p.a.heads;
  GateSums x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const float* from = p.gates + (hc * PARTS + i) * (kGateFields * kC) + lane;
    x.kz += from[0], x.other += from[kC], x.end += from[3 * kC];
    if (i == 0) x.rv = from[2 * kC];  // each part has it
  }
  finish_gates(p.a, b, hc - head * p.chunks, head - b * p.a.heads, lane, x);
}

template <typename T, int DK>
__global__ __launch_bounds__((kGradWaves<T, DK>) * 64) void delta_grad_kernel(DeltaParams p) {
  constexpr int NI = kPieces<T>, KS = DK / 32, NW = kGradWaves<T, DK>, LG = 68;
  constexpr int PAIRS = (10 + NW - 1) / NW;
  __shared__ u4 fr[12][3][64];  // fragments: dR, U, dO of 32 value columns, then those of the products between rows
  __shared__ float gl[kC * LG];
  __shared__ ChunkShared sh;
  __shared__ float sums[NW][2][kC], vsum[kC], tail[NW];
  const ccv1d_delta_args& a = p.a;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int part = blockIdx.x % kGradParts<T, DK>, tile = part * NW + w;  // the wave's elements: 16 tile ...
  const int64_t kc = blockIdx.x / kGradParts<T, DK>, c = kc % p.chunks, bk = kc / p.chunks, b = bk / a.key_heads, kh = bk - b * a.key_heads;
  const int64_t t0 = c * kC;
  const u4* kf = p.kf + kc * (4 * KS * NI * 64);
  const u4* qf = p.qf + kc * (4 * KS * NI * 64);
  const u4* kt = p.kt + kc * (DK / 16 * 2 * NI * 64);
  const u4* qt = p.qt + kc * (DK / 16 * 2 * NI * 64);
  f4 dq[4] = {}, dk[4] = {};
  // The tiles of the products between rows that a wave has: n <= m.
  int tm[PAIRS], tn[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int x = w + NW * i;
    tm[i] = x < 1 ? 0 : x < 3 ? 1 : x < 6 ? 2 : 3;
    tn[i] = x < 10 ? x - tm[i] * (tm[i] + 1) / 2 : -1;
  }

  for (int64_t h = kh * p.group; h < (kh + 1) * p.group; ++h) {
    const int64_t head = b * a.heads + h, hc = head * p.chunks + c;
    const float* rows = p.rows + hc * (kRowFields * kC);
    const float* s0 = p.s0 + hc * ((int64_t)DK * p.dvp);
    const float* ds = p.ds + hc * ((int64_t)DK * p.dvp);
    const float* u = p.u + hc * (kC * p.dvp);
    const float* dr = p.dr + hc * (kC * p.dvp);
    if (w == 0) share_rows(a, b, c, h, lane, sh, nullptr);
    f4 aq[4] = {}, az[4] = {}, ac[4] = {}, go[PAIRS] = {}, gr[PAIRS] = {};
    float through = 0.0f, along = 0.0f;  // <dS1, S0> and dR.V of the lane's elements
    lds_barrier();
    for (int d0 = 0; d0 < p.dvp; d0 += 32) {
      // dR, U and dO of 32 value columns as fragments, one tile of rows and one of the three a turn
      for (int job = w; job < 12; job += NW) {
        const int kind = job >> 2, m = job & 3, i = 16 * m + col;
        const int64_t x = i * p.dvp + d0 + 4 * g;
        if (kind < 2) {
          const float* from = kind ? u : dr;
          const f4 lo = *reinterpret_cast<const f4*>(from + x), hi = *reinterpret_cast<const f4*>(from + x + 16);
          u4 f[3];
          split8<3>(lo, hi, f);
#pragma unroll
          for (int n = 0; n < 3; ++n) fr[kind * 4 + m][n][lane] = f[n];
          if (kind == 0 && sh.live[i]) {
            const T* vp = static_cast<const T*>(a.v) + b * a.v_stride_b + (t0 + i) * a.v_stride_t + h * a.v_stride_h;
            const int64_t d = d0 + 4 * g;
            f4 y = {0, 0, 0, 0}, z = {0, 0, 0, 0};
            if (d < a.value_dim) y = load4(vp + d, a.value_dim - d);
            if (d + 16 < a.value_dim) z = load4(vp + d + 16, a.value_dim - d - 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) along = fmaf(lo[e], y[e], fmaf(hi[e], z[e], along));
          }
        } else {
          f4 y = {0, 0, 0, 0}, z = {0, 0, 0, 0};
          if (sh.live[i]) {
            const T* op = static_cast<const T*>(a.dout) + b * a.dout_stride_b + (t0 + i) * a.dout_stride_t +
                          h * a.dout_stride_h;
            const int64_t d = d0 + 4 * g;
            if (d < a.value_dim) y = load4(op + d, a.value_dim - d);
            if (d + 16 < a.value_dim) z = load4(op + d + 16, a.value_dim - d - 16);
          }
          u4 f[NI];
          split8<NI>(y, z, f);
#pragma unroll
          for (int n = 0; n < NI; ++n) fr[8 + m][n][lane] = f[n];
        }
      }
      lds_barrier();
      const int64_t x = (int64_t)(16 * tile + col) * p.dvp + d0 + 4 * g;
      const f4 slo = *reinterpret_cast<const f4*>(s0 + x), shi = *reinterpret_cast<const f4*>(s0 + x + 16);
      const f4 dlo = *reinterpret_cast<const f4*>(ds + x), dhi = *reinterpret_cast<const f4*>(ds + x + 16);
      u4 sf[3], df[3];
      split8<3>(slo, shi, sf);
      split8<3>(dlo, dhi, df);
#pragma unroll
      for (int e = 0; e < 4; ++e) through = fmaf(slo[e], dlo[e], fmaf(shi[e], dhi[e], through));
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        u4 x3[3], xo[NI];
        load_frag(&fr[m][0][lane], x3);
        az[m] = mac<2>(sf, x3, az[m]);
        load_frag(&fr[8 + m][0][lane], xo);
        aq[m] = mac<2>(sf, xo, aq[m]);
        load_frag(&fr[4 + m][0][lane], x3);
        ac[m] = mac<2>(df, x3, ac[m]);
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i)
        if (tn[i] >= 0) {
          u4 un[3], x3[3], xo[NI];
          load_frag(&fr[4 + tn[i]][0][lane], un);
          load_frag(&fr[8 + tm[i]][0][lane], xo);
          go[i] = mac<2>(un, xo, go[i]);
          load_frag(&fr[tm[i]][0][lane], x3);
          gr[i] = mac<2>(un, x3, gr[i]);
        }
      lds_barrier();
    }
    // The factors of the columns, and k.(state's part of c).
    float state_part = 0.0f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const float into = rows[16 * m + col], rest = rows[kC + 16 * m + col];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        aq[m][e] = into != 0.0f ? a.scale * into * aq[m][e] : 0.0f;
        az[m][e] = into != 0.0f ? into * az[m][e] : 0.0f;
        ac[m][e] = rest != 0.0f ? rest * ac[m][e] : 0.0f;
      }
      u4 kv[NI];
      load_frag(kf + (m * KS + tile / 2) * (NI * 64) + lane, kv);
#pragma unroll
      for (int e = 0; e < 4; ++e) state_part = fmaf(piece_sum(kv, (tile & 1) * 4 + e), ac[m][e], state_part);
    }
    // Two rounds over the products between rows: scale D dO.U^T for dq and dk, D dR.U^T for z and dk.
#pragma unroll
    for (int round = 0; round < 2; ++round) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i)
        if (tn[i] >= 0) {
          const int row = 16 * tm[i] + col;
          f4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = 16 * tn[i] + 4 * g + e;
            const bool seen = (round ? j < row : j <= row) && sh.run[row] == sh.run[j];
            const float d = seen ? exp2_of(sh.sum[row] - sh.sum[j]) : 0.0f;
            x[e] = seen ? (round ? d * gr[i][e] : a.scale * d * go[i][e]) : 0.0f;
          }
          *reinterpret_cast<f4*>(&gl[row * LG + 16 * tn[i] + 4 * g]) = x;
        }
      lds_barrier();
      // fragments 0..5: sum over j, columns i (lower); 6..11: sum over i, columns j (upper)
      for (int job = w; job < 12; job += NW) {
        const int x = job < 6 ? job : job - 6;
        const int m = job < 6 ? (x < 2 ? x : x < 4 ? 2 : 3) : (x < 2 ? 0 : x < 4 ? 1 : x - 2);
        const int s = job < 6 ? (x < 2 ? 0 : x & 1) : (x < 4 ? x & 1 : 1);
        f4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (job < 6) {
          const float* from = &gl[(16 * m + col) * LG + 32 * s + 4 * g];
          lo = *reinterpret_cast<const f4*>(from);
          if (2 * s + 1 <= m) hi = *reinterpret_cast<const f4*>(from + 16);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 32 * s + 4 * g + e;
            if (2 * s >= m) lo[e] = gl[i * LG + 16 * m + col];
            hi[e] = gl[(i + 16) * LG + 16 * m + col];
            if (round) lo[e] *= -sh.beta[i], hi[e] *= -sh.beta[i + 16];
          }
        }
        u4 f[3];
        split8<3>(lo, hi, f);
#pragma unroll
        for (int n = 0; n < 3; ++n) fr[job][n][lane] = f[n];
      }
      lds_barrier();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u4 kx[NI], qx[NI], x3[3];
        load_frag(kt + (tile * 2 + s) * (NI * 64) + lane, kx);
        if (round == 0) load_frag(qt + (tile * 2 + s) * (NI * 64) + lane, qx);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (s <= m / 2) {
            load_frag(&fr[lower_frag(m, s)][0][lane], x3);
            if (round == 0) aq[m] = mac<2>(kx, x3, aq[m]);
            else az[m] = mac<2>(kx, x3, az[m]);
          }
          if (s >= m / 2) {
            load_frag(&fr[6 + upper_frag(m, s)][0][lane], x3);
            if (round == 0) ac[m] = mac<2>(qx, x3, ac[m]);
            else ac[m] = mac<2>(kx, x3, ac[m]);
          }
        }
      }
      lds_barrier();
    }
    // Sums over the keys' elements: k.z, and q.dq - k.c.
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float kz = 0.0f, rest = 0.0f;
      const float beta = sh.beta[16 * m + col];
      u4 kv[NI], qv[NI];
      load_frag(kf + (m * KS + tile / 2) * (NI * 64) + lane, kv);
      load_frag(qf + (m * KS + tile / 2) * (NI * 64) + lane, qv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float k = piece_sum(kv, (tile & 1) * 4 + e), q = piece_sum(qv, (tile & 1) * 4 + e);
        kz = fmaf(k, az[m][e], kz);
        rest = fmaf(q, aq[m][e], fmaf(-k, ac[m][e], rest));
        dk[m][e] += ac[m][e] - beta * az[m][e];
      }
      dq[m] += aq[m];
      kz += __shfl_xor(kz, 16), rest += __shfl_xor(rest, 16);
      kz += __shfl_xor(kz, 32), rest += __shfl_xor(rest, 32);
      if (g == 0) sums[w][0][16 * m + col] = kz, sums[w][1][16 * m + col] = rest;
    }
    if (w < 4) {  // dR.V: the wave's jobs were the tile of rows of its number
      along += __shfl_xor(along, 16);
      along += __shfl_xor(along, 32);
      if (g == 0) vsum[16 * w + col] = along;
    }
    const float whole = rows[4 * kC];
    float end = state_part + (whole != 0.0f ? whole * through : 0.0f);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) end += __shfl_xor(end, d);
    if (lane == 0) tail[w] = end;
    lds_barrier();
    if (w == 0) {
      GateSums x{0.0f, 0.0f, vsum[lane], 0.0f};
#pragma unroll
      for (int n = 0; n < NW; ++n) x.kz += sums[n][0][lane], x.other += sums[n][1][lane], x.end += tail[n];
      if constexpr (kGradParts<T, DK> == 1) {
        finish_gates(a, b, c, h, lane, x);
      } else {
        float* to = p.gates + (hc * kGradParts<T, DK> + part) * (kGateFields * kC) + lane;
        to[0] = x.kz, to[kC] = x.other, to[2 * kC] = x.rv, to[3 * kC] = x.end;
      }
    }
    lds_barrier();
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int i = 16 * m + col;
    if (t0 + i >= a.seqlen) continue;
    const bool live = sh.live[i];
    const int64_t row = ((b * a.seqlen + t0 + i) * a.key_heads + kh) * a.key_dim;
    const int64_t d = 16 * tile + 4 * g;
    if (d >= a.key_dim) continue;
    const f4 none = {0, 0, 0, 0};
    store4(static_cast<T*>(a.dq) + row + d, live ? dq[m] : none, a.key_dim - d);
    store4(static_cast<T*>(a.dk) + row + d, live ? dk[m] : none, a.key_dim - d);
  }
}

template <typename T, int DK>
hipError_t delta_launch_dk(const DeltaParams& p, bool backward, hipStream_t s) {
  const ccv1d_delta_args& a = p.a;
  const int64_t chunks = a.batch * a.key_heads * p.chunks, chains = delta_chains(a, p.tiles);
  hipError_t e;
  if (!backward) {
    e = start(&delta_prep_kernel<T, DK, false>, chunks, 256, s, p);
    if (e != hipSuccess) return e;
    return p.s0 ? start(&delta_fwd_kernel<T, DK, true>, chains, kChainWaves<DK> * 64, s, p)
                : start(&delta_fwd_kernel<T, DK, false>, chains, kChainWaves<DK> * 64, s, p);
  }
  e = start(&delta_prep_kernel<T, DK, true>, chunks, 256, s, p);
  if (e == hipSuccess) e = start(&delta_bwd_kernel<T, DK>, chains, kChainWaves<DK> * 64, s, p);
  if (e == hipSuccess) e = start(&delta_grad_kernel<T, DK>, chunks * kGradParts<T, DK>, kGradWaves<T, DK> * 64, s, p);
  if constexpr (kGradParts<T, DK> > 1)
    if (e == hipSuccess)
      e = start(&delta_gates_kernel<(kGradParts<T, DK>)>, (a.batch * a.heads * p.chunks + 3) / 4, 256, s, p);
  return e;
}

template <typename T>
hipError_t delta_launch(const DeltaParams& p, bool backward, hipStream_t s) {
  switch (p.dk) {
    case 64: return delta_launch_dk<T, 64>(p, backward, s);
    case 128: return delta_launch_dk<T, 128>(p, backward, s);
    default: return delta_launch_dk<T, 256>(p, backward, s);
  }
}

}  // namespace ops
}  // namespace ccv1d

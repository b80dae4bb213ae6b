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
// pieces are the fp32 number itself, and the products of pieces i + j <= 2 leave out 2^-24 of a term in the mean, 2^-21 at
// the most. (The second piece rounded in place of cut brings the error of fp32's dlog_decay from 4.8e-7 to 4.4e-7, the
// others' by 3 %, and costs the chains 2 %.)
// bf16 inputs are one piece, fp16 inputs two (11 bits), fp32 three. Nothing but the results themselves is rounded to fewer
// than fp32's bits: with two pieces of P, U and S0 in the outputs' products, 2^-15, one bf16 output in a hundred was the
// number beside the nearest. By the rates of the instructions (16x16x32 in 16 bits 16 cycles, 16x16x4 in fp32
// 32) three pieces against a bf16 input take 3/16 of fp32's time, against three pieces 6/16.
//
// A row that holds an infinity or NaN spoils its sequence from there on and nothing else, though the products run over all
// of a chunk's rows and zero times infinity is no number: keys and rates of such a row enter A as zero and its R is
// made NaN (chunk_row), and where a product over rows comes out as no number it is made again without those rows
// (sum_apart). A and T are numbers then, unless finite keys overflow them.
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
// Units of 16 bytes a lane of a fragment of P: its pieces, or, in 16 bits, the eight fp32 numbers.
template <typename T>
constexpr int kUnitsP = sizeof(T) == 4 ? 3 : 2;

// A wave's number, known to be the same in all lanes.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

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

// Element e of the half `half` of a fragment, from its pieces.
template <int N>
__device__ __forceinline__ float piece_sum(const u4 (&f)[N], int half, int e) {
  float s = 0.0f;
#pragma unroll
  for (int n = N - 1; n >= 0; --n) {
    const uint32_t w = half ? f[n][2 + (e >> 1)] : f[n][e >> 1];
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
// the carried state reaches the end; zero elsewhere; [5] and [6] G log2 e in 64 bits, [7] the number of resets.
constexpr int kRowFields = 8;

struct ChunkRows {
  double sum;   // G log2 e, from the row's sequence's start in the chunk
  int run;      // resets in the chunk up to the row
  bool live, reset;
  bool spoilt;  // holds an infinity or NaN; its decay and rate are then zero here
  float beta;
};

// What a row's factors are made of, as it lies in memory: requested together, before anything is looked at. Past the last
// row another is read, and not used.
struct RawGates {
  uint32_t g, beta;
  int64_t id, before;
  __device__ __forceinline__ void load(const ccv1d_delta_args& a, int64_t b, int64_t c, int64_t h, int lane) {
    const int64_t t = min(c * kC + lane, a.seqlen - 1);
    auto raw = [](const void* p, int64_t at, int dtype) -> uint32_t {
      if (dtype == CCV1D_F32) return static_cast<const uint32_t*>(p)[at];
      return static_cast<const uint16_t*>(p)[at];
    };
    g = raw(a.log_decay, b * a.log_decay_stride_b + t * a.log_decay_stride_t + h * a.log_decay_stride_h,
            a.log_decay_dtype);
    beta = raw(a.beta, b * a.beta_stride_b + t * a.beta_stride_t + h * a.beta_stride_h, a.beta_dtype);
    id = before = 0;
    if (a.seq_idx) {
      const int64_t at = b * a.seqlen + t, ahead = at - (t > 0);
      if (a.seq_idx_64) {
        const int64_t* s = static_cast<const int64_t*>(a.seq_idx);
        id = s[at], before = s[ahead];
      } else {
        const int32_t* s = static_cast<const int32_t*>(a.seq_idx);
        id = s[at], before = s[ahead];
      }
    }
  }
  static __device__ __forceinline__ float number(uint32_t x, int dtype) {
    return dtype == CCV1D_F32   ? __uint_as_float(x)
           : dtype == CCV1D_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)x)
                                : __uint_as_float(x << 16);
  }
};

// Row `lane` of chunk c. A row that starts a sequence, padding, and a decay that is zero in fp32 reset the state: its
// log-decay, which multiplies nothing, counts as zero, so that no sequence's sums meet another's.
__device__ __forceinline__ ChunkRows chunk_row(const ccv1d_delta_args& a, const RawGates& raw, int64_t c, int lane,
                                               bool bad_key) {
  ChunkRows r;
  const bool in = c * kC + lane < a.seqlen;
  r.live = in && raw.id >= 0;
  r.reset = in && (raw.id < 0 || raw.id != raw.before);
  float g = r.live ? RawGates::number(raw.g, a.log_decay_dtype) : 0.0f;
  r.beta = r.live ? RawGates::number(raw.beta, a.beta_dtype) : 0.0f;
  const bool infinite = g > 88.72f && !r.reset;  // its exponential, in fp32
  r.spoilt = r.live && (bad_key || g != g || g == INFINITY || infinite || !__builtin_isfinite(r.beta));
  if (g < -104.0f) r.reset = true;
  if (r.spoilt) r.beta = 0.0f;
  if (g != g || g == INFINITY || infinite) g = 0.0f;
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

// The decay of a state to a row that it reaches: never zero, which says that it does not, so that an infinity or NaN in
// it stays there however small the decay (the hardware's is zero below 2^-126). Of numbers up to 2^20 the smallest
// denormal number leaves less than 2^-128.
__device__ __forceinline__ float reaching(double x) { return fmaxf(exp2_of(x), 0x1p-149f); }

struct ChunkShared {
  double sum[kC];
  int run[kC];
  float beta[kC];
};

// A wave makes a chunk's rows of a head and leaves them in LDS and, in the workspace, what the chain needs of them.
__device__ __forceinline__ bool share_rows(const ccv1d_delta_args& a, const RawGates& raw, int64_t c, int lane,
                                           ChunkShared& sh, float* rows, bool bad_key) {
  const ChunkRows r = chunk_row(a, raw, c, lane, bad_key);
  sh.sum[lane] = r.sum, sh.run[lane] = r.run, sh.beta[lane] = r.beta;
  const double end = __shfl(r.sum, 63);
  const int last = __shfl(r.run, 63);
  rows[lane] = r.live && r.run == 0 ? reaching(r.sum) : 0.0f;
  rows[kC + lane] = r.live && r.run == last ? reaching(end - r.sum) : 0.0f;
  rows[2 * kC + lane] = r.spoilt ? __builtin_nanf("") : r.beta;
  rows[3 * kC + lane] = r.live ? 1.0f : 0.0f;
  rows[4 * kC + lane] = lane == 0 && last == 0 ? reaching(end) : 0.0f;
  reinterpret_cast<double*>(rows + 5 * kC)[lane] = r.sum;
  reinterpret_cast<int*>(rows + 7 * kC)[lane] = r.run;
  return r.live;
}

// A chunk's rows of q or k on their way to LDS: requested all at once, past the last row or element others, and not used.
template <typename T, int DK, int LD, int THREADS>
struct RowLoader {
  typedef T v4 __attribute__((ext_vector_type(4)));
  static constexpr int kUnits = kC * DK / 4 / THREADS;
  v4 v[kUnits];
  // A thread has the same four elements of rows THREADS / (DK / 4) apart.
  static __device__ __forceinline__ int row_of(int i) { return i * (THREADS / (DK / 4)) + threadIdx.x / (DK / 4); }
  static __device__ __forceinline__ int first() { return threadIdx.x % (DK / 4) * 4; }
  __device__ __forceinline__ void load(const T* from, int64_t stride_t, int dk, int64_t t0, int64_t seqlen) {
    const int last = (int)min((int64_t)kC, seqlen - t0) - 1;
    from += t0 * stride_t;
    const int d = first();
    if (dk == DK) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) __builtin_memcpy(&v[i], from + min(row_of(i), last) * stride_t + d, sizeof v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = from[min(row_of(i), last) * stride_t + min(d + e, dk - 1)];
    }
  }
  // Zero where `live` has no row and past the last element; `bad` says which rows hold an infinity or NaN.
  __device__ __forceinline__ void store(T* to, int dk, uint64_t live, int* bad) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int row = row_of(i), d = first(), left = live >> row & 1 ? dk - d : 0;
      float none = 0.0f;  // stays zero beside numbers
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e >= left) v[i][e] = (T)0.0f;
        none = fmaf(to_f32(v[i][e]), 0.0f, none);
      }
      if (none != 0.0f) bad[row] = 1;
      *reinterpret_cast<v4*>(to + row * LD + d) = v[i];
    }
  }
};

// All chunks: the operands of the chains as fragments, T and P (forward) or their transposes (backward).
// A workgroup has a chunk of a key head and all heads of it, or, where that is too few workgroups, one of them each
// (p.prep_heads). Reads q and k, writes them three (four) times as fragments and 30 KiB a head's chunk; bound by
// latency within a workgroup, so three of them a CU: at B=4 T=4096, 16 heads of 128 72 us forward and 82 backward, of
// which the 0.31 and 0.36 GB take 60 and 71 at a copy's rate. With q and k requested row by row behind the rows'
// factors, and those a head at a time, it took 108 and 116; with two workgroups a CU 128 before that.
template <typename T, int DK, bool BWD>
__global__ __launch_bounds__(256, 3) void delta_prep_kernel(DeltaParams p) {
  constexpr int NI = kPieces<T>, KS = DK / 32, LD = DK + 16 / sizeof(T), LA = 68;
  constexpr int NP = BWD ? 3 : kUnitsP<T>;
  // q and k, and once the fragments are made, A (then T) and T's tiles on the diagonal
  constexpr size_t kRowsBytes = 2 * kC * LD * sizeof(T), kMatrixBytes = (kC * LA + 4 * 16 * 20) * sizeof(float);
  __shared__ __attribute__((aligned(16))) char room[kRowsBytes > kMatrixBytes ? kRowsBytes : kMatrixBytes];
  __shared__ ChunkShared shared[4];  // of four heads at a time, one a wave
  __shared__ int bad_rows[2][kC];    // whether a row's k, q hold an infinity or NaN
  __shared__ uint64_t live_rows;
  T *kl = reinterpret_cast<T*>(room), *ql = kl + kC * LD;
  float *al = reinterpret_cast<float*>(room), *td = al + kC * LA;
  const ccv1d_delta_args& a = p.a;
  // The wave's number is not known to be the same in all lanes here: with branches on a scalar the compiler leaves out 7 of
  // the 10 waits behind the last product of T, keys above 128, backward, and every fourth row of T lacks a term
  // (tests/test_matrix_waits.py reads the built kernels for such places).
  const int lane = threadIdx.x & 63, m = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t shares = p.group / p.prep_heads, share = blockIdx.x % shares;
  const uint32_t unit = blockIdx.x / shares;  // (batch, key head, chunk); 32 bits, in which divisions are short
  const uint32_t bkh = unit / (uint32_t)p.chunks, batch = bkh / (uint32_t)a.key_heads;
  const int64_t kc = unit, c = unit - bkh * p.chunks, b = batch, kh = bkh - batch * (uint32_t)a.key_heads;
  const int64_t t0 = c * kC;
  const int h0 = (int)kh * p.group + share * p.prep_heads, heads = h0 + p.prep_heads;
  auto rows_of = [&](int h) { return p.rows + ((b * a.heads + h) * p.chunks + c) * (kRowFields * kC); };
  // The rows' gates first, then q and k: the rows' factors are made while these are on their way.
  RawGates raw;
  RowLoader<T, DK, LD, 256> kr, qr;
  raw.load(a, b, c, min(h0 + m, heads - 1), lane);
  kr.load(static_cast<const T*>(a.k) + b * a.k_stride_b + kh * a.k_stride_h, a.k_stride_t, (int)a.key_dim, t0, a.seqlen);
  constexpr bool BOTH = kPieces<T> * DK <= 256;  // else q's are requested when k's are there: registers
  if (BOTH)
    qr.load(static_cast<const T*>(a.q) + b * a.q_stride_b + kh * a.q_stride_h, a.q_stride_t, (int)a.key_dim, t0, a.seqlen);
  if (h0 + m < heads) {
    const bool live = share_rows(a, raw, c, lane, shared[m], rows_of(h0 + m), false);
    const uint64_t all = __ballot(live);
    if (m == 0 && lane == 0) live_rows = all;
  }
  if (m == 3) bad_rows[0][lane] = bad_rows[1][lane] = 0;
  lds_barrier();
  kr.store(kl, (int)a.key_dim, live_rows, bad_rows[0]);
  if (!BOTH)
    qr.load(static_cast<const T*>(a.q) + b * a.q_stride_b + kh * a.q_stride_h, a.q_stride_t, (int)a.key_dim, t0, a.seqlen);
  qr.store(ql, (int)a.key_dim, live_rows, bad_rows[1]);
  lds_barrier();
  const uint64_t bad_k = __ballot(bad_rows[0][lane] != 0), bad_q = __ballot(bad_rows[1][lane] != 0);
  if (bad_k) {  // the same in all waves
    for (int i = threadIdx.x; i < kC * DK; i += 256)
      if (bad_k >> (i / DK) & 1) kl[i / DK * LD + i % DK] = (T)0.0f;
    raw.load(a, b, c, min(h0 + m, heads - 1), lane);
    if (h0 + m < heads) share_rows(a, raw, c, lane, shared[m], rows_of(h0 + m), bad_k >> lane & 1);
    lds_barrier();
  }

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
    if (share == 0)
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
  if (share == 0)
#pragma unroll
    for (int i = 0; i < DK / 16 / 4; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int t = m + 4 * i;
        auto column = [&](const T* from, uint64_t bad, u4* to) {
          u4 f[NI];
          f4 x, y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = to_f32(from[(32 * s + 4 * g + e) * LD + 16 * t + col]);
            y[e] = to_f32(from[(32 * s + 16 + 4 * g + e) * LD + 16 * t + col]);
          }
          if (bad)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (bad >> (32 * s + 4 * g + e) & 1) x[e] = 0.0f;
              if (bad >> (32 * s + 16 + 4 * g + e) & 1) y[e] = 0.0f;
            }
          split8<NI>(x, y, f);
#pragma unroll
          for (int n = 0; n < NI; ++n) to[((t * 2 + s) * NI + n) * 64 + lane] = f[n];
        };
        column(kl, 0, p.kt + kc * (DK / 16 * 2 * NI * 64));
        if constexpr (BWD) column(ql, bad_q, p.qt + kc * (DK / 16 * 2 * NI * 64));
      }

  for (int h = h0; h < heads; ++h) {
    const int64_t hc = (b * a.heads + h) * p.chunks + c;
    u4* tf = p.tf + hc * (kTri * 3 * 64);
    u4* pf = p.pf + hc * (kTri * NP * 64);
    const int turn = (h - h0) & 3;
    lds_barrier();
    if (turn == 0 && h > h0) {  // four more heads
      if (h + m < heads) {
        raw.load(a, b, c, h + m, lane);
        share_rows(a, raw, c, lane, shared[m], rows_of(h + m), bad_rows[0][lane]);
      }
      lds_barrier();
    }
    const ChunkShared& sh = shared[turn];
    // Of tile (n, m) a lane has one i and four j, backward four i and one j.
    double sum_m[BWD ? 4 : 1];
    int run_m[BWD ? 4 : 1];
    float beta_m[BWD ? 4 : 1];
#pragma unroll
    for (int e = 0; e < (BWD ? 4 : 1); ++e) {
      const int i = 16 * m + (BWD ? 4 * g + e : col);
      sum_m[e] = sh.sum[i], run_m[e] = sh.run[i], beta_m[e] = sh.beta[i];
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n > m + 1) continue;
      f4 pv = {0, 0, 0, 0};
      if (n <= m) {
        f4 av;
        double sum_n[BWD ? 1 : 4];
        int run_n[BWD ? 1 : 4];
#pragma unroll
        for (int e = 0; e < (BWD ? 1 : 4); ++e) {
          const int j = 16 * n + (BWD ? col : 4 * g + e);
          sum_n[e] = sh.sum[j], run_n[e] = sh.run[j];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int y = BWD ? 0 : e;
          const int x = BWD ? e : 0, i = 16 * m + (BWD ? 4 * g + e : col), j = 16 * n + (BWD ? col : 4 * g + e);
          const bool seen = (j <= i) & (run_m[x] == run_n[y]);
          const float d = exp2_of(sum_m[x] - sum_n[y]), av_e = beta_m[x] * d * kk[n][e], pv_e = a.scale * d * qk[n][e];
          av[e] = seen & (j < i) ? av_e : 0.0f;
          pv[e] = seen ? pv_e : 0.0f;
        }
        if constexpr (BWD) {
#pragma unroll
          for (int e = 0; e < 4; ++e) al[(16 * m + 4 * g + e) * LA + 16 * n + col] = av[e];
        } else {
          *reinterpret_cast<f4*>(&al[(16 * m + col) * LA + 16 * n + 4 * g]) = av;
        }
      } else if (m & 1) {
        continue;  // no half of a fragment that is read
      }
      if constexpr (NP == 2) {
        reinterpret_cast<f4*>(pf)[(lower_frag(m, n / 2) * 2 + (n & 1)) * 64 + lane] = pv;
        continue;
      }
      u2 w[3];
      split4<3>(pv, w);
      if constexpr (BWD) {
        // rows j of tile n, sum over i of tile m; the tile m of a pair in front of n's is zero
        store_half<3>(pf + upper_frag(n, m / 2) * (NP * 64) + lane, m & 1, w);
      } else {
        store_half<3>(pf + lower_frag(m, n / 2) * (NP * 64) + lane, n & 1, w);
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
        for (int j = 0; j < i; j += 4) {
          const f4 av = *reinterpret_cast<const f4*>(&al[(16 * g + i) * LA + 16 * g + j]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j + e < i) s = fmaf(-av[e], x[j + e], s);
        }
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

// Which head and which CT tiles of 16 value columns a workgroup of a chain has: workgroups go to the XCDs in turn, and all
// columns of a head to one, whose L2 then holds the head's fragments once.
struct ChainPlace {
  int64_t head;  // batch * heads + head
  int64_t dv0;
  bool any;
};
template <int CT>
__device__ __forceinline__ ChainPlace chain_place(const DeltaParams& p) {
  const int64_t xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  ChainPlace r;
  const int64_t groups = p.tiles / CT;
  r.head = xcd + 8 * (slot / groups);
  r.dv0 = slot % groups * (16 * CT);
  r.any = r.head < p.a.batch * p.a.heads;
  return r;
}

// How a chain's eight waves share the work. Four carry the states, 32 or 64 of the keys' elements each (keys of up to
// 64 elements twice over, with half of the chunk's rows each in the first product), and 16 of the chunk's rows
// in the products between rows; the other four do what no later chunk waits for.
template <int DK>
struct Chain {
  static constexpr int kKS = DK / 32;                     // steps of the sum over the keys' elements
  static constexpr int kKB = kKS < 4 ? 1 : kKS / 4;       // of a wave
  static constexpr int kParts = kKS < 4 ? kKS : 4;        // partial sums of the first product
  static constexpr int kRows = kKS < 4 ? 2 : 4;           // tiles of rows of a wave in it
  static __device__ __forceinline__ int part(int w) { return w % kParts; }
  static __device__ __forceinline__ int rows0(int w) { return kKS < 4 ? w / 2 * 2 : 0; }
};

// Whether a chain requests the next chunk's operands of k while it works on this one's: not for the largest heads
// in fp16 and fp32, whose operands alone are 130 and 200 registers.
template <typename T, int DK>
constexpr bool kLoadAhead = kPieces<T> * DK < 512;

template <int N>
__device__ __forceinline__ void load_frag(const u4* p, uint32_t lane, u4 (&o)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) o[n] = p[n * 64 + lane];
}

// An element as it lies in memory, in a register of its own: two 16-bit ones packed into one would be waited for
// where they are packed.
template <typename T>
__device__ __forceinline__ uint32_t load_raw(const T* p) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, *p);
  else return *reinterpret_cast<const uint16_t*>(p);
}
template <typename T>
__device__ __forceinline__ float raw_to_f32(uint32_t x) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(x);
  else if constexpr (kPieces<T> == 1) return __uint_as_float(x << 16);
  else return (float)__builtin_bit_cast(T, (uint16_t)x);
}

// The four rows of a lane in a tile of 16, of one column of a tensor, read one by one. Past the last row or column
// another is read, and not used.
template <typename T>
struct ColumnReader {
  const T* p;  // row 4 (lane / 16) of the tile of the first chunk
  int64_t stride;
  __device__ __forceinline__ void at(const void* base, int64_t offset, int64_t stride_t, int64_t dv, int64_t dim, int row) {
    p = static_cast<const T*>(base) + offset + min(dv, dim - 1) + row * stride_t;
    stride = stride_t;
  }
  __device__ __forceinline__ void load(int64_t c, int64_t seqlen, int row, uint32_t (&o)[4]) const {
    const T* at = p + c * (kC * stride);
    if ((c + 1) * kC <= seqlen) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = load_raw(at + e * stride);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t over = c * kC + row + e - (seqlen - 1);
        o[e] = load_raw(at + (e - max((int64_t)0, over)) * stride);
      }
    }
  }
};

template <int N>
__device__ __forceinline__ bool any_not_finite(const f4 (&x)[N]) {
  float none = 0.0f;  // stays zero beside numbers
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) none = fmaf(x[n][e], 0.0f, none);
  return __ballot(none != 0.0f) != 0;
}

// A product over the chunk's rows, a[0] f[0] + a[1] f[1] from `base` on, where it came out as no number: rows of f that hold
// none are left out, and the result's rows (the lane's four, from `row` on) of their sequences made NaN, those behind
// them or, UPPER, before them. What is a number has the bits that it has beside numbers. IN_TURN: one sum
// for both, else one each. f is [2][NB][64] units in LDS; FROM..TO of it are read.
template <bool UPPER, bool IN_TURN, int LIM, int NA, int NB>
__device__ __forceinline__ f4 sum_apart(const u4 (&a)[2][NA], const u4 (*f)[NB][64], uint32_t lane, int from, int to, f4 base,
                                        const int* run, int row) {
  asm volatile("" : "+v"(lane), "+v"(row));  // what is made of them here is made here: registers
  const uint32_t g = lane >> 4;
  uint32_t bad[2] = {0, 0};
  f4 r = base, other = {0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (s < from || s > to) continue;
    __builtin_amdgcn_sched_barrier(0);
    u4 x[NB];
    load_frag(&f[s][0][0], lane, x);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        if ((x[0][i] >> (16 * half) & 0x7f80u) == 0x7f80u) {
          bad[s] |= 1u << ((i < 2 ? 0 : 16) + 4 * g + 2 * (i & 1) + half);
#pragma unroll
          for (int n = 0; n < NB; ++n) x[n][i] &= half ? 0x0000ffffu : 0xffff0000u;
        }
    if (IN_TURN || s == from) r = mac<LIM>(a[s], x, r);
    else other = mac<LIM>(a[s], x, other);
    bad[s] |= __shfl_xor(bad[s], 16);
    bad[s] |= __shfl_xor(bad[s], 32);
  }
  r += other;
  const uint64_t starts = __ballot(lane && run[lane] != run[lane ? lane - 1 : 0]), rows = bad[0] | (uint64_t)bad[1] << 32;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    __builtin_amdgcn_sched_barrier(0);
    const int i = row + e;
    const uint64_t up_to = ~uint64_t(0) >> (63 - i), later = starts & ~up_to;
    const uint64_t own = UPPER ? ~(up_to >> 1) & (later ? (later & -later) - 1 : ~uint64_t(0))
                               : up_to & (~uint64_t(0) << (63 - __clzll((starts & up_to) | 1)));
    if (rows & own) r[e] = __builtin_nanf("");
  }
  return r;
}

// The chain of states forward: a workgroup has CT tiles of 16 value columns of a head. Bound by latency: three
// products after one another a chunk, each behind a barrier; the waves that make the outputs run beside them. At B=4
// T=4096, 16 heads of 128 in bf16, training, 300 us, of which states and corrections kept take 90 and operands out of
// the caches 80; VALUs are 23 %, matrix cores 15 %, LDS 18 % busy. Without the four waves beside 378; 64 columns a
// workgroup with the operands through LDS 490 to 914; 16 columns a wave on its own 1525; operands requested into the L2 two
// chunks ahead 306 (then 276).
template <typename T, int DK, int CT, bool SAVE>
__global__ __launch_bounds__(512) void delta_fwd_kernel(DeltaParams p) {
  using L = Chain<DK>;
  constexpr int NI = kPieces<T>, KS = L::kKS, KB = L::kKB, NP = kUnitsP<T>;
  constexpr bool AHEAD = kLoadAhead<T, DK>;
  __shared__ f4 red[CT][L::kParts][4][64];
  __shared__ u4 sp[CT][KS][3][64], rb[CT][2][3][64], ub[CT][2][3][64], uo[CT][2][3][64];
  const ccv1d_delta_args& a = p.a;
  const ChainPlace at = chain_place<CT>(p);
  if (!at.any) return;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = wave_index(), w = wave & 3;
  const int64_t b = at.head / a.heads, h = at.head - b * a.heads, kh = h / p.group;
  const int64_t dv = at.dv0 + col;
  const bool all_columns = at.dv0 + 16 * CT <= a.value_dim;
  const int64_t N = p.chunks;
  const int row = 16 * w + 4 * g;  // the lane's first row of the wave's tile of rows
  const u4* kf = p.kf + (b * a.key_heads + kh) * N * (4 * KS * NI * 64);
  const u4* qf = p.qf + (b * a.key_heads + kh) * N * (4 * KS * NI * 64);
  const u4* kt = p.kt + (b * a.key_heads + kh) * N * (DK / 16 * 2 * NI * 64);
  const u4* tf = p.tf + at.head * N * (kTri * 3 * 64);
  const u4* pf = p.pf + at.head * N * (kTri * NP * 64);
  const float* rows = p.rows + at.head * N * (kRowFields * kC);
  auto runs_of = [&](int64_t c) {
    return reinterpret_cast<const int*>(rows + c * (kRowFields * kC) + 7 * kC);
  };

  if (wave >= 4) {  // outputs: O = scale e^G Q S0 + P U of a tile of rows
    u4 qx[KS][NI], raw[2][NP], px[2][3];
    f4 into, live;
    auto load_q = [&](int64_t c) {
#pragma unroll
      for (int s = 0; s < KS; ++s) load_frag(qf + c * (4 * KS * NI * 64) + (w * KS + s) * (NI * 64), lane, qx[s]);
      into = *reinterpret_cast<const f4*>(rows + c * (kRowFields * kC) + row);
    };
    auto load_p = [&](int64_t c) {
      live = *reinterpret_cast<const f4*>(rows + c * (kRowFields * kC) + 3 * kC + row);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= w / 2) load_frag(pf + c * (kTri * NP * 64) + lower_frag(w, s) * (NP * 64), lane, raw[s]);
    };
    const int64_t stride = a.heads * a.value_dim;
    T* out = static_cast<T*>(a.out) + (b * a.seqlen + row) * stride + h * a.value_dim + dv;
    load_q(0);
    load_p(0);
    for (int64_t c = 0; c < N; ++c) {
      const int64_t next = c + 1 < N ? c + 1 : c;
      lds_barrier();
      f4 o[CT], base[CT], y[CT][2] = {};
      auto state_part = [&](int from, int to) {  // steps of Q S0
#pragma unroll
        for (int n = 0; n < CT; ++n)
#pragma unroll
          for (int s = from; s < to; ++s) {
            u4 so[3];
            load_frag(&sp[n][s][0][0], lane, so);
            y[n][s & 1] = mac<2>(qx[s], so, y[n][s & 1]);
          }
      };
      // Up to 128 of the keys' elements the chain's waves have more to do behind the next barrier than in front of it: a
      // prompt of 16384, 16 heads of 128, all steps in front 550 us, half 536, a quarter 499, none 508; with 256, T=4096, 4
      // heads, all 156, half 170, a quarter 168, none 174.
      constexpr int FRONT = DK <= 128 ? KS / 4 : KS;
      state_part(0, FRONT);
      lds_barrier();
      state_part(FRONT, KS);
#pragma unroll
      for (int n = 0; n < CT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[n][e] = a.scale * into[e] * (y[n][0][e] + y[n][1][e]);
          if (into[e] == 0.0f) o[n][e] = 0.0f;  // not a product with zero: the state may hold no number
        }
      // Here, not later: the next rows' factors would get other registers, and wait to be moved.
#pragma unroll
      for (int n = 0; n < CT; ++n) asm volatile("" : "+v"(o[n]));
      load_q(next);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= w / 2) {
          if constexpr (NP == 2) {
            asm volatile("" : "+v"(raw[s][0]), "+v"(raw[s][1]));  // not before: right behind the loads it would wait for them
            split8<3>(__builtin_bit_cast(f4, raw[s][0]), __builtin_bit_cast(f4, raw[s][1]), px[s]);
          } else {
#pragma unroll
            for (int n = 0; n < 3; ++n) px[s][n] = raw[s][n];
          }
        }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < CT; ++n) {
        base[n] = o[n];
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (s <= w / 2) {
            u4 u[3];
            load_frag(&uo[n][s][0][0], lane, u);
            o[n] = mac<2>(px[s], u, o[n]);
          }
      }
      if (any_not_finite(o))
#pragma unroll
        for (int n = 0; n < CT; ++n)
          o[n] = sum_apart<false, true, 2>(px, uo[n], lane, 0, w / 2, base[n], runs_of(c), row);
      T* to = out + c * (kC * stride);
#pragma unroll
      for (int n = 0; n < CT; ++n)
        if (dv + 16 * n < a.value_dim)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c * kC + row + e < a.seqlen) to[e * stride + 16 * n] = (T)(live[e] != 0.0f ? o[n][e] : 0.0f);
      load_p(next);
    }
    return;
  }

  const int part = L::part(w), rows0 = L::rows0(w);
  const bool keeper = L::kParts == 4 || w < L::kParts;  // of two waves with the same states, the first
  u4 kx[KB][L::kRows][NI], kc[2 * KB][2][NI], tx[2][3];
  uint32_t v[CT][4];
  f4 into, rest, beta, live;
  float whole = 0.0f, whole_now;
  ColumnReader<T> vr[CT];
#pragma unroll
  for (int n = 0; n < CT; ++n)
    vr[n].at(a.v, b * a.v_stride_b + h * a.v_stride_h, a.v_stride_t, dv + 16 * n, a.value_dim, row);
  auto load_k_of = [&](int64_t c, int i) {
#pragma unroll
    for (int m = 0; m < L::kRows; ++m)
      load_frag(kf + c * (4 * KS * NI * 64) + ((rows0 + m) * KS + part * KB + i) * (NI * 64), lane, kx[i][m]);
  };
  auto load_kc_of = [&](int64_t c, int s) {
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
      load_frag(kt + c * (DK / 16 * 2 * NI * 64) + ((2 * KB * part + t) * 2 + s) * (NI * 64), lane, kc[t][s]);
  };
  auto load_k = [&](int64_t c) {
#pragma unroll
    for (int i = 0; i < KB; ++i) load_k_of(c, i);
  };
  auto load_kc = [&](int64_t c) {
    load_kc_of(c, 0);
    load_kc_of(c, 1);
  };
  auto load_v = [&](int64_t c) {
    const float* r = rows + c * (kRowFields * kC);
    whole = r[4 * kC];
    into = *reinterpret_cast<const f4*>(r + row);
    beta = *reinterpret_cast<const f4*>(r + 2 * kC + row);
    live = *reinterpret_cast<const f4*>(r + 3 * kC + row);
#pragma unroll
    for (int n = 0; n < CT; ++n) vr[n].load(c, a.seqlen, row, v[n]);
  };
  auto load_t = [&](int64_t c) {
    rest = *reinterpret_cast<const f4*>(rows + c * (kRowFields * kC) + kC + row);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s <= w / 2) load_frag(tf + c * (kTri * 3 * 64) + lower_frag(w, s) * (3 * 64), lane, tx[s]);
  };

  f4 state[CT][2 * KB];
#pragma unroll
  for (int n = 0; n < CT; ++n)
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t d = 32 * KB * part + 16 * t + 4 * g + e;
        state[n][t][e] = a.initial_states && dv + 16 * n < a.value_dim && d < a.key_dim
                             ? a.initial_states[(at.head * a.key_dim + d) * a.value_dim + dv + 16 * n]
                             : 0.0f;
      }
  // Addresses of what is kept: a part that is the same in all lanes, and 32 bits a lane.
  float* s0 = SAVE ? p.s0 + at.head * N * (DK * (int64_t)p.dvp) + 32 * KB * part * (int64_t)p.dvp + at.dv0 : nullptr;
  float* us = SAVE ? p.u + at.head * N * (kC * (int64_t)p.dvp) + 16 * w * (int64_t)p.dvp + at.dv0 : nullptr;
  const uint32_t kept = 4 * g * p.dvp + col;
  uint32_t ld = p.dvp;
  if constexpr (AHEAD) {
    load_k(0);
    load_kc(0);
  }
  load_v(0);
  load_t(0);
  for (int64_t c = 0; c < N; ++c) {
    const int64_t next = c + 1 < N ? c + 1 : c;
    asm volatile("" : "+s"(ld));  // offsets are made anew for each chunk: registers
    {
      f4 x[CT][L::kRows] = {};
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        if constexpr (!AHEAD) load_k_of(c, i);
#pragma unroll
        for (int n = 0; n < CT; ++n) {
          u4 sb[3];
          split8<3>(state[n][2 * i], state[n][2 * i + 1], sb);
          if (keeper)
#pragma unroll
            for (int j = 0; j < 3; ++j) sp[n][part * KB + i][j][lane] = sb[j];
#pragma unroll
          for (int m = 0; m < L::kRows; ++m) x[n][m] = mac<2>(kx[i][m], sb, x[n][m]);
        }
      }
#pragma unroll
      for (int n = 0; n < CT; ++n)
#pragma unroll
        for (int m = 0; m < L::kRows; ++m) red[n][part][rows0 + m][lane] = x[n][m];
    }
    if constexpr (SAVE)
      if (keeper) {
        float* to = s0 + c * (DK * (int64_t)p.dvp);
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* line = to + (16 * t + e) * ld;
#pragma unroll
            for (int n = 0; n < CT; ++n) (line + 16 * n)[kept] = state[n][t][e];
          }
      }
    if constexpr (AHEAD) load_k(next);
    // A chunk that the carried state goes through has no reset and no padding but past the last row, where beta and
    // the keys are zero: only the others need selections in place of products with zero.
    whole_now = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(whole)));
    const bool plain = whole_now != 0.0f && all_columns;
    lds_barrier();
#pragma unroll
    for (int n = 0; n < CT; ++n) {
      f4 x = red[n][0][w][lane];
#pragma unroll
      for (int j = 1; j < L::kParts; ++j) x += red[n][j][w][lane];
      f4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = beta[e] * (raw_to_f32<T>(v[n][e]) - into[e] * x[e]);
      if (!plain)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          r[e] = beta[e] * ((live[e] != 0.0f && dv + 16 * n < a.value_dim ? raw_to_f32<T>(v[n][e]) : 0.0f) -
                            (into[e] != 0.0f ? into[e] * x[e] : 0.0f));
      u2 half[3];
      split4<3>(r, half);
      store_half<3>(&rb[n][w / 2][0][lane], w & 1, half);
    }
    load_v(next);
    lds_barrier();
    f4 u[CT];
#pragma unroll
    for (int n = 0; n < CT; ++n) {
      f4 u1 = {0, 0, 0, 0};
      u4 rx[3];
      u[n] = f4{0, 0, 0, 0};
      load_frag(&rb[n][0][0][0], lane, rx);
      u[n] = mac<2>(tx[0], rx, u[n]);
      if (w >= 2) {
        load_frag(&rb[n][1][0][0], lane, rx);
        u1 = mac<2>(tx[1], rx, u1);
      }
      u[n] += u1;
    }
    if (any_not_finite(u))
#pragma unroll
      for (int n = 0; n < CT; ++n)
        u[n] = sum_apart<false, false, 2>(tx, rb[n], lane, 0, w / 2, f4{0, 0, 0, 0}, runs_of(c), row);
#pragma unroll
    for (int n = 0; n < CT; ++n) {
      f4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = rest[e] * u[n][e];
      if (!plain)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = rest[e] != 0.0f ? y[e] : 0.0f;
      u2 half[3];
      split4<3>(y, half);
      store_half<3>(&ub[n][w / 2][0][lane], w & 1, half);
      split4<3>(u[n], half);
      store_half<3>(&uo[n][w / 2][0][lane], w & 1, half);
    }
    if constexpr (SAVE) {
      float* to = us + c * (kC * (int64_t)p.dvp);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float* line = to + e * ld;
#pragma unroll
        for (int n = 0; n < CT; ++n) (line + 16 * n)[kept] = u[n][e];
      }
    }
    load_t(next);
#pragma unroll
    for (int n = 0; n < CT; ++n)
#pragma unroll
      for (int t = 0; t < 2 * KB; ++t) {
        state[n][t] *= whole_now;
        if (whole_now == 0.0f) state[n][t] = f4{0, 0, 0, 0};
      }
    lds_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (!AHEAD) load_kc_of(c, s);
#pragma unroll
      for (int n = 0; n < CT; ++n) {
        u4 ux[3];
        load_frag(&ub[n][s][0][0], lane, ux);
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t) state[n][t] = mac<2>(kc[t][s], ux, state[n][t]);
      }
    }
    if constexpr (AHEAD) load_kc(next);
  }
  if (a.final_states && keeper)
#pragma unroll
    for (int n = 0; n < CT; ++n)
      if (dv + 16 * n < a.value_dim)
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t d = 32 * KB * part + 16 * t + 4 * g + e;
            if (d < a.key_dim) a.final_states[(at.head * a.key_dim + d) * a.value_dim + dv + 16 * n] = state[n][t][e];
          }
}

// The chain of the states' gradients, from the last chunk to the first; divided like the forward's. Leaves dS1 of
// every chunk and dR, and writes dV. The waves beside the chain make P^T dO and scale Q^T (e^G dO) a chunk ahead. Bound
// as the forward is: 300 us at the same sizes.
template <typename T, int DK, int CT>
__global__ __launch_bounds__(512) void delta_bwd_kernel(DeltaParams p) {
  using L = Chain<DK>;
  constexpr int NI = kPieces<T>, KS = L::kKS, KB = L::kKB, TQ = DK / 64;  // tiles of the keys' elements beside the chain
  constexpr bool AHEAD = kLoadAhead<T, DK>;
  __shared__ f4 red[CT][L::kParts][4][64], pd[CT][4][64], qd[CT][DK / 16][64];
  __shared__ u4 ob[CT][2][NI][64], oq[CT][2][3][64], ub[CT][2][3][64], rb[CT][2][3][64];
  const ccv1d_delta_args& a = p.a;
  const ChainPlace at = chain_place<CT>(p);
  if (!at.any) return;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = wave_index(), w = wave & 3;
  const int64_t b = at.head / a.heads, h = at.head - b * a.heads, kh = h / p.group;
  const int32_t dv = (int32_t)at.dv0 + col, dim = (int32_t)a.value_dim, seqlen = (int32_t)a.seqlen;
  const int32_t N = p.chunks;
  const int row = 16 * w + 4 * g;
  const u4* kf = p.kf + (b * a.key_heads + kh) * (int64_t)N * (4 * KS * NI * 64);
  const u4* kt = p.kt + (b * a.key_heads + kh) * (int64_t)N * (DK / 16 * 2 * NI * 64);
  const u4* qt = p.qt + (b * a.key_heads + kh) * (int64_t)N * (DK / 16 * 2 * NI * 64);
  const u4* tf = p.tf + at.head * (int64_t)N * (kTri * 3 * 64);
  const u4* pf = p.pf + at.head * (int64_t)N * (kTri * 3 * 64);
  const float* rows = p.rows + at.head * (int64_t)N * (kRowFields * kC);
  auto runs_of = [&](int32_t c) {
    return reinterpret_cast<const int*>(rows + c * (int64_t)(kRowFields * kC) + 7 * kC);
  };

  if (wave >= 4) {
    u4 px[2][3], qx[TQ][2][NI];
    f4 into, live, sum[CT][TQ], z[CT];
    uint32_t dy[CT][4];
    ColumnReader<T> yr[CT];
#pragma unroll
    for (int n = 0; n < CT; ++n)
      yr[n].at(a.dout, b * a.dout_stride_b + h * a.dout_stride_h, a.dout_stride_t, dv + 16 * n, dim, row);
    auto load_dy = [&](int32_t c) {
      into = *reinterpret_cast<const f4*>(rows + c * (int64_t)(kRowFields * kC) + row);
      live = *reinterpret_cast<const f4*>(rows + c * (int64_t)(kRowFields * kC) + 3 * kC + row);
#pragma unroll
      for (int n = 0; n < CT; ++n) yr[n].load(c, seqlen, row, dy[n]);
    };
    auto load_pq = [&](int32_t c) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= w / 2) load_frag(pf + c * (int64_t)(kTri * 3 * 64) + upper_frag(w, s) * (3 * 64), lane, px[s]);
      if constexpr (AHEAD)
#pragma unroll
        for (int t = 0; t < TQ; ++t)
#pragma unroll
          for (int s = 0; s < 2; ++s)
            load_frag(qt + c * (int64_t)(DK / 16 * 2 * NI * 64) + ((TQ * w + t) * 2 + s) * (NI * 64), lane, qx[t][s]);
    };
    auto share = [&](int32_t c) {  // dO of the wave's rows, and scale e^G dO
#pragma unroll
      for (int n = 0; n < CT; ++n) {
        f4 d, s;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] = live[e] != 0.0f && dv + 16 * n < dim ? raw_to_f32<T>(dy[n][e]) : 0.0f;
          s[e] = into[e] != 0.0f ? a.scale * into[e] * d[e] : 0.0f;
        }
        u2 half[NI], third[3];
        split4<NI>(d, half);
        store_half<NI>(&ob[n][w / 2][0][lane], w & 1, half);
        split4<3>(s, third);
        store_half<3>(&oq[n][w / 2][0][lane], w & 1, third);
      }
      load_dy(c ? c - 1 : 0);
    };
    auto products = [&](int32_t c) {
#pragma unroll
      for (int n = 0; n < CT; ++n) {
        f4 y[2] = {};
#pragma unroll
        for (int t = 0; t < TQ; ++t) sum[n][t] = f4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u4 o[NI], x[3];
          if (s >= w / 2) {
            load_frag(&ob[n][s][0][0], lane, o);
            y[s] = mac<2>(px[s], o, y[s]);
          }
          load_frag(&oq[n][s][0][0], lane, x);
#pragma unroll
          for (int t = 0; t < TQ; ++t) {
            if constexpr (!AHEAD)
              load_frag(qt + c * (int64_t)(DK / 16 * 2 * NI * 64) + ((TQ * w + t) * 2 + s) * (NI * 64), lane, qx[t][s]);
            sum[n][t] = mac<2>(qx[t][s], x, sum[n][t]);
          }
        }
        z[n] = y[0] + y[1];
      }
    };
    auto leave = [&](int32_t c) {
      if (any_not_finite(z))
#pragma unroll
        for (int n = 0; n < CT; ++n)
          z[n] = sum_apart<true, false, 2>(px, ob[n], lane, w / 2, 1, f4{0, 0, 0, 0}, runs_of(c), row);
#pragma unroll
      for (int n = 0; n < CT; ++n) pd[n][w][lane] = z[n];
      load_pq(c ? c - 1 : 0);
    };
    load_dy(N - 1);
    load_pq(N - 1);
    share(N - 1);
    lds_barrier();
    products(N - 1);
    leave(N - 1);
    for (int32_t c = N - 1; c >= 0; --c) {
      lds_barrier();
#pragma unroll
      for (int n = 0; n < CT; ++n)
#pragma unroll
        for (int t = 0; t < TQ; ++t) qd[n][TQ * w + t][lane] = sum[n][t];
      share(c ? c - 1 : 0);
      lds_barrier();
      products(c ? c - 1 : 0);
      lds_barrier();
      leave(c ? c - 1 : 0);
    }
    return;
  }

  // A zero that the compiler does not know: these addresses are not kept for both kinds of waves (scalar registers).
  int32_t zero = 0;
  asm volatile("" : "+s"(zero));
  rows += zero, tf += zero;
  const int part = L::part(w), rows0 = L::rows0(w);
  const bool keeper = L::kParts == 4 || w < L::kParts;
  u4 kx[KB][L::kRows][NI], kc[2 * KB][2][NI], tx[2][3];
  f4 into, rest, beta;
  float whole = 0.0f, whole_now;
  auto load_k_of = [&](int32_t c, int i) {
#pragma unroll
    for (int m = 0; m < L::kRows; ++m)
      load_frag(kf + c * (int64_t)(4 * KS * NI * 64) + ((rows0 + m) * KS + part * KB + i) * (NI * 64), lane, kx[i][m]);
  };
  auto load_kc_of = [&](int32_t c, int s) {
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
      load_frag(kt + c * (int64_t)(DK / 16 * 2 * NI * 64) + ((2 * KB * part + t) * 2 + s) * (NI * 64), lane, kc[t][s]);
  };
  auto load_k = [&](int32_t c) {
#pragma unroll
    for (int i = 0; i < KB; ++i) load_k_of(c, i);
  };
  auto load_kc = [&](int32_t c) {
    load_kc_of(c, 0);
    load_kc_of(c, 1);
  };
  auto load_rest = [&](int32_t c) {
    const float* r = rows + c * (int64_t)(kRowFields * kC);
    whole = r[4 * kC];
    rest = *reinterpret_cast<const f4*>(r + kC + row);
  };
  auto load_t = [&](int32_t c) {
    const float* r = rows + c * (int64_t)(kRowFields * kC);
    into = *reinterpret_cast<const f4*>(r + row);
    beta = *reinterpret_cast<const f4*>(r + 2 * kC + row);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s >= w / 2) load_frag(tf + c * (int64_t)(kTri * 3 * 64) + upper_frag(w, s) * (3 * 64), lane, tx[s]);
  };

  f4 ds[CT][2 * KB];
#pragma unroll
  for (int n = 0; n < CT; ++n)
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t d = 32 * KB * part + 16 * t + 4 * g + e;
        ds[n][t][e] = a.dfinal_states && dv + 16 * n < dim && d < a.key_dim
                          ? a.dfinal_states[(at.head * a.key_dim + d) * a.value_dim + dv + 16 * n]
                          : 0.0f;
      }
  float* dsp = p.ds + at.head * (int64_t)N * (DK * (int64_t)p.dvp) + 32 * KB * part * (int64_t)p.dvp + at.dv0;
  float* drp = p.dr + at.head * (int64_t)N * (kC * (int64_t)p.dvp) + 16 * w * (int64_t)p.dvp + at.dv0;
  const uint32_t kept = 4 * g * p.dvp + col;
  uint32_t ld = p.dvp;
  const int64_t stride = a.heads * a.value_dim;
  T* dvo = static_cast<T*>(a.dv) + (b * a.seqlen + row) * stride + h * a.value_dim + dv;
  if constexpr (AHEAD) {
    load_k(N - 1);
    load_kc(N - 1);
  }
  load_rest(N - 1);
  load_t(N - 1);
  lds_barrier();  // the waves beside the chain begin with the last chunk's dO
  for (int32_t c = N - 1; c >= 0; --c) {
    const int32_t next = c ? c - 1 : 0;
    asm volatile("" : "+s"(ld));
    {
      f4 x[CT][L::kRows] = {};
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        if constexpr (!AHEAD) load_k_of(c, i);
#pragma unroll
        for (int n = 0; n < CT; ++n) {
          u4 sb[3];
          split8<3>(ds[n][2 * i], ds[n][2 * i + 1], sb);
#pragma unroll
          for (int m = 0; m < L::kRows; ++m) x[n][m] = mac<2>(kx[i][m], sb, x[n][m]);
        }
      }
#pragma unroll
      for (int n = 0; n < CT; ++n)
#pragma unroll
        for (int m = 0; m < L::kRows; ++m) red[n][part][rows0 + m][lane] = x[n][m];
    }
    if (keeper) {
      float* to = dsp + c * (DK * (int64_t)p.dvp);
#pragma unroll
      for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* line = to + (16 * t + e) * ld;
#pragma unroll
          for (int n = 0; n < CT; ++n) (line + 16 * n)[kept] = ds[n][t][e];
        }
    }
    if constexpr (AHEAD) load_k(next);
    whole_now = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(whole)));
    lds_barrier();
#pragma unroll
    for (int n = 0; n < CT; ++n) {
      f4 y = red[n][0][w][lane];
#pragma unroll
      for (int j = 1; j < L::kParts; ++j) y += red[n][j][w][lane];
      const f4 o = pd[n][w][lane];
      f4 z;
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = fmaf(rest[e], y[e], o[e]);
      if (whole_now == 0.0f)  // a reset or padding: rows that do not reach the end
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = rest[e] != 0.0f ? z[e] : o[e];
      u2 half[3];
      split4<3>(z, half);
      store_half<3>(&ub[n][w / 2][0][lane], w & 1, half);
    }
    load_rest(next);
    lds_barrier();
    f4 r[CT];
#pragma unroll
    for (int n = 0; n < CT; ++n) {
      f4 r1 = {0, 0, 0, 0};
      u4 u[3];
      r[n] = f4{0, 0, 0, 0};
      load_frag(&ub[n][1][0][0], lane, u);
      r[n] = mac<2>(tx[1], u, r[n]);
      if (w < 2) {
        load_frag(&ub[n][0][0][0], lane, u);
        r1 = mac<2>(tx[0], u, r1);
      }
      r[n] += r1;
    }
    if (any_not_finite(r))
#pragma unroll
      for (int n = 0; n < CT; ++n)
        r[n] = sum_apart<true, false, 2>(tx, ub[n], lane, w / 2, 1, f4{0, 0, 0, 0}, runs_of(c), row);
#pragma unroll
    for (int n = 0; n < CT; ++n) {
      f4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = -beta[e] * into[e] * r[n][e];
      if (whole_now == 0.0f)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = into[e] != 0.0f ? x[e] : 0.0f;
      u2 half[3];
      split4<3>(x, half);
      store_half<3>(&rb[n][w / 2][0][lane], w & 1, half);
      float* to = drp + c * (kC * (int64_t)p.dvp) + 16 * n;
#pragma unroll
      for (int e = 0; e < 4; ++e) (to + e * ld)[kept] = r[n][e];
      if (dv + 16 * n < dim) {
        T* out = dvo + c * (kC * stride) + 16 * n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c * kC + row + e < seqlen) out[e * stride] = (T)(beta[e] != 0.0f ? beta[e] * r[n][e] : 0.0f);
      }
    }
    load_t(next);
#pragma unroll
    for (int n = 0; n < CT; ++n)
#pragma unroll
      for (int t = 0; t < 2 * KB; ++t) {
        ds[n][t] *= whole_now;
        if (whole_now == 0.0f) ds[n][t] = f4{0, 0, 0, 0};
      }
    lds_barrier();
#pragma unroll
    for (int n = 0; n < CT; ++n)
#pragma unroll
      for (int t = 0; t < 2 * KB; ++t) ds[n][t] += qd[n][2 * KB * part + t][lane];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (!AHEAD) load_kc_of(c, s);
#pragma unroll
      for (int n = 0; n < CT; ++n) {
        u4 x[3];
        load_frag(&rb[n][s][0][0], lane, x);
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t) ds[n][t] = mac<2>(kc[t][s], x, ds[n][t]);
      }
    }
    if constexpr (AHEAD) load_kc(next);
  }
  if (a.dinitial_states && keeper)
#pragma unroll
    for (int n = 0; n < CT; ++n)
      if (dv + 16 * n < dim)
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t d = 32 * KB * part + 16 * t + 4 * g + e;
            if (d < a.key_dim) a.dinitial_states[(at.head * a.key_dim + d) * a.value_dim + dv + 16 * n] = ds[n][t][e];
          }
}

// All chunks: dq, dk and, as sums over the keys' elements, what dbeta and dlog_decay need, from S0, U, dS1 and dR. A
// workgroup has a chunk of a key head, 64 or 128 of the keys' elements, and goes through the heads that share
// the key, so that their gradients are added in fp32 and in order. A wave has 16 of the elements as rows and the
// chunk's rows as columns. The sum over the value columns goes by 32: their operands are requested while the products
// of those before are made; dR, U and dO pass LDS as fragments, S0 and dS1 go to the wave that has their rows.
// Eight waves a workgroup, but four for small heads, of which a CU holds two workgroups, and in fp32, for the registers: keys
// of 64 at B=2 T=8192, 16 heads 423 -> 300 us, keys of 128 at B=4 T=4096, 16 heads with four waves 565, with eight 514.
// Bound by memory (1.23 GB read there, 255 us at a copy's rate) and by what does not run beside it: VALUs are
// 23 %, matrix cores 15 % and LDS 14 % busy, in turn more than at once.
template <typename T, int DK>
constexpr int kGradWaves = DK < 128 || sizeof(T) == 4 ? 4 : 8;
template <typename T, int DK>
constexpr int kGradParts = DK / 16 / kGradWaves<T, DK>;

// What a row's gates' gradients are made of: k.z, q.dq - k.c, dR.V; and of its chunk, what the end's sum has.
struct GateSums {
  float kz, other, rv, end;
};
constexpr int kGateFields = 4;

// What the kernels of the gradients take: 32-bit sizes and no more than they use, for the scalar registers.
struct GradArgs {
  const u4 *kf, *qf, *kt, *qt;
  const float *rows, *s0, *u, *ds, *dr;
  float* gates;
  const void *v, *dout;
  int64_t v_stride_b, v_stride_t, v_stride_h, dout_stride_b, dout_stride_t, dout_stride_h;
  void *dq, *dk, *dlog_decay, *dbeta;
  float scale;
  int32_t units, chunks, group, key_heads, heads, seqlen, key_dim, value_dim, dvp, log_decay_dtype, beta_dtype;
};

// dbeta and dlog_decay of row `lane` of a head's chunk, in a wave. A row that resets the state has no gradient of
// its decay.
__device__ __forceinline__ void finish_gates(const GradArgs& p, int64_t b, int c, int h, int lane, const float* rows,
                                             const GateSums& x) {
  const float beta = rows[2 * kC + lane];
  const bool live = rows[3 * kC + lane] != 0.0f;
  const int run = reinterpret_cast<const int*>(rows + 7 * kC)[lane];
  const int before = __shfl_up(run, 1);
  const bool reset = run != (lane ? before : 0);
  double s = (double)x.other - (double)beta * (double)x.kz + (lane == 63 ? (double)x.end : 0.0);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_down(s, d);
    const int r = __shfl_down(run, d);
    if (lane + d < 64 && r == run) s += o;
  }
  const int t = c * kC + lane;
  const int64_t o = (b * p.seqlen + t) * p.heads + h;
  if (t < p.seqlen) {
    store_as(p.dlog_decay, o, p.log_decay_dtype, live && !reset ? (float)s : 0.0f);
    store_as(p.dbeta, o, p.beta_dtype, live ? x.rv - x.kz : 0.0f);
  }
}

// The same where the keys' elements lie in several workgroups; a wave has a head's chunk.
template <int PARTS>
__global__ __launch_bounds__(256) void delta_gates_kernel(GradArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t hc = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (hc >= (int64_t)p.units * p.group) return;
  const int64_t head = hc / p.chunks, b = head / p.heads;
  GateSums x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const float* from = p.gates + (hc * PARTS + i) * (kGateFields * kC) + lane;
    x.kz += from[0], x.other += from[kC], x.end += from[3 * kC];
    if (i == 0) x.rv = from[2 * kC];  // each part has it
  }
  finish_gates(p, b, (int)(hc - head * p.chunks), (int)(head - b * p.heads), lane, p.rows + hc * (kRowFields * kC), x);
}

// Eight elements of a row, at `p` and 16 further on, as they lie in memory.
template <typename T>
struct RawRow {
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 lo, hi;
  __device__ __forceinline__ void load(const T* p, int left) {  // so many elements from p on
    if (left >= 32) {
      __builtin_memcpy(&lo, p, sizeof lo);
      __builtin_memcpy(&hi, p + 16, sizeof hi);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = e < left ? p[e] : (T)0.0f;
        hi[e] = e + 16 < left ? p[e + 16] : (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ f4 low() const { return f4{to_f32(lo[0]), to_f32(lo[1]), to_f32(lo[2]), to_f32(lo[3])}; }
  __device__ __forceinline__ f4 high() const { return f4{to_f32(hi[0]), to_f32(hi[1]), to_f32(hi[2]), to_f32(hi[3])}; }
};

template <typename T, int DK>
__global__ __launch_bounds__((kGradWaves<T, DK>) * 64, kPieces<T> > 1 ? 1 : 2) void delta_grad_kernel(GradArgs p) {
  constexpr int NI = kPieces<T>, KS = DK / 32, NW = kGradWaves<T, DK>, LG = 68, PAIRS = (10 + NW - 1) / NW;
  // fragments: dR, U, dO of 32 value columns; then those of the products between rows
  __shared__ u4 f[12][3][64];
  __shared__ float gl[kC * LG], rows[kRowFields * kC];
  __shared__ float sums[NW][2][kC], vsum[kC], tail[NW];
  const int w = wave_index(), wr = w & 3;
  // The parts of a chunk go to one XCD, whose L2 they share.
  const int slot = blockIdx.x >> 3, kc = slot / kGradParts<T, DK> * 8 + (blockIdx.x & 7);
  if (kc >= p.units) return;
  const int part = slot % kGradParts<T, DK>, tile = part * NW + w;  // the wave's elements: 16 tile ...
  const int bk = kc / p.chunks, c = kc - bk * p.chunks, b = bk / p.key_heads, kh = bk - b * p.key_heads;
  const int t0 = c * kC;
  const u4* kf0 = p.kf + (int64_t)kc * (4 * KS * NI * 64);
  const u4* qf0 = p.qf + (int64_t)kc * (4 * KS * NI * 64);
  const u4* kt0 = p.kt + (int64_t)kc * (DK / 16 * 2 * NI * 64);
  const u4* qt0 = p.qt + (int64_t)kc * (DK / 16 * 2 * NI * 64);
  const double* sum = reinterpret_cast<const double*>(rows + 5 * kC);
  const int* run = reinterpret_cast<const int*>(rows + 7 * kC);
  f4 dq[4] = {}, dk[4] = {};
  // The tiles (m, n) of the products between rows that a wave has, n <= m: of ten, those of its number and every NW
  // further.
  struct Pair {
    int m, n;
    __device__ __forceinline__ Pair(int x) {
      asm volatile("" : "+s"(x));  // made where it is used: scalar registers
      m = x < 1 ? 0 : x < 3 ? 1 : x < 6 ? 2 : 3;
      n = x - m * (m + 1) / 2;
    }
  };

  for (int h = kh * p.group; h < (kh + 1) * p.group; ++h) {
    const int64_t hc = (int64_t)(b * p.heads + h) * p.chunks + c;
    // Addresses are made and k's and q's fragments read anew for every head: kept, they would spill.
    uint32_t lane = threadIdx.x & 63;
    // (Not the pointers themselves, of which it would not know then that they are no LDS: flat loads.)
    int32_t zero = 0;
    asm volatile("" : "+s"(zero), "+v"(lane));
    const u4 *kf = kf0 + zero, *qf = qf0 + zero, *kt = kt0 + zero, *qt = qt0 + zero;
    const uint32_t col = lane & 15, g = lane >> 4;
    const int mine = 16 * wr + col;  // the row whose dR and V, or U and dO, the lane reads (four waves: all)
    const int64_t mine_t = min(t0 + mine, p.seqlen - 1);
    const float* s0 = p.s0 + hc * ((int64_t)DK * p.dvp) + (16 * tile + col) * p.dvp + 4 * g;
    const float* ds = p.ds + hc * ((int64_t)DK * p.dvp) + (16 * tile + col) * p.dvp + 4 * g;
    const float* up = p.u + hc * (kC * (int64_t)p.dvp) + mine * p.dvp + 4 * g;
    const float* rp = p.dr + hc * (kC * (int64_t)p.dvp) + mine * p.dvp + 4 * g;
    const T* vp = static_cast<const T*>(p.v) + b * p.v_stride_b + mine_t * p.v_stride_t + h * p.v_stride_h + 4 * g;
    const T* op = static_cast<const T*>(p.dout) + b * p.dout_stride_b + mine_t * p.dout_stride_t + h * p.dout_stride_h +
                  4 * g;
    f4 xr[2], xu[2], xs[2], xd[2];
    RawRow<T> xo, xv;
    auto load = [&](int d0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (NW == 4 || w < 4) xr[i] = *reinterpret_cast<const f4*>(rp + d0 + 16 * i);
        if (NW == 4 || w >= 4) xu[i] = *reinterpret_cast<const f4*>(up + d0 + 16 * i);
        xs[i] = *reinterpret_cast<const f4*>(s0 + d0 + 16 * i);
        xd[i] = *reinterpret_cast<const f4*>(ds + d0 + 16 * i);
      }
      const int left = p.value_dim - d0 >= 32 ? 32 : p.value_dim - d0 - 4 * (int)g;
      if (NW == 4 || w >= 4) xo.load(op + d0, left);
      if (NW == 4 || w < 4) xv.load(vp + d0, left);
    };
    load(0);
    if (threadIdx.x < kRowFields * kC / 4)
      reinterpret_cast<f4*>(rows)[threadIdx.x] =
          reinterpret_cast<const f4*>(p.rows + hc * (kRowFields * kC))[threadIdx.x];
    lds_barrier();
    const bool live = rows[3 * kC + mine] != 0.0f;
    f4 aq[4] = {}, az[4] = {}, ac[4] = {}, go[PAIRS] = {}, gr[PAIRS] = {};
    float through = 0.0f, along = 0.0f;  // <dS1, S0> and dR.V of the lane's elements
    for (int d0 = 0; d0 < p.dvp; d0 += 32) {
      lds_barrier();
      u4 sf[3], df[3];
      if (NW == 4 || w < 4) {
        u4 x[3];
        split8<3>(xr[0], xr[1], x);
#pragma unroll
        for (int n = 0; n < 3; ++n) f[wr][n][lane] = x[n];
        const f4 lo = xv.low(), hi = xv.high();
        if (live)
#pragma unroll
          for (int e = 0; e < 4; ++e) along = fmaf(xr[0][e], lo[e], fmaf(xr[1][e], hi[e], along));
      }
      if (NW == 4 || w >= 4) {
        u4 x[3], y[NI];
        split8<3>(xu[0], xu[1], x);
#pragma unroll
        for (int n = 0; n < 3; ++n) f[4 + wr][n][lane] = x[n];
        f4 lo = xo.low(), hi = xo.high();
        if (!live) lo = hi = f4{0, 0, 0, 0};
        split8<NI>(lo, hi, y);
#pragma unroll
        for (int n = 0; n < NI; ++n) f[8 + wr][n][lane] = y[n];
      }
      split8<3>(xs[0], xs[1], sf);
      split8<3>(xd[0], xd[1], df);
#pragma unroll
      for (int e = 0; e < 4; ++e) through = fmaf(xs[0][e], xd[0][e], fmaf(xs[1][e], xd[1][e], through));
      if (d0 + 32 < p.dvp) load(d0 + 32);
      lds_barrier();
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        __builtin_amdgcn_sched_barrier(0);  // a tile's operands at a time: registers
        u4 x3[3], y[NI];
        load_frag(&f[m][0][0], lane, x3);
        az[m] = mac<2>(sf, x3, az[m]);
        load_frag(&f[8 + m][0][0], lane, y);
        aq[m] = mac<2>(sf, y, aq[m]);
        load_frag(&f[4 + m][0][0], lane, x3);
        ac[m] = mac<2>(df, x3, ac[m]);
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i)
        if (w + NW * i < 10) {
          const Pair t(w + NW * i);
          __builtin_amdgcn_sched_barrier(0);
          u4 un[3], x3[3], y[NI];
          load_frag(&f[4 + t.n][0][0], lane, un);
          load_frag(&f[8 + t.m][0][0], lane, y);
          go[i] = mac<2>(un, y, go[i]);
          load_frag(&f[t.m][0][0], lane, x3);
          gr[i] = mac<2>(un, x3, gr[i]);
        }
    }
    // The factors of the columns, and k.(state's part of c).
    float state_part = 0.0f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const float into = rows[16 * m + col], rest = rows[kC + 16 * m + col];
      u4 kv[NI];
      load_frag(kf + (m * KS + tile / 2) * (NI * 64), lane, kv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        aq[m][e] = into != 0.0f ? p.scale * into * aq[m][e] : 0.0f;
        az[m][e] = into != 0.0f ? into * az[m][e] : 0.0f;
        ac[m][e] = rest != 0.0f ? rest * ac[m][e] : 0.0f;
        state_part = fmaf(piece_sum(kv, tile & 1, e), ac[m][e], state_part);
      }
    }
    // Two rounds over the products between rows: scale D dO.U^T for dq and dk, D dR.U^T for z and dk.
#pragma unroll
    for (int round = 0; round < 2; ++round) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i)
        if (w + NW * i < 10) {
          const Pair t(w + NW * i);
          const int r = 16 * t.m + col, j0 = 16 * t.n + 4 * g, run_r = run[r];
          const double sum_r = sum[r];
          f4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + e;
            const bool seen = (round ? j < r : j <= r) & (run_r == run[j]);
            const float d = exp2_of(sum_r - sum[j]), y = round ? d * gr[i][e] : p.scale * d * go[i][e];
            x[e] = seen ? y : 0.0f;
          }
          *reinterpret_cast<f4*>(&gl[r * LG + 16 * t.n + 4 * g]) = x;
        }
      lds_barrier();
      // fragments 0..5: sum over j, columns i (lower); 6..11: sum over i, columns j (upper)
#pragma unroll 1
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
            if (round) {  // not zero times the rate of a spoilt row, which is NaN
              lo[e] = lo[e] != 0.0f ? lo[e] * -rows[2 * kC + i] : 0.0f;
              hi[e] = hi[e] != 0.0f ? hi[e] * -rows[2 * kC + i + 16] : 0.0f;
            }
          }
        }
        u4 y[3];
        split8<3>(lo, hi, y);
#pragma unroll
        for (int n = 0; n < 3; ++n) f[job][n][lane] = y[n];
      }
      lds_barrier();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u4 kx[NI], qx[NI];
        load_frag(kt + (tile * 2 + s) * (NI * 64), lane, kx);
        if (round == 0) load_frag(qt + (tile * 2 + s) * (NI * 64), lane, qx);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          __builtin_amdgcn_sched_barrier(0);
          u4 x3[3];
          if (s <= m / 2) {
            load_frag(&f[lower_frag(m, s)][0][0], lane, x3);
            if (round == 0) aq[m] = mac<2>(kx, x3, aq[m]);
            else az[m] = mac<2>(kx, x3, az[m]);
          }
          if (s >= m / 2) {
            load_frag(&f[6 + upper_frag(m, s)][0][0], lane, x3);
            if (round == 0) ac[m] = mac<2>(qx, x3, ac[m]);
            else ac[m] = mac<2>(kx, x3, ac[m]);
          }
        }
      }
      if (round == 0) lds_barrier();
    }
    // Sums over the keys' elements: k.z, and q.dq - k.c.
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float kz = 0.0f, rest = 0.0f;
      const float beta = rows[2 * kC + 16 * m + col];
      u4 kv[NI], qv[NI];
      load_frag(kf + (m * KS + tile / 2) * (NI * 64), lane, kv);
      load_frag(qf + (m * KS + tile / 2) * (NI * 64), lane, qv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float k = piece_sum(kv, tile & 1, e), q = piece_sum(qv, tile & 1, e);
        kz = fmaf(k, az[m][e], kz);
        rest = fmaf(q, aq[m][e], fmaf(-k, ac[m][e], rest));
        dk[m][e] += ac[m][e] - beta * az[m][e];
      }
      dq[m] += aq[m];
      kz += __shfl_xor(kz, 16), rest += __shfl_xor(rest, 16);
      kz += __shfl_xor(kz, 32), rest += __shfl_xor(rest, 32);
      if (g == 0) sums[w][0][16 * m + col] = kz, sums[w][1][16 * m + col] = rest;
    }
    along += __shfl_xor(along, 16);
    along += __shfl_xor(along, 32);
    if (g == 0 && w < 4) vsum[mine] = along;
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
        finish_gates(p, b, c, h, lane, rows, x);
      } else {
        float* to = p.gates + (hc * kGradParts<T, DK> + part) * (kGateFields * kC) + lane;
        to[0] = x.kz, to[kC] = x.other, to[2 * kC] = x.rv, to[3 * kC] = x.end;
      }
    }
    lds_barrier();
  }
  const uint32_t col = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int i = 16 * m + col;
    if (t0 + i >= p.seqlen) continue;
    const bool live = rows[3 * kC + i] != 0.0f;
    const int64_t row = (((int64_t)b * p.seqlen + t0 + i) * p.key_heads + kh) * p.key_dim;
    const int d = 16 * tile + 4 * g;
    if (d >= p.key_dim) continue;
    const f4 none = {0, 0, 0, 0};
    store4(static_cast<T*>(p.dq) + row + d, live ? dq[m] : none, p.key_dim - d);
    store4(static_cast<T*>(p.dk) + row + d, live ? dk[m] : none, p.key_dim - d);
  }
}

// Two tiles of columns a workgroup where one each would be more workgroups than CUs, and the registers hold them: at B=4
// T=4096, 16 heads of 128 (512 tiles) forward 376 -> 274 us, backward 405 -> 290. A chunk then takes 2.2 times as long
// (a prompt of 16384, 128 tiles: 2.0 us a chunk; 4.3 there), so with up to 256 tiles one each is quicker.
template <typename T, int DK, int CT>
hipError_t delta_chain(const DeltaParams& p, bool backward, hipStream_t s) {
  const int64_t grid = delta_chains(p.a, p.tiles / CT);
  if (backward) return start(&delta_bwd_kernel<T, DK, CT>, grid, 512, s, p);
  return p.s0 ? start(&delta_fwd_kernel<T, DK, CT, true>, grid, 512, s, p)
              : start(&delta_fwd_kernel<T, DK, CT, false>, grid, 512, s, p);
}

template <typename T, int DK>
hipError_t delta_launch_dk(const DeltaParams& p, bool backward, hipStream_t s) {
  const ccv1d_delta_args& a = p.a;
  const int64_t chunks = a.batch * a.key_heads * p.chunks;
  const int64_t prep = chunks * (p.group / p.prep_heads);
  hipError_t e = backward ? start(&delta_prep_kernel<T, DK, true>, prep, 256, s, p)
                          : start(&delta_prep_kernel<T, DK, false>, prep, 256, s, p);
  if (e != hipSuccess) return e;
  constexpr int CT = kPieces<T> * DK <= 128 ? 2 : 1;
  e = CT > 1 && a.batch * a.heads * p.tiles > 256 ? delta_chain<T, DK, CT>(p, backward, s)
                                                  : delta_chain<T, DK, 1>(p, backward, s);
  if (e != hipSuccess || !backward) return e;
  const GradArgs ga = {p.kf, p.qf, p.kt, p.qt, p.rows, p.s0, p.u, p.ds, p.dr, p.gates, a.v, a.dout,
                       a.v_stride_b, a.v_stride_t, a.v_stride_h, a.dout_stride_b, a.dout_stride_t, a.dout_stride_h,
                       a.dq, a.dk, a.dlog_decay, a.dbeta, a.scale, (int32_t)chunks, p.chunks, p.group,
                       (int32_t)a.key_heads, (int32_t)a.heads, (int32_t)a.seqlen, (int32_t)a.key_dim,
                       (int32_t)a.value_dim, p.dvp, a.log_decay_dtype, a.beta_dtype};
  e = start(&delta_grad_kernel<T, DK>, (chunks + 7) / 8 * 8 * kGradParts<T, DK>, kGradWaves<T, DK> * 64, s, ga);
  if constexpr (kGradParts<T, DK> > 1)
    if (e == hipSuccess)
      e = start(&delta_gates_kernel<(kGradParts<T, DK>)>, (a.batch * a.heads * p.chunks + 3) / 4, 256, s, ga);
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

// The gated linear recurrence in one pass over its inputs, forward and backward.
//
// h[t] = f[t] h[t-1] + u[t] is cut along time into chunks of kRecWaves waves of R rows, a workgroup
// each; a lane holds the factors of its R rows and CPL channels in registers. A stretch of rows acts
// on the state before it as h -> A h + H, and such pairs combine: every wave forms the pair of its
// rows, the workgroup that of its chunk, and once the state in front of a wave is known it walks its
// rows again from there, from registers. So each input is read once and each output written once.
//
// The state in front of a chunk comes from the chunks before it, whose workgroups run at the same time
// on other CUs, through words in the workspace:
//   * every chunk publishes its own pair as soon as it has it;
//   * chunks form groups of kRecGroup, and the last chunk of a group publishes the state after it;
//   * a chunk takes the state after the group before its own and the pairs of the chunks between, at
//     most kRecGroup - 1, and combines them in order, so results do not depend on timing.
// A word holds its own ready mark (the sign bit of A, which is never negative; the workspace is
// cleared before), so an atomic load of 64 bits that shows the mark shows the whole word, and no fence
// or flag is needed across the caches of the XCDs. Chunks are dealt by a ticket in order of time
// (backward: from the end), not by workgroup number: a chunk waits only for words of chunks with lower
// tickets, whose workgroups have therefore started, and these publish their pairs before they wait for
// anything. The one wait on a wait is the state after a group, and by induction over tickets that ends too.
//
// A sequence's first row and padding cut the state: the row's factor is no number times zero but a
// branch (an infinity of one sequence never meets the next), and A = 0 says that a stretch contains
// one. A product of factors that underflows is held at the smallest normal number, so that zero
// means nothing else and an infinity still passes.
//
// Bytes of forward: x, gate, input_gate read, out written; backward: these and dout read, three
// gradients written. Backward makes the states again from the one in front of each chunk, which the
// forward keeps in fp32: 4 B per channel and 64 rows against 2 B per element for reading out, and
// without out's rounding.
#pragma once

#include "../ccv1d_device.h"
#include "ops_rec_math.h"

namespace ccv1d {
namespace ops {

constexpr int kRecWaves = 8;
constexpr int kRecGroup = 16;
constexpr uint32_t kReady = 0x80000000u;
constexpr float kTiny = 1.17549435e-38f;

struct RecParams {
  ccv1d_rec_args a;
  int32_t cols, chunks, groups;  // wave columns of 64 * CPL channels; chunks along time; their groups
  uint64_t* pairs;               // (batch, chunks, dim)
  uint64_t* states;              // (batch, groups, dim): word of the state after a group
  uint32_t* ticket;
  float* part;  // backward: (batch, chunks, dim) sums behind ddecay
};

__device__ __forceinline__ void publish(uint64_t* at, float A, float H) {
  const uint64_t v = ((uint64_t)__float_as_uint(H) << 32) | (__float_as_uint(A) | kReady);
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint64_t peek(const uint64_t* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint64_t await(const uint64_t* at, uint64_t v) {
  while (!((uint32_t)v & kReady)) {
    __builtin_amdgcn_s_sleep(1);
    v = peek(at);
  }
  return v;
}

// The pair (A, H) after the pair (A0, H0), or after a state: A = 0 cuts.
__device__ __forceinline__ float after(float h, float A, float H) {
  return A == 0.0f ? H : fmaf(A, h, H);
}
__device__ __forceinline__ float product(float A0, float A) {
  return A == 0.0f || A0 == 0.0f ? 0.0f : fmaxf(A0 * A, kTiny);
}

// The rows of one wave that are not plain: bit j of each mask is row t0 + j.
struct Rows {
  uint32_t first, pad;  // a sequence's first row; padding
  int valid;            // rows inside the sequence, from 0 to R
};

template <int R>
__device__ __forceinline__ Rows rows_of(const int32_t* seq, int64_t t0, int64_t T, int lane) {
  Rows w{0, 0, (int)max((int64_t)0, min((int64_t)R, T - t0))};
  if (seq && w.valid > 0) {  // lane l looks at row t0 - 1 + l
    const int64_t t = t0 - 1 + lane;
    const int32_t id = seq[min(max(t, (int64_t)0), T - 1)];
    const int32_t prev = __shfl_up(id, 1);
    const uint64_t pad = __ballot(id < 0);
    const uint64_t first = __ballot(t > 0 && id != prev);
    const uint32_t live = (1u << w.valid) - 1;
    w.pad = (uint32_t)(pad >> 1) & live;
    w.first = (uint32_t)(first >> 1) & live;
  }
  return w;
}

// Deals a chunk to this workgroup: (batch row and wave column, chunk from the walk's start).
__device__ __forceinline__ void deal(const RecParams& p, int& bc, int& chunk, uint32_t* s_ticket) {
  const uint32_t n = (uint32_t)(p.a.batch * p.cols);
  uint32_t k = blockIdx.x;
  if (p.chunks > 1) {
    if (threadIdx.x == 0)
      *s_ticket = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    k = __builtin_amdgcn_readfirstlane(*s_ticket);
  }
  chunk = (int)(k / n);
  bc = (int)(k % n);
}

// The pairs of the waves of a workgroup, and of the chunks before it, in LDS.
template <int CPL>
struct Pairs {
  float A[kRecWaves][CPL][kWave], H[kRecWaves][CPL][kWave];
};

// Combines the chunks between the group before and this chunk: wave w the two from 2 w on, into `got`;
// the state in front of the group goes to `base`. `chunk` counts from the walk's start.
template <int CPL>
__device__ __forceinline__ void look_back(const RecParams& p, int64_t b, int64_t c, int chunk, int dir,
                                          const float (&start)[CPL], Pairs<CPL>& got,
                                          float (&base)[CPL][kWave], int wave, int lane) {
  const int64_t D = p.a.dim;
  const int g = chunk / kRecGroup, j0 = g * kRecGroup;
  auto word = [&](int j) {  // chunks are stored in order of time
    const int64_t at = dir > 0 ? j : p.chunks - 1 - j;
    return p.pairs + (b * p.chunks + at) * D + c;
  };
  const int j = j0 + 2 * wave;
  uint64_t v[2][CPL], s[CPL];
  const uint64_t* gs = p.states + (b * p.groups + (g - 1)) * D + c;
#pragma unroll
  for (int i = 0; i < CPL; ++i) {  // requested together
    if (j < chunk) v[0][i] = peek(word(j) + i);
    if (j + 1 < chunk) v[1][i] = peek(word(j + 1) + i);
    if (wave == 0 && g > 0) s[i] = peek(gs + i);
  }
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    float A = 1.0f, H = 0.0f;
    if (j < chunk) {
      const uint64_t w = await(word(j) + i, v[0][i]);
      A = __uint_as_float((uint32_t)w & ~kReady);
      H = __uint_as_float((uint32_t)(w >> 32));
    }
    if (j + 1 < chunk) {
      const uint64_t w = await(word(j + 1) + i, v[1][i]);
      const float A1 = __uint_as_float((uint32_t)w & ~kReady);
      H = after(H, A1, __uint_as_float((uint32_t)(w >> 32)));
      A = product(A, A1);
    }
    got.A[wave][i][lane] = A;
    got.H[wave][i][lane] = H;
    if (wave == 0)
      base[i][lane] = g > 0 ? __uint_as_float((uint32_t)(await(gs + i, s[i]) >> 32)) : start[i];
  }
}

// ------------------------------------------------------------------------------------- forward

template <typename T, int CPL, bool DECAY, bool IG, int R>
__global__ __launch_bounds__(kRecWaves* kWave, 4) void rec_fwd_kernel(RecParams p) {
  using V = VecIO<T, CPL>;
  __shared__ Pairs<CPL> mine, got;
  __shared__ float base[CPL][kWave];
  __shared__ uint32_t s_ticket;
  const ccv1d_rec_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bc, chunk;
  deal(p, bc, chunk, &s_ticket);
  const int64_t b = bc / p.cols, T_ = a.seqlen, D = a.dim;
  const int64_t t0 = ((int64_t)chunk * kRecWaves + wave) * R;
  // The last lanes of a row share its last CPL channels and compute the same values twice.
  const int64_t c = min((int64_t)((bc % p.cols) * kWave + lane) * CPL, D - CPL);
  const int32_t* seq = a.seq_idx ? a.seq_idx + b * T_ : nullptr;
  const Rows rows = rows_of<R>(seq, t0, T_, lane);

  const T* xp = static_cast<const T*>(a.x) + b * a.x_stride_b;
  const T* gp = static_cast<const T*>(a.gate) + b * a.gate_stride_b;
  const T* ip = IG ? static_cast<const T*>(a.input_gate) + b * a.input_gate_stride_b : nullptr;
  typename V::raw xr[R], gr[R], ir[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t t = min(t0 + j, T_ - 1);
    gr[j] = V::ld(gp + t * a.gate_stride_t + c);
    xr[j] = V::ld(xp + t * a.x_stride_t + c);
    if constexpr (IG) ir[j] = V::ld(ip + t * a.input_gate_stride_t + c);
  }
  float k[CPL], start[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    k[i] = DECAY ? decay_rate(a.decay[c + i], a.decay_scale) : 0.0f;
    start[i] = a.initial_states ? a.initial_states[b * D + c + i] : 0.0f;
  }

  float f[R][CPL], u[R][CPL], A[CPL], H[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) A[i] = 1.0f, H[i] = 0.0f;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float x[CPL], g[CPL], ig[CPL];
    V::unpack(xr[j], x);
    V::unpack(gr[j], g);
    if constexpr (IG) V::unpack(ir[j], ig);
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      float beta;
      forget<T, DECAY>(k[i], g[i], f[j][i], beta);
      u[j][i] = beta * x[i];
      if constexpr (IG) u[j][i] *= sigmoid<T>(ig[i]);
    }
  }
  const uint32_t cut = rows.first | rows.pad;
  const bool plain = cut == 0 && rows.valid == R;
  if (plain) {
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        H[i] = fmaf(f[j][i], H[i], u[j][i]);
        A[i] *= f[j][i];
      }
#pragma unroll
    for (int i = 0; i < CPL; ++i) A[i] = fmaxf(A[i], kTiny);
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        if (j >= rows.valid) f[j][i] = 1.0f, u[j][i] = 0.0f;  // past the end: nothing happens
        if (rows.pad >> j & 1) u[j][i] = 0.0f;
        H[i] = cut >> j & 1 ? u[j][i] : fmaf(f[j][i], H[i], u[j][i]);
        A[i] *= f[j][i];
      }
#pragma unroll
    for (int i = 0; i < CPL; ++i) A[i] = cut ? 0.0f : fmaxf(A[i], kTiny);
  }
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    mine.A[wave][i][lane] = A[i];
    mine.H[wave][i][lane] = H[i];
  }
  __syncthreads();

  float h[CPL];
  if (p.chunks > 1) {
    if (wave == 0 && chunk + 1 < p.chunks) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float A0 = 1.0f, H0 = 0.0f;
#pragma unroll
        for (int w = 0; w < kRecWaves; ++w) {
          H0 = after(H0, mine.A[w][i][lane], mine.H[w][i][lane]);
          A0 = product(A0, mine.A[w][i][lane]);
        }
        publish(p.pairs + (b * p.chunks + chunk) * D + c + i, A0, H0);
      }
    }
    look_back<CPL>(p, b, c, chunk, 1, start, got, base, wave, lane);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      h[i] = base[i][lane];
      for (int w = 0; w < kRecWaves && chunk / kRecGroup * kRecGroup + 2 * w < chunk; ++w)
        h[i] = after(h[i], got.A[w][i][lane], got.H[w][i][lane]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < CPL; ++i) h[i] = start[i];
  }
#pragma unroll
  for (int i = 0; i < CPL; ++i)
    for (int w = 0; w < wave; ++w) h[i] = after(h[i], mine.A[w][i][lane], mine.H[w][i][lane]);
  if (wave == kRecWaves - 1 && chunk % kRecGroup == kRecGroup - 1 && chunk + 1 < p.chunks) {
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      publish(p.states + (b * p.groups + chunk / kRecGroup) * D + c + i, 0.0f, after(h[i], A[i], H[i]));
  }
  if (rows.valid == 0) return;
  if (a.saved && t0 % CCV1D_REC_SAVED_ROWS == 0) {
    const int64_t ns = (T_ + CCV1D_REC_SAVED_ROWS - 1) / CCV1D_REC_SAVED_ROWS;
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      a.saved[(b * ns + t0 / CCV1D_REC_SAVED_ROWS) * D + c + i] = h[i];
  }
  T* out = static_cast<T*>(a.out) + (b * T_ + t0) * D + c;
  if (plain) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) h[i] = fmaf(f[j][i], h[i], u[j][i]);
      V::st(out + j * D, V::pack(h));
    }
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (j < rows.valid) {
#pragma unroll
        for (int i = 0; i < CPL; ++i)
          h[i] = cut >> j & 1 ? u[j][i] : fmaf(f[j][i], h[i], u[j][i]);
        V::st(out + j * D, V::pack(h));
      }
    }
  }
  if (a.final_states && t0 + rows.valid == T_) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) a.final_states[b * D + c + i] = h[i];
  }
}

// ------------------------------------------------------------------------------------ backward
//
// dh[t] = dout[t] + f[t+1] dh[t+1]; what row t hands to the row before is c = f[t] (dout[t] + c'), so
// a stretch of rows acts on what reaches its end as c -> A c + G with the A of the forward. With
// m = h[t-1] - w (h[t-1] taken as zero where the state is cut):
//   dx = dh beta i, dinput_gate = dx x (1 - i)
//   with decay:     w = i x a / beta,  q = dh (ln a) a m,  dgate = q (1 - r),  ddecay from the sum of q
//                   (a / beta comes from d beta / d(ln a) = -a^2 / beta; 0 where a is exactly 1)
//   without decay:  w = i x,           dgate = dh a beta m

template <typename T, int CPL, bool DECAY, bool IG, int R>
__global__ __launch_bounds__(kRecWaves* kWave, 2) void rec_bwd_kernel(RecParams p) {
  using V = VecIO<T, CPL>;
  static_assert(kRecWaves * R == CCV1D_REC_SAVED_ROWS, "one saved state per chunk");
  __shared__ Pairs<CPL> mine, got;
  __shared__ float s_h[kRecWaves][CPL][kWave];
  __shared__ float base[CPL][kWave];
  __shared__ uint32_t s_ticket;
  const ccv1d_rec_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bc, from_end;
  deal(p, bc, from_end, &s_ticket);
  const int chunk = p.chunks - 1 - from_end;
  const int64_t b = bc / p.cols, T_ = a.seqlen, D = a.dim;
  const int64_t t0 = ((int64_t)chunk * kRecWaves + wave) * R;
  const int64_t c = min((int64_t)((bc % p.cols) * kWave + lane) * CPL, D - CPL);
  const int32_t* seq = a.seq_idx ? a.seq_idx + b * T_ : nullptr;
  const Rows rows = rows_of<R>(seq, t0, T_, lane);

  const T* xp = static_cast<const T*>(a.x) + b * a.x_stride_b;
  const T* gp = static_cast<const T*>(a.gate) + b * a.gate_stride_b;
  const T* ip = IG ? static_cast<const T*>(a.input_gate) + b * a.input_gate_stride_b : nullptr;
  const T* yp = static_cast<const T*>(a.dout) + b * a.dout_stride_b;
  typename V::raw xr[R], gr[R], ir[R], yr[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t t = min(t0 + j, T_ - 1);
    gr[j] = V::ld(gp + t * a.gate_stride_t + c);
    xr[j] = V::ld(xp + t * a.x_stride_t + c);
    if constexpr (IG) ir[j] = V::ld(ip + t * a.input_gate_stride_t + c);
    yr[j] = V::ld(yp + t * a.dout_stride_t + c);
  }
  float k[CPL], start[CPL], h[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    k[i] = DECAY ? decay_rate(a.decay[c + i], a.decay_scale) : 0.0f;
    start[i] = a.dfinal_states ? a.dfinal_states[b * D + c + i] : 0.0f;
    h[i] = a.saved[(b * p.chunks + chunk) * D + c + i];
  }

  const uint32_t cut = rows.first | rows.pad;
  const bool plain = cut == 0 && rows.valid == R;
  float f[R][CPL], bi[R][CPL];          // a; beta i
  float w[R][CPL];                      // then m
  float la[R][CPL], rest[R][CPL];       // decay: a ln a, 1 - r; else a beta
  float xi[R][CPL];                     // x (1 - i)
  float A[CPL], H[CPL], G[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) A[i] = 1.0f, H[i] = 0.0f, G[i] = 0.0f;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float x[CPL], g[CPL], ig[CPL];
    V::unpack(xr[j], x);
    V::unpack(gr[j], g);
    if constexpr (IG) V::unpack(ir[j], ig);
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      float in = 1.0f, not_in = 0.0f;
      if constexpr (IG) sigmoid_pair<T>(ig[i], in, not_in);
      if constexpr (DECAY) {
        float r;
        sigmoid_pair<T>(g[i], r, rest[j][i]);
        const float l = k[i] * r;
        const float av = __builtin_amdgcn_exp2f(l);
        const float s = one_minus_square(l, av);
        const float inv = s > 0.0f ? __builtin_amdgcn_rsqf(s) : s == 0.0f ? 0.0f : s;
        f[j][i] = av;
        bi[j][i] = s * inv * in;
        la[j][i] = kLn2 * l * av;
        w[j][i] = in * x[i] * av * inv;
      } else {
        float beta;
        sigmoid_pair<T>(g[i], f[j][i], beta);
        bi[j][i] = beta * in;
        la[j][i] = f[j][i] * beta;
        w[j][i] = in * x[i];
      }
      if constexpr (IG) xi[j][i] = x[i] * not_in;
    }
  }
  // Forward over the rows: the pair (A, H).
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float x[CPL];
    V::unpack(xr[j], x);
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      float u = bi[j][i] * x[i];
      if (!plain) {
        if (j >= rows.valid) f[j][i] = 1.0f, u = 0.0f;
        if (rows.pad >> j & 1) u = 0.0f;
        H[i] = cut >> j & 1 ? u : fmaf(f[j][i], H[i], u);
      } else {
        H[i] = fmaf(f[j][i], H[i], u);
      }
      A[i] *= f[j][i];
    }
  }
  // Backward over them: the pair (A, G).
#pragma unroll
  for (int j = R - 1; j >= 0; --j) {
    float y[CPL];
    V::unpack(yr[j], y);
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      if (!plain) {
        if (j >= rows.valid) y[i] = 0.0f;
        G[i] = cut >> j & 1 ? 0.0f : f[j][i] * (y[i] + G[i]);
      } else {
        G[i] = f[j][i] * (y[i] + G[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    A[i] = cut ? 0.0f : fmaxf(A[i], kTiny);
    mine.A[wave][i][lane] = A[i];
    mine.H[wave][i][lane] = G[i];
    s_h[wave][i][lane] = H[i];
  }
  __syncthreads();

  float cc[CPL];
  if (p.chunks > 1) {
    if (wave == 0 && chunk > 0) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float A0 = 1.0f, G0 = 0.0f;
#pragma unroll
        for (int v = kRecWaves - 1; v >= 0; --v) {
          G0 = after(G0, mine.A[v][i][lane], mine.H[v][i][lane]);
          A0 = product(A0, mine.A[v][i][lane]);
        }
        publish(p.pairs + (b * p.chunks + chunk) * D + c + i, A0, G0);
      }
    }
    look_back<CPL>(p, b, c, from_end, -1, start, got, base, wave, lane);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      cc[i] = base[i][lane];
      for (int v = 0; v < kRecWaves && from_end / kRecGroup * kRecGroup + 2 * v < from_end; ++v)
        cc[i] = after(cc[i], got.A[v][i][lane], got.H[v][i][lane]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < CPL; ++i) cc[i] = start[i];
  }
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    for (int v = kRecWaves - 1; v > wave; --v)
      cc[i] = after(cc[i], mine.A[v][i][lane], mine.H[v][i][lane]);
    for (int v = 0; v < wave; ++v) h[i] = after(h[i], mine.A[v][i][lane], s_h[v][i][lane]);
  }
  if (wave == 0 && from_end % kRecGroup == kRecGroup - 1 && chunk > 0) {
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      publish(p.states + (b * p.groups + from_end / kRecGroup) * D + c + i, 0.0f,
              after(cc[i], A[i], G[i]));
  }

  // The states again, row by row: w becomes m.
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float x[CPL];
    V::unpack(xr[j], x);
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const float u = bi[j][i] * x[i];
      if (!plain) {
        const bool stop = cut >> j & 1;
        w[j][i] = (stop ? 0.0f : h[i]) - w[j][i];
        h[i] = rows.pad >> j & 1 ? 0.0f : stop ? u : fmaf(f[j][i], h[i], u);
      } else {
        w[j][i] = h[i] - w[j][i];
        h[i] = fmaf(f[j][i], h[i], u);
      }
    }
  }
  float sum[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) sum[i] = 0.0f;
  const int64_t at = (b * T_ + t0) * D + c;
  T* dx = static_cast<T*>(a.dx) + at;
  T* dg = static_cast<T*>(a.dgate) + at;
  T* di = IG ? static_cast<T*>(a.dinput_gate) + at : nullptr;
#pragma unroll
  for (int j = R - 1; j >= 0; --j) {
    if (!plain && j >= rows.valid) continue;
    float y[CPL], ox[CPL], og[CPL], oi[CPL];
    V::unpack(yr[j], y);
    const bool pad = !plain && (rows.pad >> j & 1), stop = !plain && (cut >> j & 1);
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const float dh = y[i] + cc[i];
      ox[i] = dh * bi[j][i];
      if constexpr (IG) oi[i] = ox[i] * xi[j][i];
      const float q = dh * la[j][i] * w[j][i];
      og[i] = DECAY ? q * rest[j][i] : q;
      if (DECAY && !pad) sum[i] += q;
      cc[i] = stop ? 0.0f : f[j][i] * dh;
      if (pad) ox[i] = og[i] = 0.0f;
      if (IG && pad) oi[i] = 0.0f;
    }
    V::st(dx + j * D, V::pack(ox));
    V::st(dg + j * D, V::pack(og));
    if constexpr (IG) V::st(di + j * D, V::pack(oi));
  }
  if (a.dinitial_states && chunk == 0 && wave == 0) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) a.dinitial_states[b * D + c + i] = cc[i];
  }
  if constexpr (DECAY) {  // the chunk's sum, its waves in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CPL; ++i) s_h[wave][i][lane] = sum[i];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < kRecWaves; ++v) s += s_h[v][i][lane];
        p.part[(b * p.chunks + chunk) * D + c + i] = s;
      }
    }
  }
}

}  // namespace ops
}  // namespace ccv1d

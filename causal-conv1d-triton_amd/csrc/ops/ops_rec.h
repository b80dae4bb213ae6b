// The gated linear recurrence in one pass over its inputs, forward and backward.
//
// h[t] = f[t] h[t-1] + u[t] is cut along time into chunks of NW waves of R rows, a workgroup
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
// or flag is needed across the caches of the XCDs. The chunks of a wave column are dealt by a ticket in
// order of time (backward: from the end), not by workgroup number: a chunk waits only for words of chunks
// with lower tickets, whose workgroups have therefore started, and these publish their pairs before they
// wait for anything. The one wait on a wait is the state after a group, and by induction over tickets
// that ends too.
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

#include <type_traits>

#include "../ccv1d_device.h"
#include "ops_rec_math.h"

namespace ccv1d {
namespace ops {

constexpr int kRecGroup = 16;
constexpr uint32_t kReady = 0x80000000u;
constexpr float kTiny = 1.17549435e-38f;

struct RecParams {
  ccv1d_rec_args a;
  int32_t cols, chunks, groups;  // wave columns of 64 * CPL channels; chunks along time; their groups
  int32_t wide_ids;              // 1: seq_idx holds 64-bit ids, else 0
  Divisor by_cols, by_columns;   // cols; batch * cols
  uint64_t* pairs;               // (batch, chunks, dim)
  uint64_t* states;              // (batch, groups, dim): word of the state after a group
  uint32_t* tickets;             // (batch * cols,): the next chunk of each wave column
  float* part;  // backward: (batch, chunks, dim) sums behind ddecay
  // Rows whose starts and ends lie on the 128-byte lines are read and written once and kept out of the
  // caches' way (forward and backward at B=4 T=8192 D=1024 bf16: 219 us with cached accesses, 213 with
  // streamed stores, 207 with loads too). Other rows share lines with their neighbours, which another
  // wave reads at another time. (STREAM in the kernels: chosen at run time inside them, the stores'
  // branches cost B=4 T=16384 D=4096 without decay 836 -> 903 us.)
  bool stream;
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

// The pair (A, H) after the pair (A0, H0), or after a state: A = 0 cuts, which only happens in packed
// sequences (SEQ; elsewhere A is kTiny at the least).
template <bool SEQ>
__device__ __forceinline__ float after(float h, float A, float H) {
  return SEQ && A == 0.0f ? H : fmaf(A, h, H);
}
template <bool SEQ>
__device__ __forceinline__ float product(float A0, float A) {
  return SEQ && (A == 0.0f || A0 == 0.0f) ? 0.0f : fmaxf(A0 * A, kTiny);
}

// The rows of one wave that are not plain: bit j of each mask is row t0 + j.
struct Rows {
  uint32_t first, pad;  // a sequence's first row; padding
};

// A row's id: two words of 64 bits, or one of 32 twice.
struct Id {
  int32_t low, high;
};

// Lane l looks at row t0 - 1 + l (a row inside): its id is requested before the inputs and looked at once
// they are requested too (B=4 T=16384 D=4096 without decay, packed, forward and backward: looked at
// first 833 us, 812 so).
__device__ __forceinline__ Id id_of(const RecParams& p, int64_t b, int64_t t0, int lane) {
  const int64_t T = p.a.seqlen, t = min(max(t0 - 1 + lane, (int64_t)0), T - 1);
  const int32_t* at = static_cast<const int32_t*>(p.a.seq_idx) + ((b * T + t) << p.wide_ids);
  return {at[0], at[p.wide_ids]};
}

template <int R>
__device__ __forceinline__ Rows rows_of(Id id, int64_t t0, int valid, int lane) {
  const int32_t low = __shfl_up(id.low, 1), high = __shfl_up(id.high, 1);
  const uint64_t pad = __ballot(id.high < 0);
  const uint64_t first = __ballot(t0 + lane > 1 && (id.low != low || id.high != high));
  const uint32_t live = (1u << valid) - 1;
  return {(uint32_t)(first >> 1) & live, (uint32_t)(pad >> 1) & live};
}

// The rows of one tensor under a wave, from row t0 on: a uniform address (kept in scalar registers, which
// the compiler would otherwise fold into a vector address per row) and a lane's byte offset from it.
template <typename T, int CPL>
struct RowWalk {
  using V = VecIO<T, CPL>;
  typedef char __attribute__((address_space(1))) byte;
  typedef typename V::mem __attribute__((address_space(1))) cell;
  byte* row;
  int64_t step;
  __device__ __forceinline__ RowWalk(const void* base, int64_t stride_b, int64_t stride_t, int64_t b,
                                     int64_t t, int64_t c0)
      : row((byte*)base + (b * stride_b + t * stride_t + c0) * (int64_t)sizeof(T)),
        step(stride_t * (int64_t)sizeof(T)) {}
  template <bool STREAM>
  __device__ __forceinline__ typename V::raw load(uint32_t lane_bytes) const {
    if constexpr (STREAM) return __builtin_nontemporal_load((const cell*)(row + lane_bytes));
    return *(const cell*)(row + lane_bytes);
  }
  template <bool STREAM>
  __device__ __forceinline__ void store(uint32_t lane_bytes, const float (&v)[CPL]) {
    if constexpr (STREAM) __builtin_nontemporal_store(V::pack(v), (cell*)(row + lane_bytes));
    else *(cell*)(row + lane_bytes) = V::pack(v);
  }
  __device__ __forceinline__ void move(int64_t bytes) {
    row += bytes;
    asm volatile("" : "+s"(row));
  }
};

template <int CPL>
__device__ __forceinline__ void settle(float (&v)[CPL]) {
#pragma unroll
  for (int i = 0; i < CPL; ++i) asm volatile("" : "+v"(v[i]));
}

// Loads R rows; those past the last one, `valid` - 1, repeat it.
template <bool STREAM, typename T, int CPL, int R>
__device__ __forceinline__ void load_rows(RowWalk<T, CPL> w, int valid, uint32_t lane_bytes,
                                          typename VecIO<T, CPL>::raw (&to)[R]) {
#pragma unroll
  for (int j = 0; j < R; ++j) {
    to[j] = w.template load<STREAM>(lane_bytes);
    w.move(j + 1 < valid ? w.step : 0);
  }
}

// Makes the compiler forget what it knows of a loaded row: values made from it before are made again
// rather than kept, and nothing is made from it before this point. Statements of this kind keep their
// order, so a pair of them around a row's arithmetic keeps rows apart: interleaved by the scheduler, they
// needed more registers than four waves have.
template <typename RAW>
__device__ __forceinline__ void forget_row(RAW& v) {
  if constexpr (sizeof(RAW) == 2) {
    uint32_t t = v;
    asm volatile("" : "+v"(t));
    v = (RAW)t;
  } else {
#pragma unroll
    for (int i = 0; i < (int)sizeof(RAW) / 4; ++i) {
      uint32_t t = v[i];
      asm volatile("" : "+v"(t));
      v[i] = t;
    }
  }
}

// The wave column (batch row and channels) of this workgroup. Workgroups go to the 8 XCDs in turn; columns
// move on by one from n to n workgroups, or with n a multiple of 8 an XCD would have the same columns
// for good, and with rows of a power of two the same part of the memory's channels (forward and backward
// at B=4 T=8192 D=1024 219 us, 198 so). Where rows are not on cache lines, an XCD takes columns side by
// side, whose lines overlap (B=3 T=5001 D=1501 fp32 273 us, 248 so; rows on lines 1 % slower).
__device__ __forceinline__ int column_of(const RecParams& p) {
  const uint32_t n = (uint32_t)(p.a.batch * p.cols);
  const uint32_t turn = divide(blockIdx.x, p.by_columns), i = blockIdx.x - turn * n;
  const uint32_t at = (p.stream ? i : (uint32_t)xcd_remap((int)i, (int)n)) + turn;
  return (int)(at - divide(at, p.by_columns) * n);
}

// Deals this workgroup a chunk of its column, counted from the walk's start. A column's chunks have a
// counter of their own: with one for all, the 512 workgroups that start together waited in line for it
// (forward of B=16 T=256 D=2048 25 us, 18 so). `meanwhile` is what can be done before the chunk is known.
template <typename F>
__device__ __forceinline__ int deal(const RecParams& p, int bc, uint32_t* s_ticket, F&& meanwhile) {
  uint32_t ticket = 0;
  if (p.chunks > 1 && threadIdx.x == 0)
    ticket = __hip_atomic_fetch_add(p.tickets + bc, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  meanwhile();
  if (p.chunks <= 1) return 0;
  if (threadIdx.x == 0) *s_ticket = ticket;
  __syncthreads();
  return (int)__builtin_amdgcn_readfirstlane(*s_ticket);
}

// The pairs of the waves of a workgroup, and of the chunks before it, in LDS.
template <int NW, int CPL>
struct Pairs {
  float A[NW][CPL][kWave], H[NW][CPL][kWave];
};

// Words of (batch, n, dim) rows: a uniform row and the lane's place in it.
__device__ __forceinline__ uint64_t* word_row(uint64_t* words, int64_t row, int64_t D, int64_t c0) {
  return words + row * D + c0;
}

// Combines the chunks between the group before and this chunk, kLook of them a wave in order, into
// `got`; the state in front of the group goes to `base`. `chunk` counts from the walk's start.
template <int NW>
constexpr int kLook = (kRecGroup - 2) / NW + 1;

template <bool SEQ, int NW, int CPL>
__device__ __forceinline__ void look_back(const RecParams& p, int64_t b, int64_t c0, uint32_t lane_c,
                                          int chunk, int dir, const float* start,
                                          Pairs<NW, CPL>& got, float (&base)[CPL][kWave], int wave,
                                          int lane) {
  constexpr int N = kLook<NW>;
  const int64_t D = p.a.dim;
  const int g = chunk / kRecGroup, j0 = g * kRecGroup + N * wave;
  // chunks are stored in order of time
  auto pair = [&](int j) {
    return word_row(p.pairs, b * p.chunks + (dir > 0 ? j : p.chunks - 1 - j), D, c0) + lane_c;
  };
  const uint64_t* gs = word_row(p.states, b * p.groups + (g - 1), D, c0) + lane_c;
  uint64_t v[N][CPL], s[CPL];
#pragma unroll
  for (int n = 0; n < N; ++n)  // requested together
    if (j0 + n < chunk) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) v[n][i] = peek(pair(j0 + n) + i);
    }
  if (wave == 0 && g > 0) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) s[i] = peek(gs + i);
  }
  if (j0 < chunk) {
    float A[CPL], H[CPL];
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (j0 + n < chunk) {
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
          const uint64_t w = await(pair(j0 + n) + i, v[n][i]);
          const float A1 = __uint_as_float((uint32_t)w & ~kReady);
          const float H1 = __uint_as_float((uint32_t)(w >> 32));
          H[i] = n == 0 ? H1 : after<SEQ>(H[i], A1, H1);
          A[i] = n == 0 ? A1 : product<SEQ>(A[i], A1);
        }
      }
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      got.A[wave][i][lane] = A[i];
      got.H[wave][i][lane] = H[i];
    }
  }
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      base[i][lane] = g > 0 ? __uint_as_float((uint32_t)(await(gs + i, s[i]) >> 32))
                            : start ? (start + b * D + c0)[lane_c + i] : 0.0f;
  }
}

// The state in front of the chunk from what look_back left, and the chunk's pair from its waves'.
template <bool SEQ, int NW, int CPL>
__device__ __forceinline__ float look_back_state(const Pairs<NW, CPL>& got,
                                                 const float (&base)[CPL][kWave], int chunk, int i,
                                                 int lane) {
  float h = base[i][lane];
  const int n = chunk % kRecGroup;
  for (int w = 0; w * kLook<NW> < n; ++w) h = after<SEQ>(h, got.A[w][i][lane], got.H[w][i][lane]);
  return h;
}

// A lane's channels. The last lanes of a row share its last CPL channels and compute the same values twice.
template <int CPL>
struct Channels {
  int64_t b, c0;    // batch row, the wave column's first channel
  uint32_t lane_c;  // the lane's first channel, from c0 on
  __device__ __forceinline__ Channels(const RecParams& p, int bc, int lane) {
    const int64_t D = p.a.dim;
    const uint32_t row = divide(bc, p.by_cols);
    b = row;
    c0 = min((int64_t)(bc - (int)row * p.cols) * (kWave * CPL), D - CPL);
    lane_c = (uint32_t)min((int64_t)lane * CPL, D - CPL - c0);
  }
};

// The rows of a wave.
template <int NW, int R>
struct Place {
  int valid;       // rows inside the sequence
  int64_t t0, t1;  // first row (and a row inside)
  __device__ __forceinline__ Place(const RecParams& p, int chunk, int wave) {
    const int64_t T = p.a.seqlen;
    t0 = ((int64_t)chunk * NW + wave) * R;
    t1 = min(t0, T - 1);
    valid = (int)max((int64_t)0, min((int64_t)R, T - t0));
  }
};

// The rates of a lane's channels; whether all of them are slow.
template <int CPL, bool DECAY>
__device__ __forceinline__ bool rates(const ccv1d_rec_args& a, const Channels<CPL>& ch, float (&k)[CPL]) {
  bool slow = true;
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    k[i] = DECAY ? decay_rate((a.decay + ch.c0)[ch.lane_c + i], a.decay_scale) : 0.0f;
    slow = slow && slow_channel(k[i]);
  }
  return slow;
}

// Requests the inputs row by row, so that work on the first rows can begin while the rest is on its way
// (loads complete in order; tensor by tensor, with the decay after them, B=4 T=8192 D=1024 bf16 took 188 us
// forward and backward, 173 so, and 170 with the rates made while the ticket is on its way). Rows past the last one repeat it.
template <bool STREAM, bool IG, typename T, int CPL, int R, int NW>
__device__ __forceinline__ void load_inputs(const ccv1d_rec_args& a, const Channels<CPL>& ch,
                                            const Place<NW, R>& at, uint32_t lane_bytes,
                                            typename VecIO<T, CPL>::raw (&gr)[R],
                                            typename VecIO<T, CPL>::raw (&xr)[R],
                                            typename VecIO<T, CPL>::raw (&ir)[R]) {
  RowWalk<T, CPL> g(a.gate, a.gate_stride_b, a.gate_stride_t, ch.b, at.t1, ch.c0);
  RowWalk<T, CPL> x(a.x, a.x_stride_b, a.x_stride_t, ch.b, at.t1, ch.c0);
  RowWalk<T, CPL> i(a.input_gate, a.input_gate_stride_b, a.input_gate_stride_t, ch.b, at.t1, ch.c0);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    gr[j] = g.template load<STREAM>(lane_bytes);
    xr[j] = x.template load<STREAM>(lane_bytes);
    if constexpr (IG) ir[j] = i.template load<STREAM>(lane_bytes);
    const bool more = j + 1 < at.valid;
    g.move(more ? g.step : 0);
    x.move(more ? x.step : 0);
    if constexpr (IG) i.move(more ? i.step : 0);
  }
}

// ------------------------------------------------------------------------------------- forward
//
// Bound by memory without decay: B=4 T=16384 D=4096 bf16 without an input gate 295 us, 5.5 TB/s of its
// 1.61 GB. With decay (6 of its 30 operations per element are transcendental, at half rate) memory and
// arithmetic, the VALUs 60 % busy: B=4 T=8192 D=1024 bf16 62 us with the clearing, 4.3 TB/s; in fp32,
// B=3 T=5001 D=1501, 86 us, 4.2 TB/s. 8 waves of 16 rows at 4 waves per SIMD: 4 waves of 16 rows
// took 1 % more with decay and 1 % less without, 8 waves of 8 rows 6 and 14 % more.

template <typename T, int CPL, bool DECAY, bool IG, bool SEQ, bool STREAM, int NW, int R>
__global__ __launch_bounds__(NW* kWave, 4) void rec_fwd_kernel(RecParams p) {
  using V = VecIO<T, CPL>;
  static_assert(NW * R % CCV1D_REC_SAVED_ROWS == 0 && CCV1D_REC_SAVED_ROWS % R == 0, "saved states");
  __shared__ Pairs<NW, CPL> mine, got;
  __shared__ float base[CPL][kWave];
  __shared__ uint32_t s_ticket;
  const ccv1d_rec_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bc = column_of(p);
  const Channels<CPL> ch(p, bc, lane);
  float k[CPL];
  bool slow;
  const int chunk = deal(p, bc, &s_ticket, [&]() { slow = rates<CPL, DECAY>(a, ch, k); });
  const Place<NW, R> at(p, chunk, wave);
  const int valid = at.valid;
  const int64_t b = ch.b, T_ = a.seqlen, D = a.dim, t0 = at.t0, c0 = ch.c0;
  const uint32_t lane_c = ch.lane_c, lane_bytes = lane_c * (uint32_t)sizeof(T);

  Id id{0, 0};
  if constexpr (SEQ) id = id_of(p, b, t0, lane);

  typename V::raw xr[R], gr[R], ir[R];
  load_inputs<STREAM, IG, T>(a, ch, at, lane_bytes, gr, xr, ir);
  Rows rows{0, 0};
  if constexpr (SEQ) rows = rows_of<R>(id, t0, valid, lane);
  const uint32_t cut = rows.first | rows.pad;

  float f[R][CPL], u[R][CPL], A[CPL], H[CPL];
  auto coefficients = [&](auto is_slow) {
    constexpr int kTogether = decltype(is_slow)::value ? 2 : 1;  // rows
    float tail[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) tail[i] = sinh_tail(k[i]);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (j % kTogether == 0) {
#pragma unroll
        for (int n = j; n < j + kTogether; ++n) {
          forget_row(xr[n]);
          forget_row(gr[n]);
          if constexpr (IG) forget_row(ir[n]);
        }
      }
      float x[CPL], g[CPL], ig[CPL];
      V::unpack(xr[j], x);
      V::unpack(gr[j], g);
      if constexpr (IG) V::unpack(ir[j], ig);
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float beta;
        forget<T, DECAY, decltype(is_slow)::value>(k[i], tail[i], g[i], f[j][i], beta);
        u[j][i] = beta * x[i];
        if constexpr (IG) u[j][i] *= sigmoid<T>(ig[i]);
      }
      if ((j + 1) % kTogether == 0) {
#pragma unroll
        for (int n = j + 1 - kTogether; n <= j; ++n) {
          settle(f[n]);
          settle(u[n]);
        }
      }
    }
  };
  if (DECAY && !__all(slow)) coefficients(std::false_type{});
  else coefficients(std::true_type{});
  if (valid < R) {  // past the end nothing happens
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < CPL; ++i)
        if (j >= valid) f[j][i] = 1.0f, u[j][i] = 0.0f;
  }
  // One row's step from the state before it; MASKED: where a row of the wave cuts the state.
  auto step = [&](auto masked, int j, int i, float h) {
    const float next = fmaf(f[j][i], h, u[j][i]);
    if constexpr (decltype(masked)::value) return cut >> j & 1 ? u[j][i] : next;
    return next;
  };
  auto pair = [&](auto masked) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) A[i] = 1.0f, H[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        if (decltype(masked)::value && (rows.pad >> j & 1)) u[j][i] = 0.0f;
        H[i] = step(masked, j, i, H[i]);
        A[i] *= f[j][i];
      }
  };
  if (SEQ && cut) pair(std::true_type{});
  else pair(std::false_type{});
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    A[i] = SEQ && cut ? 0.0f : fmaxf(A[i], kTiny);
    mine.A[wave][i][lane] = A[i];
    mine.H[wave][i][lane] = H[i];
  }
  __syncthreads();

  float h[CPL];
  if (p.chunks > 1) {
    if (wave == NW - 1 && chunk + 1 < p.chunks) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float A0 = mine.A[0][i][lane], H0 = mine.H[0][i][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
          H0 = after<SEQ>(H0, mine.A[w][i][lane], mine.H[w][i][lane]);
          A0 = product<SEQ>(A0, mine.A[w][i][lane]);
        }
        publish(word_row(p.pairs, b * p.chunks + chunk, D, c0) + lane_c + i, A0, H0);
      }
    }
    look_back<SEQ>(p, b, c0, lane_c, chunk, 1, a.initial_states, got, base, wave, lane);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CPL; ++i) h[i] = look_back_state<SEQ>(got, base, chunk, i, lane);
  } else {
#pragma unroll
    for (int i = 0; i < CPL; ++i) h[i] = a.initial_states ? (a.initial_states + b * D + c0)[lane_c + i] : 0.0f;
  }
  for (int w = 0; w < wave; ++w)
#pragma unroll
    for (int i = 0; i < CPL; ++i) h[i] = after<SEQ>(h[i], mine.A[w][i][lane], mine.H[w][i][lane]);
  if (wave == NW - 1 && chunk % kRecGroup == kRecGroup - 1 && chunk + 1 < p.chunks) {
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      publish(word_row(p.states, b * p.groups + chunk / kRecGroup, D, c0) + lane_c + i, 0.0f,
              after<SEQ>(h[i], mine.A[wave][i][lane], mine.H[wave][i][lane]));
  }
  if (valid == 0) return;
  if (a.saved && t0 % CCV1D_REC_SAVED_ROWS == 0) {
    const int64_t ns = (T_ + CCV1D_REC_SAVED_ROWS - 1) / CCV1D_REC_SAVED_ROWS;
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      (a.saved + (b * ns + t0 / CCV1D_REC_SAVED_ROWS) * D + c0)[lane_c + i] = h[i];
  }
  RowWalk<T, CPL> out(a.out, T_ * D, D, b, t0, c0);
  auto walk = [&](auto masked) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (j < valid) {
#pragma unroll
        for (int i = 0; i < CPL; ++i) h[i] = step(masked, j, i, h[i]);
        out.template store<STREAM>(lane_bytes, h);
        out.move(out.step);
      }
    }
  };
  if (SEQ && cut) walk(std::true_type{});
  else walk(std::false_type{});
  if (a.final_states && t0 + valid == T_) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) (a.final_states + b * D + c0)[lane_c + i] = h[i];
  }
}

// ------------------------------------------------------------------------------------ backward
//
// dh[t] = dout[t] + f[t+1] dh[t+1]; what row t hands to the row before is c = f[t] (dout[t] + c'), so
// a stretch of rows acts on what reaches its end as c -> A c + G with the A of the forward. With
// m = h[t-1] - w (h[t-1] taken as zero where the state is cut):
//   dx = dh beta i, dinput_gate = dx x (1 - i)
//   with decay:     w = i x a / beta,  q = dh (ln a) a m,  dgate = q (1 - r),  ddecay from the sum of q
//                   (a / beta comes from d beta / d(ln a) = -a^2 / beta; where a is exactly 1, ln a = 0
//                   makes q zero, and 1 / beta is held finite)
//   without decay:  w = i x,           dgate = dh a beta m
//
// Bound like the forward: without decay 503 us, 5.3 TB/s of 2.68 GB, at the size given there; with decay
// (66 operations per element) the VALUs are 72 % busy: B=4 T=8192 D=1024 bf16 106 us with the clearing
// and the decay's sum, 4.4 TB/s; in fp32, B=3 T=5001 D=1501, 161 us, 3.9 TB/s. Rows per wave are half of
// the forward's, since twice as much is held per row; 4 waves of 8 rows: 128 us where 8 were 126, and
// 4 % more without decay.

template <typename T, int CPL, bool DECAY, bool IG, bool SEQ, bool STREAM, int NW, int R>
__global__ __launch_bounds__(NW* kWave, 4) void rec_bwd_kernel(RecParams p) {
  using V = VecIO<T, CPL>;
  static_assert(NW * R == CCV1D_REC_SAVED_ROWS, "one saved state per chunk");
  __shared__ Pairs<NW, CPL> mine, got;
  __shared__ float s_h[NW][CPL][kWave];
  __shared__ float base[CPL][kWave];
  // Kept per element from the coefficients to the gradients: in registers a, beta i and w (then m). One
  // channel a lane also leaves room for r, 1 - r and x (1 - i). With two, x (1 - i) goes through LDS, and for
  // the first kGate rows 1 - r, with r in registers (without decay r is a); the other rows' are made
  // again from the gate. (B=4 T=8192 D=1024 bf16, kernel and its two small ones: all made again 125 us,
  // the first in LDS 122, 4 rows' r and 1 - r too 121, 6 rows' 122; without an input gate 8 rows' need a
  // register more than there are. Without decay, B=4 T=16384 D=4096: 523 and 515.)
  constexpr bool kKeep = CPL == 1;
  constexpr int kGate = kKeep ? 0 : IG ? R / 2 : DECAY ? R - 2 : R, kRest = kKeep || !IG ? 0 : R;
  __shared__ float s_rest[kKeep ? 1 : NW][kRest + kGate + kKeep][kWave][CPL];
  __shared__ uint32_t s_ticket;
  const ccv1d_rec_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bc = column_of(p);
  const Channels<CPL> ch(p, bc, lane);
  float k[CPL];
  bool slow;
  const int from_end = deal(p, bc, &s_ticket, [&]() { slow = rates<CPL, DECAY>(a, ch, k); });
  const int chunk = p.chunks - 1 - from_end;
  const Place<NW, R> at(p, chunk, wave);
  const int valid = at.valid;
  const int64_t b = ch.b, T_ = a.seqlen, D = a.dim, t0 = at.t0, c0 = ch.c0;
  const uint32_t lane_c = ch.lane_c, lane_bytes = lane_c * (uint32_t)sizeof(T);

  Id id{0, 0};
  if constexpr (SEQ) id = id_of(p, b, t0, lane);

  typename V::raw xr[R], gr[R], ir[R], yr[R];
  load_inputs<STREAM, IG, T>(a, ch, at, lane_bytes, gr, xr, ir);
  Rows rows{0, 0};
  if constexpr (SEQ) rows = rows_of<R>(id, t0, valid, lane);
  const uint32_t cut = rows.first | rows.pad;
  load_rows<STREAM, T, CPL, R>({a.dout, a.dout_stride_b, a.dout_stride_t, b, at.t1, c0}, valid,
                                lane_bytes, yr);
  float h[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) h[i] = (a.saved + (b * p.chunks + chunk) * D + c0)[lane_c + i];

  float f[R][CPL], bi[R][CPL], w[R][CPL];
  float kr[R][CPL], kn[R][CPL], kx[R][CPL];  // kKeep: r (and of kGate rows), 1 - r, x (1 - i)
  auto coefficients = [&](auto is_slow) {
    constexpr int kTogether = decltype(is_slow)::value ? 2 : 1;  // rows
    float tail[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) tail[i] = sinh_tail(k[i]);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (j % kTogether == 0) {
#pragma unroll
        for (int n = j; n < j + kTogether; ++n) {
          forget_row(xr[n]);
          forget_row(gr[n]);
          if constexpr (IG) forget_row(ir[n]);
        }
      }
      float x[CPL], g[CPL], ig[CPL];
      V::unpack(xr[j], x);
      V::unpack(gr[j], g);
      if constexpr (IG) V::unpack(ir[j], ig);
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float in = 1.0f, r;
        if constexpr (IG && kKeep) {
          float not_in;
          sigmoid_pair<T>(ig[i], in, not_in);
          kx[j][i] = x[i] * not_in;
        } else if constexpr (IG) {
          float not_in;
          sigmoid_and_rest<T>(ig[i], in, not_in);
          s_rest[wave][j][lane][i] = x[i] * not_in;
        }
        if constexpr (DECAY) {
          if constexpr (kKeep) {
            sigmoid_pair<T>(g[i], r, kn[j][i]);
            kr[j][i] = r;
          } else if (j < kGate) {
            sigmoid_and_rest<T>(g[i], r, s_rest[wave][kRest + j][lane][i]);
            kr[j][i] = r;
          } else {
            r = sigmoid<T>(g[i]);
          }
          const float l = k[i] * r;
          f[j][i] = __builtin_amdgcn_exp2f(l);
          const float s = one_minus_square<decltype(is_slow)::value>(tail[i], l, f[j][i]);
          const float inv = __builtin_amdgcn_rsqf(fmaxf(s, kTiny));
          const float ib = in * inv;
          bi[j][i] = s * ib;
          w[j][i] = x[i] * (f[j][i] * ib);
        } else {
          float beta;
          sigmoid_pair<T>(g[i], f[j][i], beta);
          if constexpr (kKeep) kn[j][i] = beta;
          else if (j < kGate) s_rest[wave][kRest + j][lane][i] = beta;
          bi[j][i] = beta * in;
          w[j][i] = in * x[i];
        }
      }
      if ((j + 1) % kTogether == 0) {
#pragma unroll
        for (int n = j + 1 - kTogether; n <= j; ++n) {
          settle(f[n]);
          settle(bi[n]);
          settle(w[n]);
          if (DECAY && n < kGate) settle(kr[n]);
        }
      }
    }
  };
  if (DECAY && !__all(slow)) coefficients(std::false_type{});
  else coefficients(std::true_type{});
  if (valid < R) {  // past the end nothing happens
    const float zero[CPL] = {};
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (j >= valid) {
        xr[j] = yr[j] = V::pack(zero);
#pragma unroll
        for (int i = 0; i < CPL; ++i) f[j][i] = 1.0f, bi[j][i] = 0.0f;
      }
  }

  // Forward over the rows: the pair (A, H); backward over them: (A, G).
  float A[CPL], H[CPL], G[CPL];
  auto forward = [&](auto masked, int j, int i, float x, float h) {
    const float u = bi[j][i] * x;
    if constexpr (decltype(masked)::value)
      return rows.pad >> j & 1 ? 0.0f : cut >> j & 1 ? u : fmaf(f[j][i], h, u);
    return fmaf(f[j][i], h, u);
  };
  auto pairs = [&](auto masked) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) A[i] = 1.0f, H[i] = 0.0f, G[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float x[CPL];
      V::unpack(xr[j], x);
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        H[i] = forward(masked, j, i, x[i], H[i]);
        A[i] *= f[j][i];
      }
    }
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      float y[CPL];
      V::unpack(yr[j], y);
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        G[i] = f[j][i] * (y[i] + G[i]);
        if (decltype(masked)::value && (cut >> j & 1)) G[i] = 0.0f;
      }
    }
  };
  if (SEQ && cut) pairs(std::true_type{});
  else pairs(std::false_type{});
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    A[i] = SEQ && cut ? 0.0f : fmaxf(A[i], kTiny);
    mine.A[wave][i][lane] = A[i];
    mine.H[wave][i][lane] = G[i];
    s_h[wave][i][lane] = H[i];
  }
  __syncthreads();

  float cc[CPL];
  if (p.chunks > 1) {
    if (wave == NW - 1 && chunk > 0) {
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        float A0 = mine.A[NW - 1][i][lane], G0 = mine.H[NW - 1][i][lane];
#pragma unroll
        for (int v = NW - 2; v >= 0; --v) {
          G0 = after<SEQ>(G0, mine.A[v][i][lane], mine.H[v][i][lane]);
          A0 = product<SEQ>(A0, mine.A[v][i][lane]);
        }
        publish(word_row(p.pairs, b * p.chunks + chunk, D, c0) + lane_c + i, A0, G0);
      }
    }
    look_back<SEQ>(p, b, c0, lane_c, from_end, -1, a.dfinal_states, got, base, wave, lane);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CPL; ++i) cc[i] = look_back_state<SEQ>(got, base, from_end, i, lane);
  } else {
#pragma unroll
    for (int i = 0; i < CPL; ++i) cc[i] = a.dfinal_states ? (a.dfinal_states + b * D + c0)[lane_c + i] : 0.0f;
  }
  for (int v = NW - 1; v > wave; --v)
#pragma unroll
    for (int i = 0; i < CPL; ++i) cc[i] = after<SEQ>(cc[i], mine.A[v][i][lane], mine.H[v][i][lane]);
  for (int v = 0; v < wave; ++v)
#pragma unroll
    for (int i = 0; i < CPL; ++i) h[i] = after<SEQ>(h[i], mine.A[v][i][lane], s_h[v][i][lane]);
  if (wave == 0 && from_end % kRecGroup == kRecGroup - 1 && chunk > 0) {
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      publish(word_row(p.states, b * p.groups + from_end / kRecGroup, D, c0) + lane_c + i, 0.0f,
              after<SEQ>(cc[i], mine.A[wave][i][lane], mine.H[wave][i][lane]));
  }

  float sum[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    sum[i] = 0.0f;
    if constexpr (DECAY) k[i] *= kLn2;  // ln a = k r from here on
  }
  const int64_t last = t0 + valid - 1;  // stored from the last row back
  RowWalk<T, CPL> dx(a.dx, T_ * D, D, b, last, c0), dg(a.dgate, T_ * D, D, b, last, c0);
  RowWalk<T, CPL> di(a.dinput_gate, T_ * D, D, b, last, c0);
  // The states again, row by row (w becomes m), then the gradients from the last row back.
  auto walk = [&](auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if constexpr (!kKeep) forget_row(xr[j]);
      float x[CPL];
      V::unpack(xr[j], x);
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        w[j][i] = (kMasked && (cut >> j & 1) ? 0.0f : h[i]) - w[j][i];
        h[i] = forward(masked, j, i, x[i], h[i]);
      }
    }
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      if (j >= valid) continue;
      if constexpr (!kKeep) {
        if (j >= kGate) forget_row(gr[j]);
        forget_row(yr[j]);
      }
      const bool pad = kMasked && (rows.pad >> j & 1);
      float y[CPL], g[CPL], ox[CPL], og[CPL], oi[CPL];
      V::unpack(yr[j], y);
      V::unpack(gr[j], g);
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        const float dh = y[i] + cc[i];
        cc[i] = kMasked && (cut >> j & 1) ? 0.0f : f[j][i] * dh;
        ox[i] = dh * bi[j][i];
        if constexpr (IG && kKeep) {
          oi[i] = ox[i] * kx[j][i];
        } else if constexpr (IG) {
          oi[i] = ox[i] * s_rest[wave][j][lane][i];
        }
        float r, not_r;
        if constexpr (kKeep) r = kr[j][i], not_r = kn[j][i];
        else if (j < kGate) r = DECAY ? kr[j][i] : f[j][i], not_r = s_rest[wave][kRest + j][lane][i];
        else sigmoid_pair_of_number<T>(g[i], r, not_r);
        float q = dh * f[j][i] * w[j][i];
        if constexpr (DECAY) {
          q *= k[i] * r;
          sum[i] += pad ? 0.0f : q;
        }
        og[i] = q * not_r;
        if (pad) ox[i] = og[i] = oi[i] = 0.0f;
      }
      dx.template store<STREAM>(lane_bytes, ox);
      dg.template store<STREAM>(lane_bytes, og);
      dx.move(-dx.step);
      dg.move(-dg.step);
      if constexpr (IG) {
        di.template store<STREAM>(lane_bytes, oi);
        di.move(-di.step);
      }
    }
  };
  if (SEQ && cut) walk(std::true_type{});
  else walk(std::false_type{});
  if (a.dinitial_states && chunk == 0 && wave == 0) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) (a.dinitial_states + b * D + c0)[lane_c + i] = cc[i];
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
        for (int v = 0; v < NW; ++v) s += s_h[v][i][lane];
        (p.part + (b * p.chunks + chunk) * D + c0)[lane_c + i] = s;
      }
    }
  }
}

}  // namespace ops
}  // namespace ccv1d

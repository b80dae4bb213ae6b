// Launch of the gated delta rule: workspace, the empty cases, and the form for single tokens.
#include "ops_delta_launch.h"

namespace ccv1d {
namespace ops {

namespace {

constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1;

// No rows: the final states are the initial ones, and their gradients likewise.
__global__ __launch_bounds__(256) void delta_empty_kernel(const float* from, float* to, int64_t n) {
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) to[i] = from ? from[i] : 0.0f;
}

struct Sizes {
  int64_t chunks, dk, dvp, tiles;
  int64_t kfrag;  // units of 16 bytes of the fragments of k by rows in a chunk, as the others of q and k
  int64_t tri, units_p;  // units of a triangle's fragments; of one of P in the forward
};

Sizes sizes_of(const ccv1d_delta_args& a) {
  Sizes z;
  z.chunks = (a.seqlen + CCV1D_DELTA_CHUNK - 1) / CCV1D_DELTA_CHUNK;
  z.dk = a.key_dim <= 64 ? 64 : a.key_dim <= 128 ? 128 : 256;
  z.dvp = (a.value_dim + 31) / 32 * 32;
  z.tiles = z.dvp / 16;
  const int64_t pieces = a.dtype == CCV1D_BF16 ? 1 : a.dtype == CCV1D_F16 ? 2 : 3;
  z.kfrag = CCV1D_DELTA_CHUNK * z.dk / 8 * pieces;
  z.tri = 6 * 64;
  z.units_p = a.dtype == CCV1D_F32 ? 3 : 2;
  return z;
}

constexpr int64_t kRowFloats = 8 * CCV1D_DELTA_CHUNK;

struct Places {  // in bytes
  int64_t kf, qf, kt, qt, tf, pf, rows, ds, dr, gates, all;
};

Places places_of(const ccv1d_delta_args& a, const Sizes& z, bool backward) {
  Places p{};
  const int64_t kc = a.batch * a.key_heads * z.chunks, hc = a.batch * a.heads * z.chunks;
  int64_t at = 0;
  auto next = [&](int64_t bytes) {
    const int64_t here = at;
    at += bytes;
    return here;
  };
  p.kf = next(kc * z.kfrag * 16);
  p.qf = next(kc * z.kfrag * 16);
  p.kt = next(kc * z.kfrag * 16);
  p.qt = next(backward ? kc * z.kfrag * 16 : 0);
  p.tf = next(hc * z.tri * 3 * 16);
  p.pf = next(hc * z.tri * (backward ? 3 : z.units_p) * 16);
  p.rows = next(hc * kRowFloats * 4);
  p.ds = next(backward ? hc * z.dk * z.dvp * 4 : 0);
  p.dr = next(backward ? hc * CCV1D_DELTA_CHUNK * z.dvp * 4 : 0);
  // of keys whose elements lie in several workgroups, 128 in each, in fp32 64
  const int64_t parts = z.dk / (a.dtype == CCV1D_F32 ? 64 : 128);
  p.gates = next(backward && parts > 1 ? hc * parts * 4 * CCV1D_DELTA_CHUNK * 4 : 0);
  p.all = at;
  return p;
}

hipError_t run(const ccv1d_delta_args& a, bool backward, hipStream_t s) {
  if (a.seqlen == 0) {
    const int64_t n = a.batch * a.heads * a.key_dim * a.value_dim;
    const float* from = backward ? a.dfinal_states : a.initial_states;
    float* to = backward ? a.dinitial_states : a.final_states;
    if (!to) return hipSuccess;
    const int64_t blocks = (n + 1023) / 1024;
    return start(&delta_empty_kernel, blocks < 2048 ? blocks : 2048, 256, s, from, to, n);
  }
  const Sizes z = sizes_of(a);
  const Places at = places_of(a, z, backward);
  DeltaParams p{};
  p.a = a;
  p.chunks = (int32_t)z.chunks;
  p.group = (int32_t)(a.heads / a.key_heads);
  // Up to 512 workgroups run at once with some room: below that a head each is quicker, though each reads q and k anew
  // (B=4 T=256, 16 heads of 128 over 8 key heads: 128 workgroups of two heads 21 us, 256 of one 17).
  p.prep_heads = a.batch * a.key_heads * z.chunks < 512 ? 1 : p.group;
  p.dk = (int32_t)z.dk, p.dvp = (int32_t)z.dvp, p.tiles = (int32_t)z.tiles;
  char* ws = static_cast<char*>(a.workspace);
  auto unit = [&](int64_t o) { return reinterpret_cast<u4*>(ws + o); };
  auto floats = [&](int64_t o) { return reinterpret_cast<float*>(ws + o); };
  p.kf = unit(at.kf), p.qf = unit(at.qf), p.kt = unit(at.kt), p.qt = unit(at.qt), p.tf = unit(at.tf);
  p.pf = unit(at.pf), p.rows = floats(at.rows), p.ds = floats(at.ds), p.dr = floats(at.dr);
  p.gates = floats(at.gates);
  p.s0 = a.saved;
  p.u = a.saved ? a.saved + a.batch * a.heads * z.chunks * z.dk * z.dvp : nullptr;
  switch (a.dtype) {
    case CCV1D_BF16: return delta_launch_bf16(p, backward, s);
    case CCV1D_F16: return delta_launch_f16(p, backward, s);
    default: return delta_launch_f32(p, backward, s);
  }
}

// One token of a request and head, 64 value columns a workgroup: four a lane, the keys' elements over 16 groups of
// lanes, ROWS each. One reading of the state gives S^T k and S^T q, from which
//   u = beta (v - a S^T k),  o = scale (a S^T q + (q.k) u),  S <- a S + k u^T,  a = exp(g).
// Bound by memory: the states are read and written once, at 128 rows of 32 heads of 128 by 128 537 MB, 126 us a call on a
// pool that lies outside the caches (4.3 TB/s, 0.84 of a copy's rate), 107 on one that stays in them. 4 rows of 8
// heads take 6.7 us, the latency of the slot's number, a reading of its state and a sum over waves.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void delta_update_kernel(ccv1d_delta_update_args p, int32_t group, int32_t cols) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  __shared__ float sums[4][16][9];
  const int64_t rh = blockIdx.x / cols;  // (row, head)
  const int64_t r = rh / p.heads, h = rh - r * p.heads, kh = h / group;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, x = threadIdx.x & 15, y = threadIdx.x >> 4;
  const int64_t d = (int64_t)(blockIdx.x - rh * cols) * 64 + 4 * x;
  const int n = (int)max((int64_t)0, min((int64_t)4, p.value_dim - d));
  T* out = static_cast<T*>(p.out) + rh * p.value_dim + d;
  const int64_t slot = p.state_indices ? p.state_indices[r] : r;
  if (slot < 0 || slot >= p.slots) {  // the whole workgroup
    if (y == 0)
      for (int i = 0; i < n; ++i) out[i] = (T)0.0f;
    return;
  }
  float* state = p.state + slot * p.state_stride + h * p.key_dim * p.value_dim + d;
  const T* kp = static_cast<const T*>(p.k) + r * p.k_stride_r + kh * p.k_stride_h;
  const T* qp = static_cast<const T*>(p.q) + r * p.q_stride_r + kh * p.q_stride_h;
  f4 s[ROWS];
  float k[ROWS], q[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t row = y + 16 * i;
    const bool in = row < p.key_dim;
    s[i] = f4{0, 0, 0, 0};
    if (in) {
      const float* from = state + row * p.value_dim;
      if (n == 4) {
        __builtin_memcpy(&s[i], from, sizeof(f4));
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < n) s[i][e] = from[e];
      }
    }
    k[i] = in ? to_f32(kp[row]) : 0.0f;
    q[i] = in ? to_f32(qp[row]) : 0.0f;
  }
  const int64_t gat = r * p.log_decay_stride_r + h * p.log_decay_stride_h;
  const int64_t bat = r * p.beta_stride_r + h * p.beta_stride_h;
  auto element = [](const void* from, int64_t at, int type) {
    return type == CCV1D_F32   ? static_cast<const float*>(from)[at]
           : type == CCV1D_F16 ? (float)static_cast<const _Float16*>(from)[at]
                               : (float)static_cast<const __bf16*>(from)[at];
  };
  const float g = element(p.log_decay, gat, p.log_decay_dtype), beta = element(p.beta, bat, p.beta_dtype);
  const T* vp = static_cast<const T*>(p.v) + r * p.v_stride_r + h * p.v_stride_h + d;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e < n ? to_f32(vp[e]) : 0.0f;
  const bool kept = !(g < -104.0f);  // else exp(g) is zero in fp32, and what the state holds is left behind
  const float a = __builtin_amdgcn_exp2f((float)((double)g * 1.4426950408889634074));
  float t[9] = {};
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[i][e] = kept ? a * s[i][e] : 0.0f;
      t[e] = fmaf(s[i][e], k[i], t[e]);
      t[4 + e] = fmaf(s[i][e], q[i], t[4 + e]);
    }
    t[8] = fmaf(k[i], q[i], t[8]);
  }
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    t[i] += __shfl_xor(t[i], 16);
    t[i] += __shfl_xor(t[i], 32);
  }
  if (lane < 16)
#pragma unroll
    for (int i = 0; i < 9; ++i) sums[w][x][i] = t[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 9; ++i) t[i] = sums[0][x][i] + sums[1][x][i] + sums[2][x][i] + sums[3][x][i];
  f4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = beta * (v[e] - t[e]);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t row = y + 16 * i;
    if (row >= p.key_dim) continue;
    float* to = state + row * p.value_dim;
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = fmaf(k[i], u[e], s[i][e]);
    if (n == 4) {
      __builtin_memcpy(to, &s[i], sizeof(f4));
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < n) to[e] = s[i][e];
    }
  }
  if (y == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) out[e] = (T)(p.scale * fmaf(t[8], u[e], t[4 + e]));
}

int64_t update_cols(const ccv1d_delta_update_args& a) { return (a.value_dim + 63) / 64; }

template <typename T>
hipError_t update_t(const ccv1d_delta_update_args& a, hipStream_t s) {
  const int64_t cols = update_cols(a), grid = a.rows * a.heads * cols, group = a.heads / a.key_heads;
  if (a.key_dim <= 64) return start(&delta_update_kernel<T, 4>, grid, 256, s, a, group, cols);
  if (a.key_dim <= 128) return start(&delta_update_kernel<T, 8>, grid, 256, s, a, group, cols);
  return start(&delta_update_kernel<T, 16>, grid, 256, s, a, group, cols);
}

bool within(int64_t a, int64_t b, int64_t limit) { return a == 0 || b <= limit / a; }

}  // namespace

// Grids below 2^31 workgroups and 2^32 threads, row counts and offsets in a chunk's workspace in 31 bits.
bool delta_fits(const ccv1d_delta_args& a) {
  if (a.seqlen > kMaxGrid || a.value_dim > (1 << 20) || !within(a.batch, a.heads, kMaxGrid)) return false;
  const Sizes z = sizes_of(a);
  if (!within(a.batch * a.heads, z.chunks, kMaxGrid / 1024 - 8)) return false;
  return within((a.batch * a.heads + 7) / 8 * 8, z.tiles, kMaxThreads / 512);
}

size_t delta_saved(const ccv1d_delta_args& a) {
  const Sizes z = sizes_of(a);
  return (size_t)(a.batch * a.heads * z.chunks) * (size_t)((z.dk + CCV1D_DELTA_CHUNK) * z.dvp);
}

size_t delta_workspace(const ccv1d_delta_args& a, bool backward) {
  return (size_t)places_of(a, sizes_of(a), backward).all;
}

hipError_t delta_fwd(const ccv1d_delta_args& a, hipStream_t s) { return run(a, false, s); }
hipError_t delta_bwd(const ccv1d_delta_args& a, hipStream_t s) { return run(a, true, s); }

int64_t delta_update_threads(const ccv1d_delta_update_args& a) { return a.rows * a.heads * update_cols(a) * 256; }

hipError_t delta_update(const ccv1d_delta_update_args& a, hipStream_t s) {
  switch (a.dtype) {
    case CCV1D_BF16: return update_t<__bf16>(a, s);
    case CCV1D_F16: return update_t<_Float16>(a, s);
    default: return update_t<float>(a, s);
  }
}

}  // namespace ops
}  // namespace ccv1d

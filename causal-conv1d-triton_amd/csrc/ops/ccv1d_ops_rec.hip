// Launch of the gated linear recurrence: workspace, the kernels around the main ones, and the form for
// single tokens.
#include "ops_rec_launch.h"

namespace ccv1d {
namespace ops {

namespace {

// 8 B per channel and chunk, and its group's: 2.2 MB at B=4 T=8192 D=1024 forward, 3 to 6 us behind other
// work, the launch being most of it (16-byte stores and twice or half the workgroups make no difference).
__global__ __launch_bounds__(256) void rec_clear_kernel(uint64_t* words, int64_t n) {
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) words[i] = 0;
}

// No rows: the final states are the initial ones, and their gradients likewise; no decay gradient.
__global__ __launch_bounds__(256) void rec_empty_kernel(const float* from, float* to, int64_t n,
                                                        float* zero, int64_t nz) {
  const int64_t stride = (int64_t)gridDim.x * 256;
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (to)
    for (int64_t i = i0; i < n; i += stride) to[i] = from ? from[i] : 0.0f;
  if (zero)
    for (int64_t i = i0; i < nz; i += stride) zero[i] = 0.0f;
}

// ddecay from the chunks' sums: 32 channels a workgroup, thread y adds rows y, y + 32, ..., 8 requested
// at a time, and the 32 sums are added in order. Bound by latency: 512 rows of 1024 channels 4 to 5 us.
__global__ __launch_bounds__(1024) void rec_reduce_kernel(const float* part, int64_t rows, int64_t dim,
                                                          const float* decay, float* ddecay) {
  __shared__ float sums[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t d = (int64_t)blockIdx.x * 32 + x;
  float s = 0.0f;
  if (d < dim) {
    int64_t i = y;
    for (; i + 7 * 32 < rows; i += 8 * 32) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part[(i + 32 * j) * dim + d];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < rows; i += 32) s += part[i * dim + d];
  }
  sums[y][x] = s;
  __syncthreads();
  if (y == 0 && d < dim) {
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) s += sums[j][x];
    ddecay[d] = s * decay_ratio(decay[d]);
  }
}

// One token of a request: four channels a lane, the last lane of a row those that are left. Up to
// 2^17 channels the launch bounds it (3.2 us, with one channel a lane as with four), then memory: 512
// rows of 5376 channels bf16 9.2 us, 4.8 TB/s (one channel a lane 15.8); 2048 rows 33.4 us, 5.3 TB/s (60).
constexpr int kUpdateChannels = 4;

template <typename T, bool DECAY>
__global__ __launch_bounds__(64) void rec_update_kernel(ccv1d_rec_update_args p,
                                                               uint32_t cols, Divisor by_cols) {
  constexpr int CPL = kUpdateChannels;
  using V = VecIO<T, CPL>;
  using S = VecIO<float, CPL>;
  const uint32_t r = divide(blockIdx.x, by_cols);
  const int64_t row = r, d = ((int64_t)(blockIdx.x - r * cols) * 64 + threadIdx.x) * CPL;
  if (d >= p.dim) return;
  const int n = (int)min((int64_t)CPL, p.dim - d);
  const int64_t slot = p.state_indices ? p.state_indices[row] : row;
  T* out = static_cast<T*>(p.out) + row * p.dim + d;
  const bool in = slot >= 0 && slot < p.slots;
  const T* xp = static_cast<const T*>(p.x) + row * p.x_stride + d;
  const T* gp = static_cast<const T*>(p.gate) + row * p.gate_stride + d;
  const T* ip = static_cast<const T*>(p.input_gate) + row * p.input_gate_stride + d;
  float* sp = p.state + (in ? slot : 0) * p.state_stride + d;
  float x[CPL] = {}, g[CPL] = {}, ig[CPL] = {}, h[CPL] = {}, decay[CPL] = {};
  if (in) {
    if (n == CPL) {
      V::unpack(V::ld(xp), x);
      V::unpack(V::ld(gp), g);
      if (p.input_gate) V::unpack(V::ld(ip), ig);
      S::unpack(S::ld(sp), h);
      if constexpr (DECAY) S::unpack(S::ld(p.decay + d), decay);
    } else {
#pragma unroll
      for (int i = 0; i < CPL; ++i)
        if (i < n) {
          x[i] = to_f32(xp[i]);
          g[i] = to_f32(gp[i]);
          if (p.input_gate) ig[i] = to_f32(ip[i]);
          h[i] = sp[i];
          if constexpr (DECAY) decay[i] = p.decay[d + i];
        }
    }
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      float a, beta;
      const float k = DECAY ? decay_rate(decay[i], p.decay_scale) : 0.0f;
      forget<T, DECAY, false>(k, sinh_tail(k), g[i], a, beta);
      float u = beta * x[i];
      if (p.input_gate) u *= sigmoid<T>(ig[i]);
      h[i] = fmaf(a, h[i], u);
    }
  }
  if (n == CPL) {
    if (in) S::st(sp, S::pack(h));
    V::st(out, V::pack(h));
  } else {
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      if (i < n) {
        if (in) sp[i] = h[i];
        out[i] = to_store<T>(h[i]);
      }
  }
}

int64_t update_cols(const ccv1d_rec_update_args& a) {
  constexpr int kColumn = 64 * kUpdateChannels;
  return (a.dim + kColumn - 1) / kColumn;
}

template <typename T>
hipError_t update_t(const ccv1d_rec_update_args& a, hipStream_t s) {
  const int64_t cols = update_cols(a), grid = a.rows * cols;
  return a.decay ? start(&rec_update_kernel<T, true>, grid, 64, s, a, cols, divisor(cols))
                 : start(&rec_update_kernel<T, false>, grid, 64, s, a, cols, divisor(cols));
}

int64_t fill_blocks(int64_t n) {
  const int64_t b = (n + 1023) / 1024;
  return b < 1 ? 1 : b > 2048 ? 2048 : b;
}

struct Plan {
  int64_t chunks, groups, tickets, words, part;  // words of 8 bytes, cleared; floats after them
};

Plan plan_of(int64_t B, int64_t T, int64_t D, bool backward) {
  Plan p;
  const int64_t rows = backward ? kBwdWaves * kBwdRows : kFwdWaves * kFwdRows;
  p.chunks = (T + rows - 1) / rows;
  p.groups = (p.chunks + kRecGroup - 1) / kRecGroup;
  // and a ticket of 4 bytes per wave column, of 64 channels at the least
  p.tickets = B * ((D + kWave - 1) / kWave);
  p.words = p.chunks > 1 ? B * D * (p.chunks + p.groups) + (p.tickets + 1) / 2 : 0;
  p.part = backward ? B * D * p.chunks : 0;
  return p;
}

hipError_t run(const ccv1d_rec_args& a, bool backward, hipStream_t s) {
  if (a.seqlen == 0 || a.batch == 0) {
    const int64_t n = a.batch * a.dim;
    const float* from = backward ? a.dfinal_states : a.initial_states;
    float* to = backward ? a.dinitial_states : a.final_states;
    float* zero = backward ? a.ddecay : nullptr;
    if (!to && !zero) return hipSuccess;
    return start(&rec_empty_kernel, fill_blocks(n), 256, s, from, to, n, zero, a.dim);
  }
  Plan pl = plan_of(a.batch, a.seqlen, a.dim, backward);
  if (rec_one_chunk(a, backward)) pl.chunks = 1, pl.words = 0;
  RecParams p{};
  p.a = a;
  p.chunks = (int32_t)pl.chunks;
  p.groups = (int32_t)pl.groups;
  p.wide_ids = a.seq_idx_64 != 0;
  p.pairs = static_cast<uint64_t*>(a.workspace);
  p.part = reinterpret_cast<float*>(p.pairs + pl.words);
  if (pl.words) {
    p.states = p.pairs + a.batch * a.dim * pl.chunks;
    p.tickets = reinterpret_cast<uint32_t*>(p.states + a.batch * a.dim * pl.groups);
    const hipError_t err = start(&rec_clear_kernel, fill_blocks(pl.words), 256, s, p.pairs, pl.words);
    if (err != hipSuccess) return err;
  }
  hipError_t e;
  switch (a.dtype) {
    case CCV1D_BF16: e = rec_launch_bf16(p, backward, s); break;
    case CCV1D_F16: e = rec_launch_f16(p, backward, s); break;
    default: e = rec_launch_f32(p, backward, s); break;
  }
  if (e != hipSuccess || !backward || !a.decay) return e;
  return start(&rec_reduce_kernel, (a.dim + 31) / 32, 1024, s, (const float*)p.part, a.batch * pl.chunks,
               a.dim, a.decay, a.ddecay);
}

}  // namespace

size_t rec_workspace(int64_t B, int64_t T, int64_t D, bool backward) {
  const Plan p = plan_of(B, T, D, backward);
  return (size_t)p.words * 8 + (size_t)p.part * 4;
}

int64_t rec_threads(const ccv1d_rec_args& a, bool backward) {
  const int64_t width = kWave * (a.dtype == CCV1D_F32 || a.dim == 1 ? 1 : 2);  // as the launches take it
  const int64_t columns = a.batch * ((a.dim + width - 1) / width);
  const int64_t main = rec_one_chunk(a, backward)
                           ? columns * kWideWaves * kWave
                           : columns * plan_of(a.batch, a.seqlen, a.dim, backward).chunks *
                                 (backward ? kBwdWaves : kFwdWaves) * kWave;
  const int64_t sum = backward && a.decay ? (a.dim + 31) / 32 * 1024 : 0;
  return main > sum ? main : sum;
}

int64_t rec_update_threads(const ccv1d_rec_update_args& a) { return a.rows * update_cols(a) * 64; }

hipError_t rec_fwd(const ccv1d_rec_args& a, hipStream_t s) { return run(a, false, s); }
hipError_t rec_bwd(const ccv1d_rec_args& a, hipStream_t s) { return run(a, true, s); }

hipError_t rec_update(const ccv1d_rec_update_args& a, hipStream_t s) {
  switch (a.dtype) {
    case CCV1D_BF16: return update_t<__bf16>(a, s);
    case CCV1D_F16: return update_t<_Float16>(a, s);
    default: return update_t<float>(a, s);
  }
}

}  // namespace ops
}  // namespace ccv1d

// Launch of the norms around a block, and the sums of their weights' gradients.
#include "ops_norm_launch.h"

namespace ccv1d {
namespace ops {

namespace {

// The weights' gradients from the workgroups' lines: 32 columns a workgroup, thread y adds lines y, y + 32, ...,
// and the 32 sums are added in order. No lines (no rows): zero.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(NormParams p, int32_t lines) {
  __shared__ float sums[32][33];
  const ccv1d_norm_args& a = p.a;
  const int which = blockIdx.x % 3;
  void* to = which == 0 ? a.dpost_weight : which == 1 ? a.dscale_weight : a.dpre_weight;
  const int type = which == 0 ? a.post_dtype : which == 1 ? a.scale_dtype : a.pre_dtype;
  if (!to) return;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t d = (int64_t)(blockIdx.x / 3) * 32 + x;
  float s = 0.0f;
  if (d < a.dim) {
    const float* at = p.lines + which * a.dim + d;
    const int64_t line = 3 * a.dim;
    int n = y;
    for (; n + 7 * 32 < lines; n += 8 * 32) {  // eight requested at a time
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = at[(n + 32 * j) * line];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; n < lines; n += 32) s += at[n * line];
  }
  sums[y][x] = s;
  __syncthreads();
  if (y == 0 && d < a.dim) {
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) s += sums[j][x];
    if (type == CCV1D_F32) static_cast<float*>(to)[d] = s;
    else if (type == CCV1D_F16) static_cast<_Float16*>(to)[d] = (_Float16)s;
    else static_cast<__bf16*>(to)[d] = (__bf16)s;
  }
}

hipError_t run(const ccv1d_norm_args& a, bool backward, hipStream_t s) {
  NormParams p{};
  p.a = a;
  p.rows = a.outer * a.inner;
  p.by_dim = 1.0f / (float)a.dim;
  p.lines = static_cast<float*>(a.workspace);
  hipError_t e = hipSuccess;
  if (p.rows > 0) {
    switch (a.dtype) {
      case CCV1D_BF16: e = norm_launch_bf16(p, backward, s); break;
      case CCV1D_F16: e = norm_launch_f16(p, backward, s); break;
      default: e = norm_launch_f32(p, backward, s); break;
    }
  }
  if (e != hipSuccess || !backward) return e;
  const int32_t lines = p.rows > 0 ? (int32_t)norm_lines(a) : 0;
  return start(&norm_reduce_kernel, (a.dim + 31) / 32 * 3, 1024, s, p, lines);
}

}  // namespace

int64_t norm_threads(const ccv1d_norm_args& a) {
  const int64_t groups = (a.outer * a.inner + norm_at_once(a.dim) - 1) / norm_at_once(a.dim);
  return groups * norm_lanes(a.dim) * norm_at_once(a.dim);
}

size_t norm_workspace(const ccv1d_norm_args& a) { return (size_t)norm_lines(a) * 3 * (size_t)a.dim * 4; }

hipError_t norm_fwd(const ccv1d_norm_args& a, hipStream_t s) { return run(a, false, s); }
hipError_t norm_bwd(const ccv1d_norm_args& a, hipStream_t s) { return run(a, true, s); }

}  // namespace ops
}  // namespace ccv1d

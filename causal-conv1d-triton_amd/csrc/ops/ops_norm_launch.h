// Launch parameters of the norms, shared by their units.
#pragma once

#include "ops_common.h"

namespace ccv1d {
namespace ops {

struct NormParams {
  ccv1d_norm_args a;
  int64_t rows;
  float by_dim;
  float* lines;  // backward: (lines, 3, dim)
};

// Lanes of a row, and rows that a workgroup has at once.
inline int norm_lanes(int64_t dim) { return dim <= 128 ? 16 : dim <= 512 ? 64 : dim <= 2048 ? 256 : 512; }
inline int norm_at_once(int64_t dim) { return norm_lanes(dim) < 256 ? 256 / norm_lanes(dim) : 1; }

// Workgroups of the backward, each of which leaves a line of sums.
constexpr int64_t kNormLines = 1024;
inline int64_t norm_lines(const ccv1d_norm_args& a) {
  const int64_t n = (a.outer * a.inner + norm_at_once(a.dim) - 1) / norm_at_once(a.dim);
  return n < kNormLines ? n : kNormLines;
}

hipError_t norm_launch_bf16(const NormParams& p, bool backward, hipStream_t s);
hipError_t norm_launch_f16(const NormParams& p, bool backward, hipStream_t s);
hipError_t norm_launch_f32(const NormParams& p, bool backward, hipStream_t s);

}  // namespace ops
}  // namespace ccv1d

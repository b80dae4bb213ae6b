// Norms around a block, f32 elements.
#include "ops_norm.h"

namespace ccv1d {
namespace ops {
hipError_t norm_launch_f32(const NormParams& p, bool backward, hipStream_t s) {
  return norm_types<float, float>(p, backward, s);
}
}  // namespace ops
}  // namespace ccv1d

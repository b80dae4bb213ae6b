// Norms around a block, f16 elements.
#include "ops_norm.h"

namespace ccv1d {
namespace ops {
hipError_t norm_launch_f16(const NormParams& p, bool backward, hipStream_t s) {
  if (p.a.residual_dtype != p.a.dtype) return norm_types<_Float16, float>(p, backward, s);
  return norm_types<_Float16, _Float16>(p, backward, s);
}
}  // namespace ops
}  // namespace ccv1d

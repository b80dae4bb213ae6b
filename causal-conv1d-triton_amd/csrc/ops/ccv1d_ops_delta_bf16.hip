// The gated delta rule over whole sequences, bf16 elements.
#include "ops_delta.h"

namespace ccv1d {
namespace ops {
hipError_t delta_launch_bf16(const DeltaParams& p, bool backward, hipStream_t s) {
  return delta_launch<__bf16>(p, backward, s);
}
}  // namespace ops
}  // namespace ccv1d

#include "ops_rec_launch.h"

namespace ccv1d {
namespace ops {

// One channel a lane, 256 bytes a row and wave.
hipError_t rec_launch_f32(const RecParams& p, bool backward, hipStream_t s) {
  return rec_launch<float, 1>(p, backward, s);
}

}  // namespace ops
}  // namespace ccv1d

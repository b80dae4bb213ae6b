#include "ops_rec_launch.h"

namespace ccv1d {
namespace ops {

// Two channels a lane, 256 bytes a row and wave; a single channel has no pair.
hipError_t rec_launch_f16(const RecParams& p, bool backward, hipStream_t s) {
  return p.a.dim == 1 ? rec_launch<_Float16, 1>(p, backward, s) : rec_launch<_Float16, 2>(p, backward, s);
}

}  // namespace ops
}  // namespace ccv1d

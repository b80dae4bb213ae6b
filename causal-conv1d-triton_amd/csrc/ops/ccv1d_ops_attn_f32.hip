#include "ops_attn.h"

namespace ccv1d {
namespace ops {

hipError_t paged_attn_f32(const AttnParams& p, int mode, hipStream_t s) {
  return paged_attn_type<float>(p, mode, s);
}

}  // namespace ops
}  // namespace ccv1d

#include "ops_attn.h"

namespace ccv1d {
namespace ops {

hipError_t paged_attn_f16(const AttnParams& p, int mode, hipStream_t s) {
  return paged_attn_type<_Float16>(p, mode, s);
}

}  // namespace ops
}  // namespace ccv1d

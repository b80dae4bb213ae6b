#include "ops_attn.h"

namespace ccv1d {
namespace ops {

hipError_t paged_attn_bf16(const AttnParams& p, int mode, hipStream_t s) {
  return paged_attn_type<__bf16>(p, mode, s);
}

}  // namespace ops
}  // namespace ccv1d

// Launch parameters of the gated delta rule, shared by its units.
#pragma once

#include "ops_common.h"

namespace ccv1d {
namespace ops {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct DeltaParams {
  ccv1d_delta_args a;
  int32_t chunks, group;  // of a sequence; heads of a key head
  int32_t prep_heads;     // of a key head in one workgroup of the first kernel
  int32_t dk;             // key_dim as the kernels have it: 64, 128 or 256
  int32_t dvp, tiles;     // value_dim up to a multiple of 32; its groups of 16
  // Workspace, in 16-byte units a lane: fragments of k and q by rows, k and q by elements (per key head's chunk),
  // T and P (per head's chunk), the rows' factors
  u4 *kf, *qf, *kt, *qt, *tf, *pf;
  float* rows;
  float *s0, *u;   // kept by the forward for the backward: (.., dk, dvp) and (.., 64, dvp); or null
  float *ds, *dr;  // the backward's, alike
  float* gates;    // sums for the gates' gradients, where a key's elements lie in two workgroups
};

// Workgroups of a chain: 8 XCDs, each with every eighth head.
inline int64_t delta_chains(const ccv1d_delta_args& a, int64_t tiles) {
  return 8 * ((a.batch * a.heads + 7) / 8) * tiles;
}

hipError_t delta_launch_bf16(const DeltaParams& p, bool backward, hipStream_t s);
hipError_t delta_launch_f16(const DeltaParams& p, bool backward, hipStream_t s);
hipError_t delta_launch_f32(const DeltaParams& p, bool backward, hipStream_t s);

}  // namespace ops
}  // namespace ccv1d

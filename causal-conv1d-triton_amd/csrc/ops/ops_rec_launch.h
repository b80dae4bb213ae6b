// Launch of the gated recurrence for one element type (a translation unit each).
#pragma once

#include "ops_rec.h"

namespace ccv1d {
namespace ops {

constexpr int kRecFwdRows = 16;  // rows of a wave
constexpr int kRecBwdRows = 8;

template <typename T, int CPL>
hipError_t rec_launch(RecParams p, bool backward, hipStream_t s) {
  const ccv1d_rec_args& a = p.a;
  p.cols = (int32_t)((a.dim + kWave * CPL - 1) / (kWave * CPL));
  const dim3 grid((unsigned)(a.batch * p.cols * p.chunks)), block(kRecWaves * kWave);
  if (backward) {
    if (a.decay && a.input_gate) rec_bwd_kernel<T, CPL, true, true, kRecBwdRows><<<grid, block, 0, s>>>(p);
    else if (a.decay) rec_bwd_kernel<T, CPL, true, false, kRecBwdRows><<<grid, block, 0, s>>>(p);
    else if (a.input_gate) rec_bwd_kernel<T, CPL, false, true, kRecBwdRows><<<grid, block, 0, s>>>(p);
    else rec_bwd_kernel<T, CPL, false, false, kRecBwdRows><<<grid, block, 0, s>>>(p);
  } else {
    if (a.decay && a.input_gate) rec_fwd_kernel<T, CPL, true, true, kRecFwdRows><<<grid, block, 0, s>>>(p);
    else if (a.decay) rec_fwd_kernel<T, CPL, true, false, kRecFwdRows><<<grid, block, 0, s>>>(p);
    else if (a.input_gate) rec_fwd_kernel<T, CPL, false, true, kRecFwdRows><<<grid, block, 0, s>>>(p);
    else rec_fwd_kernel<T, CPL, false, false, kRecFwdRows><<<grid, block, 0, s>>>(p);
  }
  return hipGetLastError();
}

hipError_t rec_launch_bf16(const RecParams& p, bool backward, hipStream_t s);
hipError_t rec_launch_f16(const RecParams& p, bool backward, hipStream_t s);
hipError_t rec_launch_f32(const RecParams& p, bool backward, hipStream_t s);

}  // namespace ops
}  // namespace ccv1d

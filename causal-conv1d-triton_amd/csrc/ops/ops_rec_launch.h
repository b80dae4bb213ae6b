// Launch of the gated recurrence for one element type (a translation unit each).
#pragma once

#include "ops_rec.h"

namespace ccv1d {
namespace ops {

// Waves of a workgroup and rows of a wave.
constexpr int kFwdWaves = 8, kFwdRows = 16;
constexpr int kBwdWaves = 8, kBwdRows = 8;

template <typename T, int CPL>
hipError_t rec_launch(RecParams p, bool backward, hipStream_t s) {
  const ccv1d_rec_args& a = p.a;
  p.cols = (int32_t)((a.dim + kWave * CPL - 1) / (kWave * CPL));
  const dim3 grid((unsigned)(a.batch * p.cols * p.chunks));
  const dim3 block((backward ? kBwdWaves : kFwdWaves) * kWave);
  auto with = [&](auto decay, auto input_gate, auto seq) {
    constexpr bool kDecay = decltype(decay)::value, kGate = decltype(input_gate)::value;
    constexpr bool kSeq = decltype(seq)::value;
    if (backward)
      rec_bwd_kernel<T, CPL, kDecay, kGate, kSeq, kBwdWaves, kBwdRows><<<grid, block, 0, s>>>(p);
    else
      rec_fwd_kernel<T, CPL, kDecay, kGate, kSeq, kFwdWaves, kFwdRows><<<grid, block, 0, s>>>(p);
  };
  auto with_gate = [&](auto decay, auto seq) {
    if (a.input_gate) with(decay, std::true_type{}, seq);
    else with(decay, std::false_type{}, seq);
  };
  auto with_seq = [&](auto decay) {
    if (a.seq_idx) with_gate(decay, std::true_type{});
    else with_gate(decay, std::false_type{});
  };
  if (a.decay) with_seq(std::true_type{});
  else with_seq(std::false_type{});
  return hipGetLastError();
}

hipError_t rec_launch_bf16(const RecParams& p, bool backward, hipStream_t s);
hipError_t rec_launch_f16(const RecParams& p, bool backward, hipStream_t s);
hipError_t rec_launch_f32(const RecParams& p, bool backward, hipStream_t s);

}  // namespace ops
}  // namespace ccv1d

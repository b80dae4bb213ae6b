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
  const int64_t grid = a.batch * p.cols * p.chunks;
  hipError_t status = hipErrorInvalidValue;
  const auto lines = [](const void* at, int64_t stride_b, int64_t stride_t) {
    return !at || (reinterpret_cast<uintptr_t>(at) % 128 == 0 && stride_b * (int64_t)sizeof(T) % 128 == 0 &&
                   stride_t * (int64_t)sizeof(T) % 128 == 0);
  };
  const int64_t sb = a.seqlen * a.dim;
  p.stream = a.dim * (int64_t)sizeof(T) % 128 == 0 && lines(a.x, a.x_stride_b, a.x_stride_t) &&
             lines(a.gate, a.gate_stride_b, a.gate_stride_t) &&
             lines(a.input_gate, a.input_gate_stride_b, a.input_gate_stride_t) &&
             (backward ? lines(a.dout, a.dout_stride_b, a.dout_stride_t) && lines(a.dx, sb, a.dim) &&
                             lines(a.dgate, sb, a.dim) && lines(a.dinput_gate, sb, a.dim)
                       : lines(a.out, sb, a.dim));
  auto run = [&](auto decay, auto input_gate, auto seq, auto stream) {
    constexpr bool kDecay = decltype(decay)::value, kGate = decltype(input_gate)::value;
    constexpr bool kSeq = decltype(seq)::value, kStream = decltype(stream)::value;
    if (backward)
      status = start(&rec_bwd_kernel<T, CPL, kDecay, kGate, kSeq, kStream, kBwdWaves, kBwdRows>, grid,
                     kBwdWaves * kWave, s, p);
    else
      status = start(&rec_fwd_kernel<T, CPL, kDecay, kGate, kSeq, kStream, kFwdWaves, kFwdRows>, grid,
                     kFwdWaves * kWave, s, p);
  };
  // A flag at a time becomes a type.
  auto choose = [](bool flag, auto&& then) {
    if (flag) then(std::true_type{});
    else then(std::false_type{});
  };
  choose(a.decay != nullptr, [&](auto decay) {
    choose(a.input_gate != nullptr, [&](auto gate) {
      choose(a.seq_idx != nullptr, [&](auto seq) {
        if constexpr (CPL * sizeof(T) >= 4)
          choose(p.stream, [&](auto stream) { run(decay, gate, seq, stream); });
        else  // a single channel
          run(decay, gate, seq, std::false_type{});
      });
    });
  });
  return status;
}

hipError_t rec_launch_bf16(const RecParams& p, bool backward, hipStream_t s);
hipError_t rec_launch_f16(const RecParams& p, bool backward, hipStream_t s);
hipError_t rec_launch_f32(const RecParams& p, bool backward, hipStream_t s);

}  // namespace ops
}  // namespace ccv1d

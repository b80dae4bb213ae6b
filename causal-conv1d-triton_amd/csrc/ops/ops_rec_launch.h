// Launch of the gated recurrence for one element type (a translation unit each).
#pragma once

#include "ops_rec.h"

namespace ccv1d {
namespace ops {

// Waves of a workgroup and rows of a wave.
constexpr int kFwdWaves = 8, kFwdRows = 16;
constexpr int kBwdWaves = 8, kBwdRows = 8;
// Rows of one chunk of 16 waves.
constexpr int kWideWaves = 16, kWideRows = kWideWaves * kFwdRows;

// Forward of 129 to 256 rows in one chunk of twice the waves: no words to clear and no wait for another
// chunk, but one workgroup a CU. B=16 T=256 D=2048 bf16 18.5 us in two chunks, 16.0 in one (14.6 since); D=1024
// without decay 9.9, 8.2; B=64 T=200 61.9, 58; few columns leave CUs idle (B=4 T=256 D=2048 12.2, 12.7;
// B=2 D=512 11.4, 12.0), hence the bound of a wave column for every other CU. Shorter rows are one chunk as
// it is (B=16 T=128 10 us in 8 waves, 14 in 16).
inline bool rec_one_chunk(const ccv1d_rec_args& a, bool backward) {
  const int64_t columns = a.dtype == CCV1D_F32 ? kWave : 2 * kWave;
  return !backward && a.seqlen > kFwdWaves * kFwdRows && a.seqlen <= kWideRows &&
         a.batch * ((a.dim + columns - 1) / columns) >= 128;
}

template <typename T, int CPL>
hipError_t rec_launch(RecParams p, bool backward, hipStream_t s) {
  const ccv1d_rec_args& a = p.a;
  p.cols = (int32_t)((a.dim + kWave * CPL - 1) / (kWave * CPL));
  p.by_cols = divisor(p.cols);
  p.by_columns = divisor(a.batch * p.cols);
  const int64_t grid = a.batch * p.cols * p.chunks;  // chunks: 1 where rec_one_chunk holds
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
    else if (rec_one_chunk(a, backward))
      status = start(&rec_fwd_kernel<T, CPL, kDecay, kGate, kSeq, kStream, kWideWaves, kFwdRows>, grid,
                     kWideWaves * kWave, s, p);
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

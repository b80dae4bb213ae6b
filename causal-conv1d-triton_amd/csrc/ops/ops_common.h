// Shared by the operators around the convolution: element access, launch helpers and the launchers
// that the C ABI (ccv1d_ops_api.hip) calls after it has checked the arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>

#include "ccv1d_layer.h"
#include "ccv1d_ops.h"

namespace ccv1d {

// Defined in ccv1d_api.hip: the thread-local message behind ccv1d_last_error().
int report_error(int code, const char* message);
void clear_error();

namespace ops {

constexpr int kWave = 64;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}

// x / d for 0 <= x < 2^31 and 1 <= d < 2^31 as a product: with magic = 2^(31 + s) / d rounded up, 2^s the
// power of two from d on, the excess is below d <= 2^s and stays below 2^(31 + s) times any x.
struct Divisor {
  uint32_t magic, shift;
};

inline Divisor divisor(int64_t d) {
  uint32_t s = 0;
  while ((int64_t(1) << s) < d) ++s;
  const uint64_t one = uint64_t(1) << (31 + s);
  return {(uint32_t)((one + (uint64_t)d - 1) / (uint64_t)d), 31 + s};
}

__device__ __forceinline__ uint32_t divide(uint32_t x, Divisor d) {
  return (uint32_t)(((uint64_t)x * d.magic) >> d.shift);
}

// Launches a kernel; the status is this launch's own.
template <typename... P, typename... A>
hipError_t start(void (*kernel)(P...), int64_t grid, int block, hipStream_t s, const A&... args) {
  std::tuple<P...> held(static_cast<P>(args)...);
  return std::apply(
      [&](P&... a) {
        void* at[] = {(void*)&a...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((unsigned)grid),
                               dim3((unsigned)block), at, 0, s);
      },
      held);
}

// Threads of a call's largest launch, which have to be fewer than 2^32.
int64_t rec_threads(const ccv1d_rec_args& a, bool backward);
int64_t rec_update_threads(const ccv1d_rec_update_args& a);
int64_t paged_write_threads(const ccv1d_paged_write_args& a);

// Launchers (arguments checked, device current).
hipError_t rec_fwd(const ccv1d_rec_args& a, hipStream_t s);
hipError_t rec_bwd(const ccv1d_rec_args& a, hipStream_t s);
size_t rec_workspace(int64_t B, int64_t T, int64_t D, bool backward);
hipError_t rec_update(const ccv1d_rec_update_args& a, hipStream_t s);
hipError_t paged_plan(const ccv1d_paged_plan_args& a, hipStream_t s);
hipError_t paged_write(const ccv1d_paged_write_args& a, hipStream_t s);
hipError_t paged_attn(const ccv1d_paged_attn_args& a, hipStream_t s);
size_t paged_attn_workspace(const ccv1d_paged_attn_args& a);
bool delta_fits(const ccv1d_delta_args& a);  // whether its launches and sizes are in range
size_t delta_saved(const ccv1d_delta_args& a);
size_t delta_workspace(const ccv1d_delta_args& a, bool backward);
hipError_t delta_fwd(const ccv1d_delta_args& a, hipStream_t s);
hipError_t delta_bwd(const ccv1d_delta_args& a, hipStream_t s);
int64_t delta_update_threads(const ccv1d_delta_update_args& a);
hipError_t delta_update(const ccv1d_delta_update_args& a, hipStream_t s);
int64_t norm_threads(const ccv1d_norm_args& a);
size_t norm_workspace(const ccv1d_norm_args& a);
hipError_t norm_fwd(const ccv1d_norm_args& a, hipStream_t s);
hipError_t norm_bwd(const ccv1d_norm_args& a, hipStream_t s);

}  // namespace ops
}  // namespace ccv1d

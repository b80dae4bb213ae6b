// Attention of one token per row over a paged cache: a wave per (row, query head), its lanes along
// the head's elements, one position after the other with the running maximum and sum of a softmax.
#include "ops_common.h"

namespace ccv1d {
namespace ops {

namespace {

template <typename T>
__global__ __launch_bounds__(64) void paged_attn_kernel(ccv1d_paged_attn_args p) {
  const int64_t row = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads;
  const int64_t kvh = head / (p.q_heads / p.kv_heads);
  const int lane = threadIdx.x, Dh = (int)p.head_dim;
  float q[4], o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 64 * j;
    q[j] = d < Dh ? to_f32(static_cast<const T*>(p.q)[row * p.q_stride_r + head * p.q_stride_h + d]) : 0;
  }
  const int64_t req = p.request_ids ? p.request_ids[row] : row;
  int64_t len = req >= 0 && req < p.requests ? p.seq_lens[row] : 0;
  len = min(len, p.max_pages * p.page_size);
  const int64_t first = p.window && len > p.window ? len - p.window : 0;
  float m = -3.4028235e38f, l = 0.0f;  // finite, so that no difference of infinities arises
  for (int64_t t = first; t < len; ++t) {
    const int64_t page = p.block_tables[req * p.block_table_stride + t / p.page_size];
    if (page < 0 || page >= p.num_pages) continue;
    const int64_t off = t % p.page_size;
    const T* k = static_cast<const T*>(p.k_cache) + page * p.k_cache_stride_p + off * p.k_cache_stride_t +
                 kvh * p.k_cache_stride_h;
    const T* v = static_cast<const T*>(p.v_cache) + page * p.v_cache_stride_p + off * p.v_cache_stride_t +
                 kvh * p.v_cache_stride_h;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 64 * j;
      if (d < Dh) s = fmaf(q[j], to_f32(k[d]), s);
    }
#pragma unroll
    for (int w = 32; w; w /= 2) s += __shfl_xor(s, w);
    s *= p.scale;
    const float mn = fmaxf(m, s);
    const float f = expf(m - mn), e = expf(s - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 64 * j;
      if (d < Dh) o[j] = o[j] * f + e * to_f32(v[d]);
    }
  }
  T* out = static_cast<T*>(p.out) + (row * p.q_heads + head) * Dh;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 64 * j;
    if (d < Dh) out[d] = static_cast<T>(l > 0.0f ? o[j] / l : l == 0.0f ? 0.0f : l);
  }
  if (p.lse && lane == 0) p.lse[row * p.q_heads + head] = m + logf(l);
}

}  // namespace

size_t paged_attn_workspace(const ccv1d_paged_attn_args&) { return 0; }

hipError_t paged_attn(const ccv1d_paged_attn_args& a, hipStream_t s) {
  const unsigned grid = (unsigned)(a.rows * a.q_heads);
  switch (a.dtype) {
    case CCV1D_BF16: paged_attn_kernel<__bf16><<<grid, 64, 0, s>>>(a); break;
    case CCV1D_F16: paged_attn_kernel<_Float16><<<grid, 64, 0, s>>>(a); break;
    default: paged_attn_kernel<float><<<grid, 64, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

}  // namespace ops
}  // namespace ccv1d

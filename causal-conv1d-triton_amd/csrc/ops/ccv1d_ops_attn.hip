// Launch of the paged attention: how rows are split, and the join of their spans.
#include "ops_attn.h"

namespace ccv1d {
namespace ops {

namespace {

// Joins the spans of a row and query head: 4 waves take the spans in turn, 64 lanes the elements, and
// the waves' sums meet in LDS. Rows of one span have been written by the main kernel.
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(AttnParams p) {
  const ccv1d_paged_attn_args& a = p.a;
  const int64_t at = blockIdx.x, row = at / a.q_heads;
  int64_t request;
  const Span sp = span_of(p, row, request);
  const int spans = (sp.end - sp.base + p.span - 1) / p.span;
  if (spans <= 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, Dh = (int)a.head_dim;
  const float* ml = p.part_ml + at * p.splits * 2;
  const float* part = p.part + at * p.splits * Dh;
  float top = kLowest;
  for (int i = lane; i < spans; i += 64) top = fmaxf(top, ml[2 * i]);
#pragma unroll
  for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
  float total = 0.0f, sum[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = wave; i < spans; i += 4) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * i] - top);
    total = fmaf(ml[2 * i + 1], f, total);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lane + 64 * j < Dh) sum[j] = fmaf(part[(int64_t)i * Dh + lane + 64 * j], f, sum[j]);
  }
  __shared__ float s_sum[4][256], s_total[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) s_sum[wave][lane + 64 * j] = sum[j];
  if (lane == 0) s_total[wave] = total;
  __syncthreads();
  total = s_total[0] + s_total[1] + s_total[2] + s_total[3];
  const int d = threadIdx.x;
  if (d < Dh) {
    const float s = s_sum[0][d] + s_sum[1][d] + s_sum[2][d] + s_sum[3][d];
    static_cast<T*>(a.out)[at * Dh + d] = static_cast<T>(total == 0.0f ? 0.0f : s / total);
  }
  if (a.lse && d == 0) a.lse[at] = (top + __log2f(total)) * 0.69314718055994530942f;
}

AttnParams plan(const ccv1d_paged_attn_args& a) {
  AttnParams p{};
  p.a = a;
  uint32_t s = 0;
  while ((int64_t(1) << s) < a.page_size) ++s;
  p.by_page.shift = 31 + s;
  p.by_page.magic = (uint32_t)(((uint64_t(1) << p.by_page.shift) + (uint64_t)a.page_size - 1) /
                               (uint64_t)a.page_size);
  const int64_t group = a.q_heads / a.kv_heads;
  p.tiles = (int32_t)((group + kAttnHeads - 1) / kAttnHeads);
  int64_t limit = a.max_pages * a.page_size;
  if (a.max_seq_len && a.max_seq_len < limit) limit = a.max_seq_len;
  p.limit = (int32_t)limit;
  // Spans: as many as fill the card with 1024 workgroups, of at least two steps a wave (256
  // positions), and of at most 2048 positions, so that one long row beside short ones is spread too;
  // at most 256 of them.
  int64_t most = a.window && a.window + 31 < limit ? a.window + 31 : limit;
  if (most < 1) most = 1;
  const int64_t wgs = a.rows * a.kv_heads * p.tiles;
  int64_t splits = (1024 + wgs - 1) / wgs;
  int64_t span = (most + splits - 1) / splits;
  if (span > 2048) span = 2048;
  if (span < 256) span = 256;
  if (span < (most + 255) / 256) span = (most + 255) / 256;
  span = (span + 127) / 128 * 128;
  p.span = (int32_t)span;
  p.splits = (int32_t)((most + span - 1) / span);
  return p;
}

}  // namespace

size_t paged_attn_workspace(const ccv1d_paged_attn_args& a) {
  const AttnParams p = plan(a);
  if (p.splits <= 1) return 0;
  return (size_t)(a.rows * a.q_heads * p.splits * (a.head_dim + 2)) * 4;
}

hipError_t paged_attn(const ccv1d_paged_attn_args& a, hipStream_t s) {
  AttnParams p = plan(a);
  p.part = static_cast<float*>(a.workspace);
  p.part_ml = p.part + a.rows * a.q_heads * p.splits * a.head_dim;
  const int step = a.dtype == CCV1D_F32 ? 16 : 32;
  const int mode = a.page_size % step == 0 ? kPageStep : a.page_size % 4 == 0 ? kPageFour : kPageAny;
  hipError_t e;
  switch (a.dtype) {
    case CCV1D_BF16: e = paged_attn_bf16(p, mode, s); break;
    case CCV1D_F16: e = paged_attn_f16(p, mode, s); break;
    default: e = paged_attn_f32(p, mode, s); break;
  }
  if (e != hipSuccess || p.splits <= 1) return e;
  const unsigned grid = (unsigned)(a.rows * a.q_heads);
  switch (a.dtype) {
    case CCV1D_BF16: paged_join_kernel<__bf16><<<grid, 256, 0, s>>>(p); break;
    case CCV1D_F16: paged_join_kernel<_Float16><<<grid, 256, 0, s>>>(p); break;
    default: paged_join_kernel<float><<<grid, 256, 0, s>>>(p); break;
  }
  return hipGetLastError();
}

}  // namespace ops
}  // namespace ccv1d

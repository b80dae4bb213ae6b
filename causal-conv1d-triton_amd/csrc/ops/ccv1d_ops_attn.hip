// Launch of the paged attention: how rows are split, and the join of their spans.
#include "ops_attn.h"

namespace ccv1d {
namespace ops {

namespace {

// Joins the spans of a row and query head: the workgroup's waves (kJoinWaves at most, one for
// kJoinSpans spans where there are fewer) take the spans in turn, 64 lanes the elements, and the waves'
// sums meet in LDS.
// Rows of one span have been written by the main kernel. Bound by its two dependent reads (the length,
// then maxima and sums together): two rows of 128 spans and 32 heads of 128 take 6 us (4 waves that read
// the maxima first 17); many rows by their workgroups' waves: with a wave a span, 64 rows of 8 spans made the
// whole call 225 us, with one for 4 222, and 32 rows of 64 heads of 64 and 8 spans 43 and 39.
constexpr int kJoinWaves = 16, kJoinSpans = 4;

template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void paged_join_kernel(AttnParams p) {
  __shared__ float s_sum[kJoinWaves][256], s_total[kJoinWaves];
  const ccv1d_paged_attn_args& a = p.a;
  const int64_t at = blockIdx.x, row = divide(blockIdx.x, p.by_q_heads);
  int64_t request;
  const Span sp = span_of(p, row, request);
  const int spans = (int)divide(sp.end - sp.base + p.span - 1, p.by_span);
  if (spans <= 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int Dh = (int)a.head_dim;
  const float* ml = p.part_ml + at * p.splits * 2;
  const float* part = p.part + at * p.splits * Dh;
  float top = kLowest, total = 0.0f, sum[4] = {0, 0, 0, 0};
  constexpr int kBatch = 8;  // spans of a wave that are requested together, the first before the maxima
  for (int i0 = wave; i0 < spans; i0 += kBatch * waves) {
    float v[kBatch][4];
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const float* from = part + (int64_t)min(i0 + n * waves, spans - 1) * Dh;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[n][j] = lane + 64 * j < Dh ? from[lane + 64 * j] : 0.0f;
    }
    if (i0 == wave) {
      for (int i = lane; i < spans; i += 64) top = fmaxf(top, ml[2 * i]);
#pragma unroll
      for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    }
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int i = i0 + n * waves;
      if (i < spans) {
        const float f = __builtin_amdgcn_exp2f(ml[2 * i] - top);
        total = fmaf(ml[2 * i + 1], f, total);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = fmaf(v[n][j], f, sum[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s_sum[wave][lane + 64 * j] = sum[j];
  if (lane == 0) s_total[wave] = total;
  __syncthreads();
  total = 0.0f;
  for (int w = 0; w < waves; ++w) total += s_total[w];
  for (int d = threadIdx.x; d < Dh; d += blockDim.x) {
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += s_sum[w][d];
    static_cast<T*>(a.out)[at * Dh + d] = static_cast<T>(total == 0.0f ? 0.0f : s / total);
  }
  if (a.lse && threadIdx.x == 0) a.lse[at] = (top + __log2f(total)) * 0.69314718055994530942f;
}

AttnParams plan(const ccv1d_paged_attn_args& a) {
  AttnParams p{};
  p.a = a;
  // A window that no int32 length passes is none (and sums with it stay in range).
  if (a.window >= INT32_MAX) p.a.window = 0;
  const int64_t window = p.a.window;
  p.by_page = divisor(a.page_size);
  p.group = (int32_t)(a.q_heads / a.kv_heads);
  p.tiles = (p.group + kAttnHeads - 1) / kAttnHeads;
  int64_t limit = a.max_pages * a.page_size;
  if (a.max_seq_len && a.max_seq_len < limit) limit = a.max_seq_len;
  p.limit = (int32_t)limit;
  // Spans: as many as make `target` workgroups, twice what the card holds or more, of at least a step of
  // every wave (128 positions) and at most 1024 positions, so that a long row beside short ones is spread
  // too; at most 256 of them. The wider a head, the fewer workgroups hold as many bytes, and the more
  // each writes for the join: 2^18 over the bytes of a row, i.e. 2048, 1024, 512 for 16-bit heads of 64,
  // 128, 256. (Targets 512, 1024, 2048: 64 rows of 512 to 4096 positions, 16 query heads of 256 over 2
  // key heads 77, 79, 88 us, over one 46, 53, 59; 128 rows of 300 to 700, 8 key heads of 128 64, 64, 70;
  // 16 rows of 512 to 4096 of those 47, 43, 42; 32 rows of 1000 to 3000, heads of 64 46, 48, 44. Most
  // positions: 64 requests of 512 to 8192, 8 key heads of 128: 2048 254 us, 1024 228; two rows of 131072:
  // 197, 196. Least: 16 rows of a 1024 window, one key head of 256: 256 15.7 us, 128 13.1.)
  const int64_t row_bytes = a.head_dim * (a.dtype == CCV1D_F32 ? 4 : 2);
  const int64_t target = (int64_t(1) << 18) / row_bytes;
  int64_t most = window && window + 31 < limit ? window + 31 : limit;
  if (most < 1) most = 1;
  const int64_t wgs = a.rows * a.kv_heads * p.tiles;
  int64_t splits = (target + wgs - 1) / wgs;
  int64_t span = (most + splits - 1) / splits;
  if (span > 1024) span = 1024;
  if (span < 128) span = 128;
  // One span, and with it no join, where that saves more than the split: with 256 workgroups, one a CU, up
  // to 1024 positions (and a window's 31 of rounding), with fewer up to 512 positions of 100 KiB of keys.
  // (Split and whole, us, every row of the stated length, then lengths from 1 to it: heads of 128 bf16, 512
  // workgroups, 384 positions 30.2 and 22.9, 19.8 and 15.1; 1024 62.2 and 53.1, 40.2 and 38.4; 256
  // workgroups, 1024 35.9 and 29.2, 24.3 and 25.3; 64 workgroups, 384 9.9 and 9.2, 9.5 and 8.9; 512 10.5
  // and 11.0, 9.6 and 10.7; heads of 64, 64 workgroups, 512 9.0 and 8.9, 8.3 and 7.6; heads of 256, 64
  // workgroups, 200 12.2 and 10.6, 11.7 and 10.0; 384 13.3 and 14.5.)
  if (wgs >= 256 ? most <= 1024 + 31 : most <= 512 && most * row_bytes <= 100 << 10) span = most;
  // The sums of the spans take at most 512 MiB: many rows (a prompt's, say) beside a long table fill the card
  // with fewer spans each. It bounds the workgroups too: below 2^24, as a launch of 256 threads each has to be.
  // (Spans of 1024 and so, 32 query over 8 key heads of 128 bf16, a table of 131072 positions: 1024 rows of 1 to 600
  // 1555 and 311 us, 1023 rows of 300 beside one of 131072 1628 and 487, the 2048 rows of one prompt 4387 and 751;
  // a prompt of 8192 with its own table 17.6 and 11.0 ms.)
  const int64_t sums = a.rows * a.q_heads * (a.head_dim + 2) * 4;
  int64_t spans = (int64_t(512) << 20) / (sums > 0 ? sums : 1);
  if (spans > 256) spans = 256;
  if (spans < 1) spans = 1;
  if (span < (most + spans - 1) / spans) span = (most + spans - 1) / spans;
  span = (span + 127) / 128 * 128;
  p.span = (int32_t)span;
  p.splits = (int32_t)((most + span - 1) / span);
  p.block = (int32_t)(8 * a.kv_heads * p.tiles);
  p.by_block = divisor(p.block);
  p.by_tiles = divisor(p.tiles);
  p.by_kv_heads = divisor(a.kv_heads);
  p.by_splits = divisor(p.splits);
  p.by_q_heads = divisor(a.q_heads);
  p.by_span = divisor(p.span);
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
  const int64_t grid = a.rows * a.q_heads;
  const int waves = (p.splits + kJoinSpans - 1) / kJoinSpans;
  const int block = 64 * (waves < kJoinWaves ? waves : kJoinWaves);
  switch (a.dtype) {
    case CCV1D_BF16: return start(&paged_join_kernel<__bf16>, grid, block, s, p);
    case CCV1D_F16: return start(&paged_join_kernel<_Float16>, grid, block, s, p);
    default: return start(&paged_join_kernel<float>, grid, block, s, p);
  }
}

}  // namespace ops
}  // namespace ccv1d

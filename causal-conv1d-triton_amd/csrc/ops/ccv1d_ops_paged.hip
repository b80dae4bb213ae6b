// The plan of a batch over paged caches, and the write of keys and values into them.
#include "ops_common.h"

namespace ccv1d {
namespace ops {

namespace {

// ---------------------------------------------------------------------------------------------
// Plan. Everything follows from two running sums over the requests: of the new tokens (where a
// request's tokens lie) and of the pages that each needs (which free pages are its own). A launch
// of its own for the sums would cost more than they do, so every workgroup makes them again, 1024
// requests at a time, and then serves its share: every kPlanTokens-th range of token places that
// falls into those requests, and the table rows of every gridDim.x-th of them. Nothing that one
// workgroup writes is read by another: the table entries written are past the cached pages, and
// those read are before them. Bound by latency: the lengths, a scan, a search, the page: 5 us of 16 requests,
// 6 of 512 with 16384 places (11 with 64-bit divisions and 1024 places a workgroup).
// ---------------------------------------------------------------------------------------------

constexpr int kPlanThreads = 256;
constexpr int kPlanItems = 4;
constexpr int kPlanChunk = kPlanThreads * kPlanItems;
constexpr int kPlanTokens = 256;  // token places of a workgroup: one a lane

__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const int64_t w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  return v;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(ccv1d_paged_plan_args p,
                                                                  Divisor by_page) {
  __shared__ int64_t s_wave[2][kPlanThreads / kWave];
  __shared__ int64_t s_start[kPlanChunk];  // first token place of a request
  __shared__ int64_t s_nth[kPlanChunk];    // pages needed by the requests before it
  __shared__ int32_t s_cached[kPlanChunk];
  __shared__ int32_t s_have[kPlanChunk], s_need[kPlanChunk];  // need: -1 when not admitted
  __shared__ int64_t s_used[kPlanThreads / kWave];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t R = p.requests, capacity = p.max_pages * p.page_size;  // below 2^31
  const uint32_t ps = (uint32_t)p.page_size;
  const int64_t free = min((int64_t)max(*p.num_free, 0), p.num_free_pages);
  const int64_t t0 = (int64_t)blockIdx.x * kPlanTokens;
  const int64_t t1 = min(t0 + kPlanTokens, p.max_tokens);
  const bool lead = blockIdx.x == 0;
  int64_t tokens = 0, pages = 0, used = 0;  // over the requests before this chunk; used: my share

  for (int64_t r0 = 0; r0 < R; r0 += kPlanChunk) {
    int32_t c[kPlanItems], n[kPlanItems], have[kPlanItems], need[kPlanItems];
    bool fits[kPlanItems];
    int64_t st = 0, sp = 0;
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int64_t r = r0 + tid * kPlanItems + i;
      c[i] = r < R ? max(p.cached_lens[r], 0) : 0;
      n[i] = r < R ? max(p.new_lens[r], 0) : 0;
      fits[i] = (int64_t)c[i] + n[i] <= capacity;
      have[i] = need[i] = 0;
      if (fits[i]) {
        // pages of x tokens: (x - 1) / ps + 1, none of none
        have[i] = c[i] ? (int32_t)divide(c[i] - 1, by_page) + 1 : 0;
        need[i] = (c[i] + n[i] ? (int32_t)divide(c[i] + n[i] - 1, by_page) + 1 : 0) - have[i];
      }
      st += n[i];
      sp += need[i];
    }
    const int64_t it = wave_scan(st, lane), ip = wave_scan(sp, lane);
    __syncthreads();  // the last chunk's tables have been read
    if (lane == kWave - 1) {
      s_wave[0][wave] = it;
      s_wave[1][wave] = ip;
    }
    __syncthreads();
    int64_t et = tokens + it - st, ep = pages + ip - sp;  // before this lane's first request
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      if (w < wave) {
        et += s_wave[0][w];
        ep += s_wave[1][w];
      }
      tokens += s_wave[0][w];
      pages += s_wave[1][w];
    }
    const int64_t chunk_start = tokens;  // end of this chunk's tokens
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int j = tid * kPlanItems + i;
      const int64_t r = r0 + j;
      const bool ok = fits[i] && (need[i] == 0 || ep + need[i] <= free);
      s_start[j] = et;
      s_nth[j] = ep;
      s_cached[j] = c[i];
      s_have[j] = have[i];
      s_need[j] = ok ? need[i] : -1;
      if (ok && need[i] > 0) used = ep + need[i];
      if (lead && r < R) {
        p.seq_lens[r] = ok ? c[i] + n[i] : c[i];
        p.query_start[r] = (int32_t)et;
      }
      et += n[i];
      ep += need[i];
    }
    __syncthreads();

    // New pages of every gridDim.x-th request, a wave each.
    const int live = (int)min((int64_t)kPlanChunk, R - r0);
    for (int64_t j = blockIdx.x + (int64_t)wave * gridDim.x; j < live;
         j += (int64_t)gridDim.x * (kPlanThreads / kWave)) {
      int32_t* row = p.block_tables + (r0 + j) * p.block_table_stride;
      for (int i = lane; i < s_need[j]; i += kWave)
        row[s_have[j] + i] = p.free_pages[free - 1 - (s_nth[j] + i)];
    }

    // My token places inside this chunk's tokens: the last request that starts at or before each.
    const int64_t lo = max(t0, s_start[0]), hi = min(t1, chunk_start);
    for (int64_t t = lo + tid; t < hi; t += kPlanThreads) {
      int a = 0, b = live;  // s_start[a] <= t < s_start[b]
      while (b - a > 1) {
        const int m = (a + b) / 2;
        if (s_start[m] <= t) a = m;
        else b = m;
      }
      int32_t pos = -1, id = -1;
      int64_t slot = -1;
      if (s_need[a] >= 0) {
        id = (int32_t)(r0 + a);
        pos = s_cached[a] + (int32_t)(t - s_start[a]);
        const uint32_t pg = divide(pos, by_page), off = pos - pg * ps;
        const int32_t page = (int32_t)pg < s_have[a]
                                 ? p.block_tables[(r0 + a) * p.block_table_stride + pg]
                                 : p.free_pages[free - 1 - (s_nth[a] + pg - s_have[a])];
        if (page >= 0) slot = (int64_t)page * ps + off;
      }
      p.positions[t] = pos;
      p.request_ids[t] = id;
      p.slot_mapping[t] = slot;
    }
  }

  for (int64_t t = max(t0, tokens) + tid; t < t1; t += kPlanThreads) {
    p.positions[t] = -1;
    p.request_ids[t] = -1;
    p.slot_mapping[t] = -1;
  }
  if (lead) {
#pragma unroll
    for (int o = kWave / 2; o; o /= 2) used = max(used, (int64_t)__shfl_xor(used, o));
    if (lane == 0) s_used[wave] = used;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kPlanThreads / kWave; ++w) used = max(used, s_used[w]);
      p.query_start[R] = (int32_t)tokens;
      *p.num_free_out = (int32_t)(free - used);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Write: a copy, bound by memory. Lanes go over the pieces of V of a few tokens' keys and values: 16
// bytes where heads are whole numbers of them, else an element. 7168 tokens of 8 heads of 128 (bf16,
// 58.7 MB) take 11.4 us, the rate of a large copy.
// ---------------------------------------------------------------------------------------------

constexpr int kWriteThreads = 256;

template <typename V>
__global__ __launch_bounds__(kWriteThreads) void paged_write_kernel(ccv1d_paged_write_args p, int per_head,
                                                                    int tokens) {
  const int n = (int)p.kv_heads * per_head;  // pieces of a token's keys
  const int es = p.dtype == CCV1D_F32 ? 4 : 2;
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  for (int i = threadIdx.x; i < tokens * 2 * n; i += kWriteThreads) {
    const int64_t token = t0 + i / (2 * n);
    if (token >= p.tokens) return;
    const int64_t slot = p.slot_mapping[token];
    if (slot < 0 || slot >= p.num_pages * p.page_size) continue;
    const int64_t page = slot / p.page_size, off = slot - page * p.page_size;
    int j = i % (2 * n);
    const bool val = j >= n;
    if (val) j -= n;
    const int64_t h = j / per_head, w = j % per_head;
    const char* src = static_cast<const char*>(val ? p.v : p.k);
    char* dst = static_cast<char*>(val ? p.v_cache : p.k_cache);
    const int64_t from = val ? token * p.v_stride_t + h * p.v_stride_h
                             : token * p.k_stride_t + h * p.k_stride_h;
    const int64_t to = val ? page * p.v_cache_stride_p + off * p.v_cache_stride_t + h * p.v_cache_stride_h
                           : page * p.k_cache_stride_p + off * p.k_cache_stride_t + h * p.k_cache_stride_h;
    *reinterpret_cast<V*>(dst + to * es + w * sizeof(V)) =
        *reinterpret_cast<const V*>(src + from * es + w * sizeof(V));
  }
}

// Whether heads are whole numbers of 16-byte pieces.
bool write_wide(const ccv1d_paged_write_args& a) { return a.head_dim % (a.dtype == CCV1D_F32 ? 4 : 8) == 0; }

int write_per_head(const ccv1d_paged_write_args& a) {
  return (int)(a.head_dim * (a.dtype == CCV1D_F32 ? 4 : 2) / (write_wide(a) ? 16 : 2));
}

// Tokens of a workgroup: small ones share it, two pieces a lane.
int write_tokens(const ccv1d_paged_write_args& a) {
  const int64_t pieces = 2 * a.kv_heads * write_per_head(a);
  return pieces < 2 * kWriteThreads ? (int)(2 * kWriteThreads / pieces) : 1;
}

int64_t write_grid(const ccv1d_paged_write_args& a) {
  const int tokens = write_tokens(a);
  return (a.tokens + tokens - 1) / tokens;
}

template <typename V>
hipError_t write_as(const ccv1d_paged_write_args& a, hipStream_t s) {
  return start(&paged_write_kernel<V>, write_grid(a), kWriteThreads, s, a, write_per_head(a), write_tokens(a));
}

}  // namespace

hipError_t paged_plan(const ccv1d_paged_plan_args& a, hipStream_t s) {
  const int64_t blocks = (a.max_tokens + kPlanTokens - 1) / kPlanTokens;
  return start(&paged_plan_kernel, blocks > 0 ? blocks : 1, kPlanThreads, s, a, divisor(a.page_size));
}

hipError_t paged_write(const ccv1d_paged_write_args& a, hipStream_t s) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  return write_wide(a) ? write_as<u4>(a, s) : write_as<uint16_t>(a, s);
}

int64_t paged_write_threads(const ccv1d_paged_write_args& a) { return write_grid(a) * kWriteThreads; }

}  // namespace ops
}  // namespace ccv1d

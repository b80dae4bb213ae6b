// Attention of one token per row over a paged cache.
//
// A workgroup takes one row, one key head with up to 16 of its query heads, and a span of positions;
// its waves take the span's steps of kStep positions in turn, each with a running maximum and sum of
// its own, and join at the end. Spans of one row are joined by a second kernel. The cache is read once
// (once per 16 query heads of a key head), which is what bounds the operator; per position and query
// head there are 4 head_dim operations, so the products run on the matrix cores, where a key head's
// query heads are the columns.
//
// A step's two products, with n = lane % 16 and g = lane / 16 in the 16x16 matrix instructions (first
// operand: row n, second: column n, both at depth g; result: column n, rows 4 g .. 4 g + 3):
//   S = K q:  rows are positions, columns query heads. Lane (n, g) loads position n's elements
//             8 (4 c + g) .. + 7 for c = 0, 1, ..: one 16-byte load is one operand (fp32: 4 elements, one
//             instruction each). It ends up with the scores of positions 4 g .. 4 g + 3 for query head n.
//   O = V p:  rows are elements, columns query heads, the depth positions. The weights of a lane are
//             its scores': with the depth's order chosen as the positions that each g has scores of,
//             they are the second operand where they stand. The first operand needs, for one
//             element, the values of those same positions: a lane loads 16-byte pieces (elements 8 n ..
//             8 n + 7) of each of its positions, and byte permutations turn 8 positions of 8 elements
//             into one operand per element. (The order of elements over rows is free too: it is undone
//             when the result is stored.)
// So neither keys, values, scores nor weights pass through LDS.
//
// fp32 throughout except the operands: q, K and V as they are stored; a weight goes in as 16-bit pieces, since
// one piece's rounding would be as large as that of the result (fp32 caches: as it is). In bf16 the sum of
// three is the fp32 weight (of two 2^-16 of it away, which moves one result in 500 to the next bf16 number; the
// third takes no time: 64 rows of 512 to 8192 positions 229.7 and 228.8 us). In fp16 the sum of two is the weight
// to 2^-22 of it, or to 2^-25 where that is more, the type's smallest step: so a maximum's weight is 2^7 there,
// and what is lost of a weight stays below 2^-32 of the wave's largest (with 1, positions at 2^-25 of a wave's
// largest fell out of the sum). The running
// maximum is raised only when a score passes it by more than 2^8 in weight, which spares most steps the
// reduction across lanes and the scaling of O; the sums hold 2^8, and fp16 pieces 2^15, without loss.
//
// Positions outside [first, end), or in pages outside the cache, have weight zero: their scores are
// dropped, and their values replaced by zeros, since a cache's unused rows may hold anything and zero
// times infinity is no number. Only steps with such positions take that path.
#pragma once

#include "../ccv1d_device.h"
#include "ops_common.h"

namespace ccv1d {
namespace ops {

constexpr int kAttnWaves = 4;
constexpr int kAttnHeads = 16;  // query heads of a workgroup
constexpr float kLowest = -3.402823466e38f;

struct AttnParams {
  ccv1d_paged_attn_args a;
  Divisor by_page, by_block, by_tiles, by_kv_heads, by_splits, by_q_heads, by_span;
  int32_t group;      // query heads of a key head
  int32_t block;      // workgroups of 8 spans of a row, or of neighbouring rows
  int32_t tiles;      // workgroups of kAttnHeads query heads per key head
  int32_t span;       // positions of a workgroup, a multiple of a step of all waves
  int32_t splits;     // most spans of a row
  int32_t limit;      // no position at or past it
  float* part;        // (rows * q_heads, splits, head_dim): sums of a span
  float* part_ml;     // (rows * q_heads, splits, 2): its maximum (base 2) and sum of weights
};

// The positions of a row: [first, end), in spans counted from `base`.
struct Span {
  int32_t first, end, base;
};

// The window is the last of the row's length, also where that passes the table or the bound of the lengths,
// which cut the end off; a window wholly past them leaves nothing.
__device__ __forceinline__ Span span_of(const AttnParams& p, int64_t row, int64_t& request) {
  request = p.a.request_ids ? p.a.request_ids[row] : row;
  Span s{0, 0, 0};
  int32_t length = 0;
  if (request >= 0 && request < p.a.requests && p.a.num_pages > 0) length = max(0, p.a.seq_lens[row]);
  s.end = min(length, p.limit);
  if (p.a.window && length > p.a.window) s.first = length - (int32_t)p.a.window;
  if (s.first >= s.end) s.first = s.end = 0;
  s.base = s.first & ~31;
  return s;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Dwords from any element address.
template <int N, typename T>
__device__ __forceinline__ void load_words(const T* p, uint32_t* to) {
  using V = typename RawOf<4 * N>::type;
  const V v = *reinterpret_cast<const typename AlignedAs<V, (int)sizeof(T)>::type*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) to[i] = v[i];
}

// The shape of a step for an element type.
template <typename T>
struct Step {
  static constexpr int kPer = 4 / (int)sizeof(T);  // elements of a dword
  static constexpr int kStep = 16 * kPer;          // positions of a step: 32 (16 in fp32)
  static constexpr int kMine = 4 * kPer;           // positions that a lane has scores of
};

// A lane's elements of a row of values: DH / 16, in pieces of at most 16 bytes, each the largest power
// of two of elements that is left. A piece of w elements covers 16 w elements of the row, the lane's
// at n w of them; the pieces before it cover 16 times theirs.
template <typename T, int DH>
struct Pieces {
  static constexpr int kElems = DH / 16;
  static constexpr int kWide = 16 / (int)sizeof(T);
  static constexpr int before(int k) {  // elements of the lane in the pieces before piece k
    int done = 0;
    for (int i = 0; i < k; ++i) done += width_at(done);
    return done;
  }
  static constexpr int width(int k) { return width_at(before(k)); }
  static constexpr int width_at(int done) {
    int w = kWide;
    while (w > kElems - done) w /= 2;
    return w;
  }
  static constexpr int count() {
    int k = 0;
    for (int done = 0; done < kElems; ++k) done += width_at(done);
    return k;
  }
  static constexpr int kCount = count();
};

template <typename T>
__device__ __forceinline__ f32x4 product32(const uint32_t* a, const uint32_t* b, f32x4 c) {
  const u32x4 x = {a[0], a[1], a[2], a[3]}, y = {b[0], b[1], b[2], b[3]};
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, x),
                                                   __builtin_bit_cast(bf8, y), c, 0, 0, 0);
  else if constexpr (__is_same(T, _Float16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y),
                                                  c, 0, 0, 0);
  else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
}

// Two fp32 values to a dword of T, what the rounding left over to the next, and so on.
template <typename T, int N>
__device__ __forceinline__ void pieces_of(float a, float b, uint32_t (&to)[N]) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const t2 piece = __builtin_convertvector((f2){a, b}, t2);
    const f2 back = __builtin_convertvector(piece, f2);
    a -= back.x, b -= back.y;
    to[i] = __builtin_bit_cast(uint32_t, piece);
  }
}

// An infinite value times a later piece of zero or below is no number or the other infinity. So an element
// that is no number, though the weights are, is looked at again: it is infinite where all its infinite
// values of a weight above zero have one sign, and none of its values is no number (else 0 is returned). For
// one element, by its lane, in the span of a workgroup; `top` is what its weights are relative to. The launch's
// parameters are read anew, so that the kernel holds none of them for this: held, 10 scalar registers spilled,
// and 16 rows of a 1024 window, one key head of 256, took 13.1 us, 12.9 so (12.7 without this). Values with an
// infinite channel take 6 times as long, infinite throughout 20 times (64 rows of 4096, 8 heads of 128).
template <typename T>
__device__ __forceinline__ float infinite(int64_t row, int split, int head, int d, float top) {
  const AttnParams* args = (const AttnParams*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const AttnParams& p = *args;
  const ccv1d_paged_attn_args& a = p.a;
  int64_t request;
  const Span sp = span_of(p, row, request);
  const int begin = sp.base + split * p.span, end = min(sp.end, begin + p.span), first = max(begin, sp.first);
  const int kvh = head / p.group, Dh = (int)a.head_dim;
  const float to2 = a.scale * 1.44269504088896340736f;
  const T* qp = static_cast<const T*>(a.q) + row * a.q_stride_r + head * a.q_stride_h;
  const T* kc = static_cast<const T*>(a.k_cache) + kvh * a.k_cache_stride_h;
  const T* vc = static_cast<const T*>(a.v_cache) + kvh * a.v_cache_stride_h + d;
  const int32_t* table = a.block_tables + request * a.block_table_stride;
  constexpr int kBatch = 8;  // positions whose values are requested together
  bool plus = false, minus = false;
#pragma unroll 1
  for (int p0 = first; p0 < end; p0 += kBatch) {
    uint32_t up = 0, down = 0;  // bit i: the value of position p0 + i is infinite
    bool none = false;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int pos = min(p0 + i, end - 1), at = (int)divide(pos, p.by_page);
      const uint32_t page = (uint32_t)table[at];
      const bool in = page < (uint64_t)a.num_pages;
      const float v = to_f32(vc[(in ? page : 0) * a.v_cache_stride_p +
                                (pos - at * a.page_size) * a.v_cache_stride_t]);
      up |= (in && v == INFINITY ? 1u : 0u) << i;
      down |= (in && v == -INFINITY ? 1u : 0u) << i;
      none = none || (in && v != v);
    }
    if (none) return 0.0f;
#pragma unroll 1
    for (uint32_t left = up | down; left; left &= left - 1) {
      const int i = __builtin_ctz(left), pos = min(p0 + i, end - 1), at = (int)divide(pos, p.by_page);
      const bool sign = up >> i & 1;
      if (sign ? plus : minus) continue;
      const T* kp = kc + (int64_t)table[at] * a.k_cache_stride_p + (pos - at * a.page_size) * a.k_cache_stride_t;
      float score = 0.0f;
#pragma unroll 1
      for (int e = 0; e < Dh; ++e) score = fmaf(to_f32(qp[e]), to_f32(kp[e]), score);
      const bool weighs = __builtin_amdgcn_exp2f(score * to2 - top) > 0.0f;
      plus = plus || (sign && weighs);
      minus = minus || (!sign && weighs);
    }
    if (plus && minus) return 0.0f;
  }
  return plus ? INFINITY : minus ? -INFINITY : 0.0f;
}

// Measured, with the join: 64 rows of 512 to 8192 positions, 32 query over 8 key heads of 128, bf16, pages of
// 16: 223 to 230 us on different cards, 5.0 to 5.1 TB/s of 1.14 GB, a large copy's rate; two rows of 100001 to
// 131072, fp16, pages of 64: 196 us, 4.8 TB/s. Wide heads with many query heads write and join more per position: 16 query heads of 256
// over 2 key heads, 64 rows of 512 to 4096: 77 us, 3.9 TB/s. One step a wave is latency: 16 rows of a 1024
// window, one key head of 256: 12.9 us, 4 of them the join. fp32: the first with 2.28 GB 388 us, 5.9 TB/s. The
// matrix cores are idle most of the time (6.5 % busy in the first).

// How pages meet steps: one page holds a whole step (page_size a multiple of it); a page holds
// whole groups of 4 positions; anything else.
enum PageMode : int { kPageStep = 0, kPageFour = 1, kPageAny = 2 };

template <typename T, int DH, int MODE>
__global__ __launch_bounds__(kAttnWaves* kWave, sizeof(T) * DH > 768 ? 1 : 2) void paged_attn_kernel(
    AttnParams p) {
  using St = Step<T>;
  using Pc = Pieces<T, DH>;
  constexpr int kStep = St::kStep, kMine = St::kMine, kTiles = kStep / 16;
  constexpr int kChunks = DH * (int)sizeof(T) / 64;  // 16-byte loads of a lane for one position's key
  constexpr int kE = 16 / (int)sizeof(T);            // elements of such a load
  constexpr int kVW = DH / 16 / St::kPer;            // dwords of a lane for one position's values

  const ccv1d_paged_attn_args& a = p.a;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Dh = (int)a.head_dim, group = p.group;
  // Workgroups go to the 8 XCDs in turn: ids are dealt anew so that the key heads of one span, whose rows
  // lie side by side in memory, share an XCD's L2 at the same time (256 rows of 1000 to 3000 positions,
  // heads of 64: 278 -> 246 us). The spans move on by one XCD from 8 to 8, or with 8 spans a row one XCD
  // would get all the last ones, which short rows do not have.
  uint32_t id = blockIdx.x;
  const uint32_t nth = divide(id, p.by_block), start = nth * p.block, in = id - start;
  if (start + p.block <= gridDim.x) id = start + (in + nth) % 8 * (p.block / 8) + in / 8;
  // id = ((row * splits + split) * kv_heads + key head) * tiles + tile
  const uint32_t kvs = divide(id, p.by_tiles), spans = divide(kvs, p.by_kv_heads);
  const int tile = (int)(id - kvs * p.tiles);
  const int64_t kvh = kvs - spans * (uint32_t)a.kv_heads;
  const int64_t row = divide(spans, p.by_splits);
  const int split = (int)(spans - (uint32_t)row * p.splits);

  int64_t request;
  const Span sp = span_of(p, row, request);
  const int64_t head0 = kvh * group + tile * kAttnHeads;
  const int heads = min(kAttnHeads, group - tile * kAttnHeads);
  const int begin = sp.base + split * p.span;
  if (split > 0 && begin >= sp.end) return;
  const int end = min(sp.end, begin + p.span), first = max(begin, sp.first);
  const bool only = sp.base + p.span >= sp.end;  // the row's one span

  uint32_t q[kChunks][4];
  {
    const T* qp = static_cast<const T*>(a.q) + row * a.q_stride_r + (head0 + min(n, heads - 1)) * a.q_stride_h;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int d = (4 * c + g) * kE;
      const bool in = n < heads && d < Dh;
      load_words<4>(qp + (d < Dh ? d : 0), q[c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[c][i] = in ? q[c][i] : 0;
    }
  }

  f32x4 o[Pc::kElems];
#pragma unroll
  for (int j = 0; j < Pc::kElems; ++j) o[j] = (f32x4){0, 0, 0, 0};
  // The weight of a position is 2^(x - m); m is 7 below the maximum in fp16.
  constexpr float kHead = __is_same(T, _Float16) ? 7.0f : 0.0f;
  float m = kLowest, l = 0.0f;
  const float to2 = a.scale * 1.44269504088896340736f;
  const int32_t* table = a.block_tables + request * a.block_table_stride;
  const T* kc = static_cast<const T*>(a.k_cache) + kvh * a.k_cache_stride_h;
  const T* vc = static_cast<const T*>(a.v_cache) + kvh * a.v_cache_stride_h;
  const uint32_t last_page = (uint32_t)a.max_pages - 1, ps = (uint32_t)a.page_size;

  // A position's page (0 for none) and place in it; whether it has one.
  auto locate = [&](uint32_t pos, uint32_t& page, uint32_t& off) {
    const uint32_t i = min(divide(pos, p.by_page), last_page);
    off = pos - i * ps;
    if (off >= ps) off = 0;  // past the table: not attended to
    page = (uint32_t)table[i];
    const bool in = page < (uint64_t)a.num_pages;
    page = in ? page : 0;
    return in;
  };

  for (int p0 = begin + wave * kStep; p0 < end; p0 += kAttnWaves * kStep) {
    // The keys are requested before the places of the values are worked out (64 rows of 512 to 8192
    // positions, 8 key heads of 128: 230.7 us after them, 228.1 so).
    uint32_t kw[kTiles][kChunks][4];
    {
      const T* kp[kTiles];
      uint32_t page, off;
      if constexpr (MODE == kPageStep) {
        locate(p0, page, off);
        const T* kb = kc + (int64_t)page * a.k_cache_stride_p + (int64_t)off * a.k_cache_stride_t;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) kp[t] = kb + (16 * t + n) * a.k_cache_stride_t;
      } else {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          locate(p0 + 16 * t + n, page, off);
          kp[t] = kc + (int64_t)page * a.k_cache_stride_p + (int64_t)off * a.k_cache_stride_t;
        }
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int d = (4 * c + g) * kE;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) load_words<4>(kp[t] + (d < Dh ? d : 0), kw[t][c]);
      }
    }
    const T* vp[kMine];
    uint32_t ok = 0;  // bit e: my position e counts
    if constexpr (MODE == kPageStep) {
      uint32_t page, off;
      const bool in = locate(p0, page, off);
      const T* vb = vc + (int64_t)page * a.v_cache_stride_p + (int64_t)off * a.v_cache_stride_t;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) vp[4 * t + i] = vb + (16 * t + 4 * g + i) * a.v_cache_stride_t;
      ok = in ? ~0u : 0u;
    } else {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        uint32_t page, off;
        if constexpr (MODE == kPageFour) {
          const bool in = locate(p0 + 16 * t + 4 * g, page, off);
          const T* v0 = vc + (int64_t)page * a.v_cache_stride_p + (int64_t)off * a.v_cache_stride_t;
#pragma unroll
          for (int i = 0; i < 4; ++i) vp[4 * t + i] = v0 + i * a.v_cache_stride_t;
          ok |= (in ? 15u : 0u) << (4 * t);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool in = locate(p0 + 16 * t + 4 * g + i, page, off);
            vp[4 * t + i] = vc + (int64_t)page * a.v_cache_stride_p + (int64_t)off * a.v_cache_stride_t;
            ok |= (in ? 1u : 0u) << (4 * t + i);
          }
        }
      }
    }
    bool whole = p0 >= first && p0 + kStep <= end;
    if (!whole) {
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        const int pos = p0 + 16 * (e / 4) + 4 * g + e % 4;
        if (pos < first || pos >= end) ok &= ~(1u << e);
      }
    }
    constexpr uint32_t kAll = kMine == 8 ? 255u : 15u;
    whole = __all((ok & kAll) == kAll);

    uint32_t vw[kMine][kVW];
    auto load_values = [&]() {
#pragma unroll
      for (int e = 0; e < kMine; ++e)
#pragma unroll
        for (int k = 0; k < Pc::kCount; ++k) {
          constexpr int kPer = St::kPer;
          const int d = 16 * Pc::before(k) + n * Pc::width(k);
          const T* v = vp[e] + (d < Dh ? d : 0);
          if (Pc::width(k) / kPer == 4) load_words<4>(v, &vw[e][Pc::before(k) / kPer]);
          else if (Pc::width(k) / kPer == 2) load_words<2>(v, &vw[e][Pc::before(k) / kPer]);
          else load_words<1>(v, &vw[e][Pc::before(k) / kPer]);
        }
    };
    // Requested with the keys, except where the registers of both would leave one wave per SIMD (heads
    // of 256, 64 rows of 512 to 4096 positions: 119 us so, 92 with the values requested after the scores).
    constexpr bool kLate = DH == 256 || (sizeof(T) == 4 && DH > 128);
    if constexpr (!kLate) load_values();

    // Scores.
    float x[kMine];
    const bool tail = Dh % (4 * kE) != 0 || Dh < DH;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      f32x4 s = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (tail && (4 * c + g) * kE >= Dh) {
#pragma unroll
          for (int i = 0; i < 4; ++i) kw[t][c][i] = 0;
        }
        s = product32<T>(kw[t][c], q[c], s);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * t + i] = s[i] * to2;
    }
    if constexpr (kLate) {
      __builtin_amdgcn_sched_barrier(0);
      load_values();
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        const bool in = ok >> e & 1;
        x[e] = in ? x[e] : -INFINITY;
#pragma unroll
        for (int i = 0; i < kVW; ++i) vw[e][i] = in ? vw[e][i] : 0;
      }
    }

    // Weights.
    float top = x[0];
#pragma unroll
    for (int e = 1; e < kMine; ++e) top = fmaxf(top, x[e]);
    if (__any(top > m + (8.0f + kHead))) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top - kHead), f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int j = 0; j < Pc::kElems; ++j) o[j] *= f;
    }
    // A step's weights are summed before they meet the others': one by one, small ones beside a large sum
    // would all be rounded away.
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
      x[e] = __builtin_amdgcn_exp2f(x[e] - m);
      sum += x[e];
    }
    l += sum;

    // Values.
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < Pc::kElems; ++j)
#pragma unroll
        for (int e = 0; e < kMine; ++e)
          o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vw[e][j]), x[e], o[j], 0, 0, 0);
    } else {
      constexpr int kPieces = __is_same(T, __bf16) ? 3 : 2;
      uint32_t w[kPieces][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t piece[kPieces];
        pieces_of<T>(x[2 * i], x[2 * i + 1], piece);
#pragma unroll
        for (int c = 0; c < kPieces; ++c) w[c][i] = piece[c];
      }
#pragma unroll
      for (int j = 0; j < Pc::kElems; ++j) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)  // the 16-bit half j % 2 of two positions
          v[i] = __builtin_amdgcn_perm(vw[2 * i + 1][j / 2], vw[2 * i][j / 2],
                                       j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int c = kPieces - 1; c >= 0; --c) o[j] = product32<T>(v, w[c], o[j]);
      }
    }
  }

  // Join the waves. Query head n's m is the same in all g; its sum is over them.
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  __shared__ float s_m[kAttnWaves][16], s_l[kAttnWaves][16];
  __shared__ alignas(16) float s_o[kAttnWaves][16][DH + 4];
  if (g == 0) {
    s_m[wave][n] = m;
    s_l[wave][n] = l;
  }
#pragma unroll
  for (int k = 0; k < Pc::kCount; ++k) {
    constexpr int kMost = Pc::kWide;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kMost; ++j)
        if (j < Pc::width(k))
          s_o[wave][n][16 * Pc::before(k) + (4 * g + i) * Pc::width(k) + j] = o[Pc::before(k) + j][i];
  }
  __syncthreads();
  // 16 to 64 lanes a head, which needs the waves' factors once, and 4 elements at a time (an element at a
  // time, factors and all, 16 heads of 256 took 4 us).
  const int lanes = heads > 8 ? 16 : heads > 4 ? 32 : 64;
  const int h = threadIdx.x / lanes;
  if (h >= heads) return;
  float top = s_m[0][h], f[kAttnWaves], total = 0.0f;
#pragma unroll
  for (int v = 1; v < kAttnWaves; ++v) top = fmaxf(top, s_m[v][h]);
#pragma unroll
  for (int v = 0; v < kAttnWaves; ++v) {
    f[v] = __builtin_amdgcn_exp2f(s_m[v][h] - top);
    total = fmaf(s_l[v][h], f[v], total);
  }
  const int64_t at = row * a.q_heads + head0 + h;
  T* out = static_cast<T*>(a.out) + at * Dh;
  float* part = p.part + (at * p.splits + split) * Dh;
  const float by = 1.0f / total;
  bool odd = false;  // one of my elements is no number (or infinite beside another of the other sign)
  for (int d = threadIdx.x % lanes * 4; d < Dh; d += lanes * 4) {
    float sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < kAttnWaves; ++v) {
      const f32x4 o4 = *reinterpret_cast<const f32x4*>(&s_o[v][h][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = fmaf(o4[i], f[v], sum[i]);
    }
    const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    odd = odd || all != all;
    if (only) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = total == 0.0f ? 0.0f : sum[i] * by;
      VecIO<T, 4>::st(out + d, VecIO<T, 4>::pack(sum));
    } else {
      VecIO<float, 4>::st(part + d, VecIO<float, 4>::pack(sum));
    }
  }
  if (threadIdx.x % lanes == 0) {
    if (only) {
      if (a.lse) a.lse[at] = (top + __log2f(total)) * 0.69314718055994530942f;
    } else {
      p.part_ml[(at * p.splits + split) * 2] = top;
      p.part_ml[(at * p.splits + split) * 2 + 1] = total;
    }
  }
  if (sizeof(T) == 2 && odd && total == total) {
#pragma unroll 1
    for (int j = 0, d = threadIdx.x % lanes * 4; d < Dh; d += ++j % 4 ? 1 : lanes * 4 - 3) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < kAttnWaves; ++v) sum = fmaf(s_o[v][h][d], f[v], sum);
      if (sum == sum) continue;
      const float value = infinite<T>(row, split, (int)head0 + h, d, top);
      if (value == 0.0f) continue;
      if (only) out[d] = static_cast<T>(value);
      else part[d] = value;
    }
  }
}

hipError_t paged_attn_bf16(const AttnParams& p, int mode, hipStream_t s);
hipError_t paged_attn_f16(const AttnParams& p, int mode, hipStream_t s);
hipError_t paged_attn_f32(const AttnParams& p, int mode, hipStream_t s);

template <typename T, int DH>
hipError_t paged_attn_mode(const AttnParams& p, int mode, hipStream_t s) {
  const int64_t grid = p.a.rows * p.splits * p.a.kv_heads * p.tiles;
  constexpr int kBlock = kAttnWaves * kWave;
  switch (mode) {
    case kPageStep: return start(&paged_attn_kernel<T, DH, kPageStep>, grid, kBlock, s, p);
    case kPageFour: return start(&paged_attn_kernel<T, DH, kPageFour>, grid, kBlock, s, p);
    default: return start(&paged_attn_kernel<T, DH, kPageAny>, grid, kBlock, s, p);
  }
}

// The kernels' row sizes: a head_dim takes the next one.
template <typename T>
hipError_t paged_attn_type(const AttnParams& p, int mode, hipStream_t s) {
  const int64_t d = p.a.head_dim;
  if (d <= 64) return paged_attn_mode<T, 64>(p, mode, s);
  if (d <= 96) return paged_attn_mode<T, 96>(p, mode, s);
  if (d <= 128) return paged_attn_mode<T, 128>(p, mode, s);
  if (d <= 192) return paged_attn_mode<T, 192>(p, mode, s);
  return paged_attn_mode<T, 256>(p, mode, s);
}

}  // namespace ops
}  // namespace ccv1d

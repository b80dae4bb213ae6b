// C ABI of include/ccv1d_ops.h: argument checks before anything is launched, then the launchers.
#include <cstdarg>
#include <cstdio>

#include "ops_common.h"

using namespace ccv1d;

namespace {

constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1;  // of a launch

int fail(int code, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return report_error(code, buf);
}

int invalid(const char* what) { return report_error(CCV1D_ERR_INVALID, what); }

bool dtype_ok(int dt) { return dt == CCV1D_F32 || dt == CCV1D_F16 || dt == CCV1D_BF16; }

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// a * b within [0, limit], for non-negative factors.
bool product_within(int64_t a, int64_t b, int64_t limit) { return a == 0 || b <= limit / a; }

// Makes `device` current for the launch and restores the caller's.
struct Device {
  int prev = -1, want;
  hipError_t err;
  explicit Device(int device) : want(device) {
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != want) err = hipSetDevice(want);
  }
  ~Device() {
    if (prev >= 0 && prev != want) (void)hipSetDevice(prev);
  }
};

template <typename A>
int launch(const A& a, hipError_t (*fn)(const A&, hipStream_t)) {
  Device d(a.device);
  hipError_t e = d.err;
  if (e == hipSuccess) e = fn(a, static_cast<hipStream_t>(a.stream));
  if (e != hipSuccess) return fail(CCV1D_ERR_HIP, "%s", hipGetErrorString(e));
  return CCV1D_OK;
}

int check_rec(const ccv1d_rec_args* a, bool backward) {
  if (!a) return invalid("args is null");
  if (a->batch < 0 || a->seqlen < 0 || a->dim < 0) return invalid("negative size");
  if (!dtype_ok(a->dtype)) return invalid("dtype must be fp32, fp16 or bf16");
  if (!(a->decay_scale >= 0.0f)) return invalid("decay_scale must not be negative");
  // Rows, row offsets and workgroup numbers are 32-bit, the product of all three 64-bit.
  if (a->seqlen > kMaxGrid || a->dim > kMaxGrid ||
      !product_within(a->batch, cdiv(a->dim, 64), kMaxGrid) ||
      !product_within(a->batch * cdiv(a->dim, 64), cdiv(a->seqlen, CCV1D_REC_SAVED_ROWS), kMaxGrid))
    return fail(CCV1D_ERR_UNSUPPORTED, "batch, seqlen and dim too large for one launch");
  if (ops::rec_threads(*a, backward) > kMaxThreads)
    return fail(CCV1D_ERR_UNSUPPORTED, "batch, seqlen and dim too large for one launch");
  if (a->batch == 0 || a->dim == 0) return CCV1D_OK;
  if (a->seqlen > 0) {
    if (!a->x || !a->gate) return invalid("x or gate is null");
    if (backward) {
      if (!a->dout || !a->dx || !a->dgate) return invalid("dout, dx or dgate is null");
      if ((a->input_gate != nullptr) != (a->dinput_gate != nullptr))
        return invalid("dinput_gate goes with input_gate");
      if (!a->saved) return invalid("saved is null");
    } else if (!a->out) {
      return invalid("out is null");
    }
  }
  if (backward && (a->decay != nullptr) != (a->ddecay != nullptr))
    return invalid("ddecay goes with decay");
  const size_t need = ccv1d_rec_workspace_bytes(a->batch, a->seqlen, a->dim, backward);
  if (need && (!a->workspace || a->workspace_bytes < need))
    return fail(CCV1D_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  return CCV1D_OK;
}

int check_attn(const ccv1d_paged_attn_args* a) {
  if (!a) return invalid("args is null");
  if (a->rows < 0 || a->requests < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->num_pages < 0 ||
      a->max_pages < 0 || a->window < 0 || a->max_seq_len < 0)
    return invalid("negative size");
  if (!dtype_ok(a->dtype)) return invalid("dtype must be fp32, fp16 or bf16");
  if (a->page_size < 1) return invalid("page_size must be at least 1");
  if (a->head_dim < 8 || a->head_dim > CCV1D_PAGED_MAX_HEAD_DIM || a->head_dim % 8)
    return fail(CCV1D_ERR_INVALID, "head_dim must be a multiple of 8, at most %d",
                CCV1D_PAGED_MAX_HEAD_DIM);
  if (a->kv_heads == 0 ? a->q_heads != 0 : a->q_heads % a->kv_heads != 0)
    return invalid("q_heads must be a multiple of kv_heads");
  if (a->page_size > (int64_t(1) << 30) || !product_within(a->max_pages, a->page_size, int64_t(1) << 30))
    return fail(CCV1D_ERR_UNSUPPORTED, "max_pages * page_size must be at most 2^30");
  // The spans are planned for fewer than 2^32 threads where this holds.
  if (!product_within(a->rows, a->q_heads, kMaxGrid / 256))
    return fail(CCV1D_ERR_UNSUPPORTED, "rows * q_heads too large for one launch");
  return CCV1D_OK;
}

}  // namespace

extern "C" {

size_t ccv1d_rec_workspace_bytes(int64_t batch, int64_t seqlen, int64_t dim, int backward) {
  if (batch <= 0 || seqlen <= 0 || dim <= 0) return 0;
  return ops::rec_workspace(batch, seqlen, dim, backward != 0);
}

int ccv1d_rec_fwd(const struct ccv1d_rec_args* args) {
  clear_error();
  if (int rc = check_rec(args, false)) return rc;
  if (args->batch == 0 || args->dim == 0) return CCV1D_OK;
  return launch(*args, ops::rec_fwd);
}

int ccv1d_rec_bwd(const struct ccv1d_rec_args* args) {
  clear_error();
  if (int rc = check_rec(args, true)) return rc;
  if (args->dim == 0 || (args->batch == 0 && !args->ddecay)) return CCV1D_OK;
  return launch(*args, ops::rec_bwd);
}

int ccv1d_rec_update(const struct ccv1d_rec_update_args* args) {
  clear_error();
  if (!args) return invalid("args is null");
  const ccv1d_rec_update_args& a = *args;
  if (a.rows < 0 || a.slots < 0 || a.dim < 0) return invalid("negative size");
  if (!dtype_ok(a.dtype)) return invalid("dtype must be fp32, fp16 or bf16");
  if (!(a.decay_scale >= 0.0f)) return invalid("decay_scale must not be negative");
  if (!a.state_indices && a.rows > a.slots) return invalid("more rows than slots");
  if (!product_within(a.rows, cdiv(a.dim, 64), kMaxGrid) || ops::rec_update_threads(a) > kMaxThreads)
    return fail(CCV1D_ERR_UNSUPPORTED, "rows and dim too large for one launch");
  if (a.rows == 0 || a.dim == 0) return CCV1D_OK;
  if (!a.x || !a.gate || !a.out || (a.slots && !a.state))
    return invalid("x, gate, state or out is null");
  return launch(a, ops::rec_update);
}

int ccv1d_paged_plan(const struct ccv1d_paged_plan_args* args) {
  clear_error();
  if (!args) return invalid("args is null");
  const ccv1d_paged_plan_args& a = *args;
  if (a.requests < 0 || a.max_pages < 0 || a.num_free_pages < 0 || a.max_tokens < 0)
    return invalid("negative size");
  if (a.page_size < 1) return invalid("page_size must be at least 1");
  if (a.requests >= kMaxGrid || a.max_tokens > kMaxGrid || a.num_free_pages > kMaxGrid ||
      a.page_size > (int64_t(1) << 30) || !product_within(a.max_pages, a.page_size, kMaxGrid))
    return fail(CCV1D_ERR_UNSUPPORTED,
                "requests, max_tokens, page_size and max_pages * page_size too large");
  if (!a.num_free || !a.num_free_out || !a.query_start) return invalid("num_free or query_start is null");
  if (a.requests &&
      (!a.cached_lens || !a.new_lens || !a.seq_lens || (a.max_pages && !a.block_tables)))
    return invalid("cached_lens, new_lens, seq_lens or block_tables is null");
  if (a.num_free_pages && !a.free_pages) return invalid("free_pages is null");
  if (a.max_tokens && (!a.positions || !a.request_ids || !a.slot_mapping))
    return invalid("positions, request_ids or slot_mapping is null");
  return launch(a, ops::paged_plan);
}

int ccv1d_paged_write(const struct ccv1d_paged_write_args* args) {
  clear_error();
  if (!args) return invalid("args is null");
  const ccv1d_paged_write_args& a = *args;
  if (a.tokens < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.num_pages < 0)
    return invalid("negative size");
  if (!dtype_ok(a.dtype)) return invalid("dtype must be fp32, fp16 or bf16");
  if (a.page_size < 1) return invalid("page_size must be at least 1");
  if (a.tokens > kMaxGrid || !product_within(a.kv_heads, a.head_dim, kMaxGrid / 8))
    return fail(CCV1D_ERR_UNSUPPORTED, "tokens or kv_heads * head_dim too large for one launch");
  if (!product_within(a.num_pages, a.page_size, INT64_MAX)) return invalid("cache too large");
  if (a.tokens == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.num_pages == 0) return CCV1D_OK;
  if (ops::paged_write_threads(a) > kMaxThreads)
    return fail(CCV1D_ERR_UNSUPPORTED, "tokens too large for one launch");
  if (!a.k || !a.v || !a.k_cache || !a.v_cache || !a.slot_mapping)
    return invalid("k, v, a cache or slot_mapping is null");
  return launch(a, ops::paged_write);
}

size_t ccv1d_paged_attn_workspace_bytes(const struct ccv1d_paged_attn_args* args) {
  if (check_attn(args) || args->rows == 0 || args->q_heads == 0) return 0;
  return ops::paged_attn_workspace(*args);
}

int ccv1d_paged_attn(const struct ccv1d_paged_attn_args* args) {
  clear_error();
  if (int rc = check_attn(args)) return rc;
  const ccv1d_paged_attn_args& a = *args;
  if (a.rows == 0 || a.q_heads == 0) return CCV1D_OK;
  if (!a.q || !a.out || !a.seq_lens) return invalid("q, out or seq_lens is null");
  if (a.num_pages && (!a.k_cache || !a.v_cache)) return invalid("a cache is null");
  if (a.requests && a.max_pages && !a.block_tables) return invalid("block_tables is null");
  if (!a.request_ids && a.rows > a.requests) return invalid("more rows than requests");
  const size_t need = ops::paged_attn_workspace(a);
  if (need && (!a.workspace || a.workspace_bytes < need))
    return fail(CCV1D_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  return launch(a, ops::paged_attn);
}

}  // extern "C"

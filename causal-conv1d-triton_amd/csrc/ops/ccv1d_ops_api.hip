// C ABI of include/ccv1d_ops.h and include/ccv1d_layer.h: argument checks before anything is launched, then the launchers.
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

int check_delta(const ccv1d_delta_args* a) {
  if (!a) return invalid("args is null");
  if (a->batch < 0 || a->seqlen < 0) return invalid("negative size");
  if (!dtype_ok(a->dtype) || !dtype_ok(a->log_decay_dtype) || !dtype_ok(a->beta_dtype))
    return invalid("dtypes must be fp32, fp16 or bf16");
  if (a->key_heads < 1 || a->heads < 1 || a->heads % a->key_heads)
    return invalid("heads must be a multiple of key_heads");
  if (a->key_dim < 1 || a->key_dim > CCV1D_DELTA_MAX_KEY_DIM)
    return fail(CCV1D_ERR_INVALID, "key_dim must be 1 to %d", CCV1D_DELTA_MAX_KEY_DIM);
  if (a->value_dim < 1) return invalid("value_dim must be at least 1");
  if (!ops::delta_fits(*a)) return fail(CCV1D_ERR_UNSUPPORTED, "batch, seqlen, heads and dims too large for one launch");
  return CCV1D_OK;
}

int check_delta_call(const ccv1d_delta_args* a, bool backward) {
  if (int rc = check_delta(a)) return rc;
  if (a->batch == 0 || a->seqlen == 0) return CCV1D_OK;
  if (!a->q || !a->k || !a->v || !a->log_decay || !a->beta) return invalid("q, k, v, log_decay or beta is null");
  if (backward) {
    if (!a->dout || !a->dq || !a->dk || !a->dv || !a->dlog_decay || !a->dbeta)
      return invalid("dout, dq, dk, dv, dlog_decay or dbeta is null");
    if (!a->saved) return invalid("saved is null");
  } else if (!a->out) {
    return invalid("out is null");
  }
  const size_t need = ops::delta_workspace(*a, backward);
  if (!a->workspace || a->workspace_bytes < need)
    return fail(CCV1D_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  return CCV1D_OK;
}

int check_norm(const ccv1d_norm_args* a) {
  if (!a) return invalid("args is null");
  if (a->outer < 0 || a->inner < 0) return invalid("negative size");
  if (a->dim < 1 || a->dim > CCV1D_NORM_MAX_DIM)
    return fail(CCV1D_ERR_INVALID, "dim must be 1 to %d", CCV1D_NORM_MAX_DIM);
  if (!dtype_ok(a->dtype)) return invalid("dtype must be fp32, fp16 or bf16");
  if (a->residual_dtype != a->dtype && a->residual_dtype != CCV1D_F32)
    return invalid("residual_dtype must be dtype or fp32");
  if (a->residual_dtype != a->dtype && !a->residual && a->outer > 0 && a->inner > 0)  // of no rows a residual is null, too
    return invalid("residual_dtype is dtype without residual");
  if (!a->post_weight && !a->pre_weight) return invalid("post_weight and pre_weight are null");
  if ((a->post_weight && !dtype_ok(a->post_dtype)) || (a->scale_weight && !dtype_ok(a->scale_dtype)) ||
      (a->pre_weight && !dtype_ok(a->pre_dtype)))
    return invalid("the weights' dtypes must be fp32, fp16 or bf16");
  if (!(a->eps >= 0.0f)) return invalid("eps must not be negative");
  if (a->activation < CCV1D_NORM_IDENTITY || a->activation > CCV1D_NORM_SIGMOID) return invalid("unknown activation");
  if (!product_within(a->outer, a->inner, kMaxGrid) || ops::norm_threads(*a) > kMaxThreads)
    return fail(CCV1D_ERR_UNSUPPORTED, "too many rows for one launch");
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

size_t ccv1d_delta_saved_floats(const struct ccv1d_delta_args* args) {
  if (check_delta(args) || args->batch == 0 || args->seqlen == 0) return 0;
  return ops::delta_saved(*args);
}

size_t ccv1d_delta_workspace_bytes(const struct ccv1d_delta_args* args, int backward) {
  if (check_delta(args) || args->batch == 0 || args->seqlen == 0) return 0;
  return ops::delta_workspace(*args, backward != 0);
}

int ccv1d_delta_fwd(const struct ccv1d_delta_args* args) {
  clear_error();
  if (int rc = check_delta_call(args, false)) return rc;
  if (args->batch == 0) return CCV1D_OK;
  return launch(*args, ops::delta_fwd);
}

int ccv1d_delta_bwd(const struct ccv1d_delta_args* args) {
  clear_error();
  if (int rc = check_delta_call(args, true)) return rc;
  if (args->batch == 0) return CCV1D_OK;
  return launch(*args, ops::delta_bwd);
}

int ccv1d_delta_update(const struct ccv1d_delta_update_args* args) {
  clear_error();
  if (!args) return invalid("args is null");
  const ccv1d_delta_update_args& a = *args;
  if (a.rows < 0 || a.slots < 0) return invalid("negative size");
  if (!dtype_ok(a.dtype) || !dtype_ok(a.log_decay_dtype) || !dtype_ok(a.beta_dtype))
    return invalid("dtypes must be fp32, fp16 or bf16");
  if (a.key_heads < 1 || a.heads < 1 || a.heads % a.key_heads) return invalid("heads must be a multiple of key_heads");
  if (a.key_dim < 1 || a.key_dim > CCV1D_DELTA_MAX_KEY_DIM)
    return fail(CCV1D_ERR_INVALID, "key_dim must be 1 to %d", CCV1D_DELTA_MAX_KEY_DIM);
  if (a.value_dim < 1) return invalid("value_dim must be at least 1");
  if (!a.state_indices && a.rows > a.slots) return invalid("more rows than slots");
  if (!product_within(a.rows, a.heads, kMaxGrid) || !product_within(a.rows * a.heads, cdiv(a.value_dim, 64), kMaxGrid) ||
      ops::delta_update_threads(a) > kMaxThreads)
    return fail(CCV1D_ERR_UNSUPPORTED, "rows, heads and value_dim too large for one launch");
  if (a.rows == 0) return CCV1D_OK;
  if (!a.q || !a.k || !a.v || !a.log_decay || !a.beta || !a.out || (a.slots && !a.state))
    return invalid("q, k, v, log_decay, beta, state or out is null");
  return launch(a, ops::delta_update);
}

size_t ccv1d_norm_workspace_bytes(const struct ccv1d_norm_args* args) {
  if (check_norm(args)) return 0;
  return ops::norm_workspace(*args);
}

int ccv1d_norm_fwd(const struct ccv1d_norm_args* args) {
  clear_error();
  if (int rc = check_norm(args)) return rc;
  const ccv1d_norm_args& a = *args;
  if (a.outer * a.inner == 0) return CCV1D_OK;
  if (!a.x) return invalid("x is null");
  if ((a.pre_weight != nullptr) != (a.y != nullptr)) return invalid("y goes with pre_weight");
  if (!a.pre_weight && !a.r) return invalid("r is null");
  return launch(a, ops::norm_fwd);
}

int ccv1d_norm_bwd(const struct ccv1d_norm_args* args) {
  clear_error();
  if (int rc = check_norm(args)) return rc;
  const ccv1d_norm_args& a = *args;
  if ((a.post_weight != nullptr) != (a.dpost_weight != nullptr) ||
      (a.scale_weight != nullptr) != (a.dscale_weight != nullptr) ||
      (a.pre_weight != nullptr) != (a.dpre_weight != nullptr))
    return invalid("the weights' gradients go with the weights");
  if (a.dy && !a.pre_weight) return invalid("dy goes with pre_weight");
  if (a.outer * a.inner > 0) {
    if (!a.x || !a.dx) return invalid("x or dx is null");
    if ((a.gate != nullptr) != (a.dgate != nullptr)) return invalid("dgate goes with gate");
    if (a.dresidual && !a.residual) return invalid("dresidual goes with residual");
    const size_t need = ops::norm_workspace(a);
    if (!a.workspace || a.workspace_bytes < need)
      return fail(CCV1D_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  }
  return launch(a, ops::norm_bwd);
}

}  // extern "C"

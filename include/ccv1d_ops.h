/*
 * ccv1d_ops.h - C ABI of the operators around the convolution (libccv1d.so): the gated linear
 * recurrence of a recurrent block, and the paged key-value caches of the attention layers beside it.
 *
 * Conventions are those of ccv1d.h: device pointers on `device`, every buffer the caller's, work
 * enqueued on `stream` and nothing synchronised, the calling thread's device restored, a status from
 * enum ccv1d_status and a thread-local message (ccv1d_last_error). Arguments travel in one struct per
 * entry point, which the library reads during the call only. Element types are enum ccv1d_dtype
 * (F32, F16, BF16), and pointers are aligned to an element; workspaces to 8 bytes, their contents on
 * entry do not matter, and calls that may overlap in time need one each. Calls can be captured in a graph:
 * no memset nodes, no allocation.
 */
#ifndef CCV1D_OPS_H
#define CCV1D_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "ccv1d.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------------------------
 * Gated linear recurrence, over channels-last (batch, seqlen, dim):
 *
 *   r = sigmoid(gate), i = sigmoid(input_gate) (1 without one)
 *   with decay:     a = exp(-decay_scale * softplus(decay[d]) * r),  beta = sqrt(1 - a^2)
 *   without decay:  a = r,                                           beta = 1 - r
 *   h[t] = a[t] * h[t-1] + beta[t] * i[t] * x[t],   h[-1] = initial_states (zero without)
 *
 * computed in fp32 whatever the element type. A sequence's first row has the beta of any other (some models
 * of this family take 1 there). With seq_idx the state starts at zero in each row whose
 * id differs from the row before it; initial_states belong to the sequence of seq_idx[:, 0]; rows of a
 * negative id are padding: their h is zero, whatever x and the gates hold there, and no gradient
 * leaves them.
 * ------------------------------------------------------------------------------------------- */

/* Rows per saved state: the forward hands the backward the state in front of every 64th row. */
#define CCV1D_REC_SAVED_ROWS 64

struct ccv1d_rec_args {
  /* inputs (batch, seqlen, dim) of type dtype, unit channel stride, batch and time strides in elements */
  const void* x;
  int64_t x_stride_b, x_stride_t;
  const void* gate;
  int64_t gate_stride_b, gate_stride_t;
  const void* input_gate; /* may be NULL */
  int64_t input_gate_stride_b, input_gate_stride_t;
  int dtype;
  const float* decay; /* (dim,) or NULL */
  float decay_scale; /* not negative */
  int seq_idx_64;              /* 0: seq_idx holds int32_t, else int64_t */
  const void* seq_idx;         /* (batch, seqlen) contiguous, or NULL */
  const float* initial_states; /* (batch, dim) or NULL */
  int64_t batch, seqlen, dim;
  /* forward */
  void* out;           /* (batch, seqlen, dim) contiguous, type dtype: h rounded once */
  float* final_states; /* (batch, dim): h of the last row; or NULL */
  float* saved;        /* (batch, ceil(seqlen / CCV1D_REC_SAVED_ROWS), dim): forward: written when not
                          NULL; backward: what the forward wrote */
  /* backward */
  const void* dout; /* (batch, seqlen, dim), type dtype, unit channel stride */
  int64_t dout_stride_b, dout_stride_t;
  const float* dfinal_states; /* (batch, dim) or NULL */
  void* dx;                   /* contiguous, type dtype, as dgate and dinput_gate */
  void* dgate;
  void* dinput_gate;      /* required iff input_gate */
  float* ddecay;          /* (dim,), required iff decay */
  float* dinitial_states; /* (batch, dim) or NULL */
  void* workspace;
  size_t workspace_bytes;
  int device;
  void* stream;
};

/* Bytes of workspace of the forward (backward = 0) or the backward (1): a function of the shape. */
size_t ccv1d_rec_workspace_bytes(int64_t batch, int64_t seqlen, int64_t dim, int backward);
int ccv1d_rec_fwd(const struct ccv1d_rec_args* args);
/* ddecay is deterministic: its order of summation depends on the shape alone. */
int ccv1d_rec_bwd(const struct ccv1d_rec_args* args);

/* One token of each request: h = a * state + beta * i * x, the states in a pool of slots, in place.
 * A row whose index is outside [0, slots) is left out: its out is zero. Two rows of one slot race: what they
 * leave there and return is not defined. */
struct ccv1d_rec_update_args {
  const void* x; /* (rows, dim) of type dtype, unit channel stride; so gate and input_gate */
  int64_t x_stride;
  const void* gate;
  int64_t gate_stride;
  const void* input_gate; /* may be NULL */
  int64_t input_gate_stride;
  int dtype;
  const float* decay; /* (dim,) or NULL */
  float decay_scale; /* not negative */
  float* state; /* (slots, dim), unit channel stride */
  int64_t state_stride;
  const int32_t* state_indices; /* (rows,) or NULL: row r uses slot r */
  void* out;                    /* (rows, dim) contiguous, type dtype */
  int64_t rows, slots, dim;
  int device;
  void* stream;
};
int ccv1d_rec_update(const struct ccv1d_rec_update_args* args);

/* ---------------------------------------------------------------------------------------------
 * Paged caches. A cache is (num_pages, page_size, kv_heads, head_dim) with any strides but a unit
 * last one; token p of a request lies in page block_tables[request, p / page_size] at p % page_size.
 * ------------------------------------------------------------------------------------------- */

/* Plans a batch on the GPU. Request r has cached_lens[r] tokens in its pages and brings new_lens[r]
 * (negative lengths count as zero). A request is admitted when its pages fit its row of the block
 * table and it needs no new page or the pages that it and the requests before it need (those that fit
 * their rows) are free; an admitted request's new pages come from the end of the free list, in order
 * of request and position, and are noted in block_tables. The tokens of all requests lie one after the
 * other in max_tokens places; places past the last token, and those of requests that were not admitted,
 * get -1. No output shares memory with an input, block_tables apart, which is both. */
struct ccv1d_paged_plan_args {
  const int32_t* cached_lens; /* (requests,) */
  const int32_t* new_lens;    /* (requests,) */
  int32_t* block_tables;      /* (requests, max_pages), rows block_table_stride apart */
  int64_t block_table_stride;
  const int32_t* free_pages; /* (num_free_pages,): the first num_free are free */
  const int32_t* num_free;   /* (1,); more than num_free_pages counts as num_free_pages */
  int64_t requests, max_pages, num_free_pages, page_size, max_tokens;
  int32_t* seq_lens;     /* (requests,): cached + new of the admitted, cached of the others */
  int32_t* query_start;  /* (requests + 1,): places of the requests' first tokens, and their total */
  int32_t* positions;    /* (max_tokens,): a token's place in its sequence */
  int32_t* request_ids;  /* (max_tokens,) */
  int64_t* slot_mapping; /* (max_tokens,): page * page_size + offset; -1 also where a page is negative */
  int32_t* num_free_out; /* (1,): free pages left */
  int device;
  void* stream;
};
int ccv1d_paged_plan(const struct ccv1d_paged_plan_args* args);

/* Writes keys and values (tokens, kv_heads, head_dim) to their slots; slots outside the cache are left
 * out. The caches' rows do not overlap; two tokens of one slot leave one of them there, or pieces of both. */
struct ccv1d_paged_write_args {
  const void* k; /* unit last stride */
  int64_t k_stride_t, k_stride_h;
  const void* v;
  int64_t v_stride_t, v_stride_h;
  int dtype;
  void* k_cache;
  int64_t k_cache_stride_p, k_cache_stride_t, k_cache_stride_h;
  void* v_cache;
  int64_t v_cache_stride_p, v_cache_stride_t, v_cache_stride_h;
  const int64_t* slot_mapping; /* (tokens,) */
  int64_t tokens, kv_heads, head_dim, num_pages, page_size;
  int device;
  void* stream;
};
int ccv1d_paged_write(const struct ccv1d_paged_write_args* args);

/* Attention of one token per row over a paged cache. Row r attends to positions
 * [max(0, L - window), L), L = seq_lens[r], of request request_ids[r] (r without request_ids):
 *   out[r, h] = sum_p softmax_p(scale * q[r, h] . k[p, h / group]) v[p, h / group],  group = q_heads / kv_heads
 * A row with no position (L <= 0, a request outside the table) gets zeros and a log-sum-exp of -inf.
 * Positions past max_pages * page_size or max_seq_len, or in pages outside the cache, are left out; L is not
 * cut by them. */
struct ccv1d_paged_attn_args {
  const void* q; /* (rows, q_heads, head_dim), unit last stride */
  int64_t q_stride_r, q_stride_h;
  int dtype; /* of q, the caches and out */
  const void* k_cache;
  int64_t k_cache_stride_p, k_cache_stride_t, k_cache_stride_h;
  const void* v_cache;
  int64_t v_cache_stride_p, v_cache_stride_t, v_cache_stride_h;
  const int32_t* block_tables; /* (requests, max_pages), rows block_table_stride apart */
  int64_t block_table_stride;
  const int32_t* seq_lens;    /* (rows,) */
  const int32_t* request_ids; /* (rows,) or NULL */
  void* out;                  /* (rows, q_heads, head_dim) contiguous */
  float* lse;                 /* (rows, q_heads) or NULL: natural logarithm */
  float scale;
  int64_t window; /* 0: none */
  int64_t rows, requests, q_heads, kv_heads, head_dim, num_pages, page_size, max_pages;
  int64_t max_seq_len; /* no position at or past it (0: max_pages * page_size): sizes the launch */
  void* workspace;
  size_t workspace_bytes;
  int device;
  void* stream;
};
/* Largest head_dim, a multiple of 8. */
#define CCV1D_PAGED_MAX_HEAD_DIM 256
/* Bytes of workspace of the call (its pointers are not read). */
size_t ccv1d_paged_attn_workspace_bytes(const struct ccv1d_paged_attn_args* args);
int ccv1d_paged_attn(const struct ccv1d_paged_attn_args* args);

#ifdef __cplusplus
}
#endif

#endif /* CCV1D_OPS_H */

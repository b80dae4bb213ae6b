/*
 * ccv1d_layer.h - C ABI of the operators of a linear-attention layer (libccv1d.so): the gated delta rule
 * that the convolution's queries, keys and values go through, and the norms around a block.
 *
 * Conventions are those of ccv1d.h and ccv1d_ops.h: device pointers on `device`, every buffer the
 * caller's, work enqueued on `stream` and nothing synchronised, the calling thread's device restored, a
 * status from enum ccv1d_status and a thread-local message (ccv1d_last_error). Arguments travel in one
 * struct per entry point, which the library reads during the call only. Element types are enum ccv1d_dtype
 * (F32, F16, BF16), and pointers are aligned to an element; workspaces to 16 bytes, their contents on entry
 * do not matter, and calls that may overlap in time need one each. Calls can be captured in a graph: no
 * memset nodes, no allocation. Inputs and outputs of a call share no memory, but where it says in place.
 */
#ifndef CCV1D_LAYER_H
#define CCV1D_LAYER_H

#include <stddef.h>
#include <stdint.h>

#include "ccv1d.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------------------------
 * Gated delta rule. A head keeps a state S (key_dim, value_dim); a token brings a query and a key
 * (key_dim), a value (value_dim), a log-decay g and a rate beta:
 *
 *   S' = exp(g) S,  u = beta (v - S'^T k),  S = S' + k u^T,  o = scale S^T q
 *
 * heads is a multiple of key_heads: head h has the queries and keys of key head h / (heads / key_heads).
 * Sums and states are fp32 whatever the element type. A log-decay below -104 (whose exponential is zero in
 * fp32) empties the state. With seq_idx the state starts at zero in each row whose id differs from the row
 * before it; initial_states belong to the sequence of seq_idx[:, 0]; rows of a negative id are padding:
 * their output is zero, the state behind them zero, whatever they hold, and no gradient leaves them. An
 * infinity or NaN in another row, or a log-decay above 88.7 (whose exponential is infinite in fp32) on a state, spoils its
 * own sequence alone: outputs from that row on (in q: that row's; in v: its column's), gradients. Only finite keys so long,
 * or log-decays of several rows so far above zero, that 64 rows' products overflow fp32 can spoil more.
 * ------------------------------------------------------------------------------------------- */

/* Rows of a chunk: the forward hands the backward the state in front of every chunk, and the corrections u
 * of all rows. */
#define CCV1D_DELTA_CHUNK 64
/* Largest key_dim. */
#define CCV1D_DELTA_MAX_KEY_DIM 256

struct ccv1d_delta_args {
  /* inputs of type dtype, unit last stride, the others in elements: q, k (batch, seqlen, key_heads, key_dim),
     v (batch, seqlen, heads, value_dim) */
  const void* q;
  int64_t q_stride_b, q_stride_t, q_stride_h;
  const void* k;
  int64_t k_stride_b, k_stride_t, k_stride_h;
  const void* v;
  int64_t v_stride_b, v_stride_t, v_stride_h;
  int dtype;
  const void* log_decay; /* (batch, seqlen, heads), any strides */
  int64_t log_decay_stride_b, log_decay_stride_t, log_decay_stride_h;
  int log_decay_dtype;
  int beta_dtype;
  const void* beta; /* (batch, seqlen, heads), any strides */
  int64_t beta_stride_b, beta_stride_t, beta_stride_h;
  float scale;
  int seq_idx_64;              /* 0: seq_idx holds int32_t, else int64_t */
  const void* seq_idx;         /* (batch, seqlen) contiguous, or NULL */
  const float* initial_states; /* (batch, heads, key_dim, value_dim) or NULL */
  int64_t batch, seqlen, key_heads, heads, key_dim, value_dim;
  /* forward */
  void* out;           /* (batch, seqlen, heads, value_dim) contiguous, type dtype */
  float* final_states; /* (batch, heads, key_dim, value_dim): the state behind the last row; or NULL */
  float* saved;        /* ccv1d_delta_saved_floats() floats, aligned to 16 bytes: forward: written when not NULL;
                          backward: what the forward wrote */
  /* backward */
  const void* dout; /* (batch, seqlen, heads, value_dim), type dtype, unit last stride */
  int64_t dout_stride_b, dout_stride_t, dout_stride_h;
  const float* dfinal_states; /* (batch, heads, key_dim, value_dim) or NULL */
  void* dq;                   /* contiguous, of type dtype, as dk and dv */
  void* dk;
  void* dv;
  void* dlog_decay; /* contiguous, of type log_decay_dtype */
  void* dbeta;      /* contiguous, of type beta_dtype */
  float* dinitial_states; /* (batch, heads, key_dim, value_dim) or NULL */
  void* workspace;
  size_t workspace_bytes;
  int device;
  void* stream;
};

/* Floats that a forward keeps for its backward; of the sizes alone. */
size_t ccv1d_delta_saved_floats(const struct ccv1d_delta_args* args);
/* Bytes of workspace of the forward (backward = 0) or the backward (1), of the sizes and dtype alone. */
size_t ccv1d_delta_workspace_bytes(const struct ccv1d_delta_args* args, int backward);
int ccv1d_delta_fwd(const struct ccv1d_delta_args* args);
/* Every gradient is deterministic. */
int ccv1d_delta_bwd(const struct ccv1d_delta_args* args);

/* One token of each request, the states in a pool of slots, in place. A row whose index is outside
 * [0, slots) is left out: its out is zero. Two rows of one slot race: what they leave there and return is
 * not defined. */
struct ccv1d_delta_update_args {
  const void* q; /* (rows, key_heads, key_dim) of type dtype, unit last stride; so k */
  int64_t q_stride_r, q_stride_h;
  const void* k;
  int64_t k_stride_r, k_stride_h;
  const void* v; /* (rows, heads, value_dim) */
  int64_t v_stride_r, v_stride_h;
  int dtype;
  const void* log_decay; /* (rows, heads) */
  int64_t log_decay_stride_r, log_decay_stride_h;
  int log_decay_dtype;
  int beta_dtype;
  const void* beta; /* (rows, heads) */
  int64_t beta_stride_r, beta_stride_h;
  float scale;
  float* state; /* (slots, heads, key_dim, value_dim), each slot contiguous */
  int64_t state_stride;
  const int32_t* state_indices; /* (rows,) or NULL: row r uses slot r */
  void* out;                    /* (rows, heads, value_dim) contiguous, type dtype */
  int64_t rows, slots, key_heads, heads, key_dim, value_dim;
  int device;
  void* stream;
};
int ccv1d_delta_update(const struct ccv1d_delta_update_args* args);

/* ---------------------------------------------------------------------------------------------
 * Norms around a block, over rows of dim elements; each part is left out where its pointer is NULL (one of the two norms is there):
 *
 *   m = x * post_weight / sqrt(mean(x^2) + eps)     (x without post_weight)
 *   m = m * act(gate)
 *   r = residual + scale * m                        (scale: a number, times scale_weight per channel)
 *   y = r * pre_weight / sqrt(mean(r^2) + eps)      with pre_weight only
 *
 * computed in fp32 whatever the types, each result rounded once (y from the unrounded r). Rows are counted by
 * two indices, outer and inner, with a stride for each.
 * ------------------------------------------------------------------------------------------- */
enum ccv1d_norm_activation { CCV1D_NORM_IDENTITY = 0, CCV1D_NORM_SILU = 1, CCV1D_NORM_SIGMOID = 2 };

/* Largest dim. */
#define CCV1D_NORM_MAX_DIM 8192

struct ccv1d_norm_args {
  const void* x; /* (outer, inner, dim) of type dtype, unit last stride; so gate and residual */
  int64_t x_stride_o, x_stride_i;
  const void* gate; /* type dtype, or NULL */
  int64_t gate_stride_o, gate_stride_i;
  const void* residual; /* type residual_dtype (dtype or F32), or NULL */
  int64_t residual_stride_o, residual_stride_i;
  int dtype;
  int residual_dtype;      /* of residual, r and their gradients; dtype without residual */
  const void* post_weight; /* (dim,) contiguous, or NULL */
  const void* scale_weight;
  const void* pre_weight;
  int post_dtype, scale_dtype, pre_dtype;
  float scale;
  float eps;
  int activation; /* enum ccv1d_norm_activation, of the gate */
  int64_t outer, inner, dim;
  /* forward */
  void* r; /* (outer, inner, dim) contiguous, type residual_dtype; NULL: not wanted (with pre_weight only) */
  void* y; /* (outer, inner, dim) contiguous, type dtype; required iff pre_weight */
  /* backward */
  const void* dr; /* type residual_dtype, unit last stride, or NULL */
  int64_t dr_stride_o, dr_stride_i;
  const void* dy; /* type dtype, unit last stride, or NULL; with pre_weight only */
  int64_t dy_stride_o, dy_stride_i;
  void* dx;           /* contiguous, type dtype */
  void* dgate;        /* contiguous, type dtype; required iff gate */
  void* dresidual;    /* contiguous, type residual_dtype; or NULL */
  void* dpost_weight; /* (dim,) of the weight's type; required iff post_weight */
  void* dscale_weight;
  void* dpre_weight;
  void* workspace;
  size_t workspace_bytes;
  int device;
  void* stream;
};
/* Bytes of workspace of the backward (the forward needs none): of the sizes and of which weights there are. */
size_t ccv1d_norm_workspace_bytes(const struct ccv1d_norm_args* args);
int ccv1d_norm_fwd(const struct ccv1d_norm_args* args);
/* The weights' gradients are deterministic: their order of summation depends on the sizes alone. */
int ccv1d_norm_bwd(const struct ccv1d_norm_args* args);

#ifdef __cplusplus
}
#endif

#endif /* CCV1D_LAYER_H */

"""Paged key-value caches for the attention layers that stand beside recurrent blocks in a model:

* `paged_plan` plans a batch of requests on the GPU from their lengths: pages from a free list, block
  tables, the slot of every new token, its position, and its request (which is also the seq_idx of
  causal_conv1d_fn and gated_recurrence_fn over the same batch of tokens);
* `paged_cache_write` writes new keys and values to their slots;
* `paged_attention` attends with one token per row over the cache.

A cache is (num_pages, page_size, kv_heads, head_dim), any strides but a unit last one; token p of
request r lies in page block_tables[r, p // page_size], at p % page_size. The kernels are hand-written
HIP kernels of libccv1d.so (include/ccv1d_ops.h). Nothing here waits for the GPU or reads a length on
the host, so a step can be captured in a graph. The reference package has no such operators.
"""

from typing import NamedTuple

from torch import Tensor

from ._ops import native


class PagedPlan(NamedTuple):
    """What paged_plan computes. `max_tokens` places hold the new tokens of all requests, one request
    after the other; places past the last token, and those of requests that were not admitted, hold
    -1."""

    seq_lens: Tensor      # (requests,) int32: cached + new tokens; cached only where not admitted
    query_start: Tensor   # (requests + 1,) int32: each request's first place, and their total
    positions: Tensor     # (max_tokens,) int32: a token's place in its sequence
    request_ids: Tensor   # (max_tokens,) int32
    slot_mapping: Tensor  # (max_tokens,) int64: page * page_size + offset
    num_free: Tensor      # (1,) int32: free pages left


def paged_plan(
    cached_lens: Tensor,
    new_lens: Tensor,
    block_tables: Tensor,
    free_pages: Tensor,
    num_free: Tensor,
    page_size: int,
    max_tokens: int,
) -> PagedPlan:
    """Plans a batch: request r has cached_lens[r] tokens in its pages and brings new_lens[r].

    Arguments:
      cached_lens, new_lens: (requests,) int32; negative lengths count as zero.
      block_tables: (requests, max_pages) int32 with contiguous rows, updated in place: the pages of
         the new tokens are noted after those of the cached ones.
      free_pages: (pages,) int32, a list whose first num_free entries are free pages. New pages are
         taken from its end, in order of request and position, so the list itself stays as it is and
         the plan's num_free says how much of it is left; pages given back are stored there.
      num_free: (1,) int32.
      page_size: tokens of a page.
      max_tokens: token places of the batch; tokens past them are not listed.

    A request is admitted when its tokens fit its row of block_tables and it either needs no new page
    or finds the pages that it and the requests before it need. Requests that are not admitted change
    nothing, and their tokens are padding.
    """
    return PagedPlan(*native().paged_plan(cached_lens, new_lens, block_tables, free_pages, num_free,
                                          page_size, max_tokens))


def paged_cache_write(
    k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slot_mapping: Tensor
) -> None:
    """Writes k and v, (tokens, kv_heads, head_dim) with a unit last stride, to the slots that
    slot_mapping (tokens,) names, in place. Tokens whose slot lies outside the cache (-1: padding) are
    left out. Caches and tokens have one type; rows of the caches must not overlap, nor the caches each
    other. Two tokens of one slot leave one of them there, or pieces of both. No backward."""
    native().paged_cache_write(k, v, k_cache, v_cache, slot_mapping)


def paged_attention(
    q: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    block_tables: Tensor,
    seq_lens: Tensor,
    softmax_scale: float | None = None,
    window: int | None = None,
    request_ids: Tensor | None = None,
    max_seq_len: int | None = None,
    return_lse: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """Attention of one token per row over a paged cache; query head h reads key head
    h // (q_heads // kv_heads). No backward.

    Arguments:
      q: (rows, q_heads, head_dim), unit last stride; head_dim a multiple of 8, at most 256. q and the
         caches are bf16, fp16 or fp32, one type for all.
      block_tables: (requests, max_pages) int32 with contiguous rows. Pages outside the cache are
         left out.
      seq_lens: (rows,) integers: row r attends to the positions before seq_lens[r], with `window`
         to the last `window` of them, counted from seq_lens[r] also where that passes the table or
         max_seq_len. A row with none (a length of zero) gets zeros.
      softmax_scale: head_dim ** -0.5 by default.
      request_ids: optional (rows,) integers: the request of each row (row r is request r without), for
         the tokens of a prompt (seq_lens = positions + 1). A negative one makes a row empty.
      max_seq_len: optional bound of seq_lens, which sizes the launch; the table's capacity by default,
         and where it is 0. Positions past it are left out.
      return_lse: also return the log-sum-exp of the scores, (rows, q_heads) fp32, -inf for empty rows.

    Returns out (rows, q_heads, head_dim) in q's dtype, or (out, lse). Softmax and sums are fp32.
    """
    assert window is None or window >= 1, "window must be at least 1"
    out, lse = native().paged_attention(q, k_cache, v_cache, block_tables, seq_lens, request_ids,
                                        softmax_scale, window or 0, max_seq_len or 0, return_lse)
    return (out, lse) if return_lse else out

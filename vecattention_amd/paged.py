"""A key-value cache in pages, and the step of a batch of requests over it, on
the MI355X kernels.

``single_decode_with_kv_cache`` attends over one sequence's contiguous cache.
Here the caches of several requests share pages of ``page_size`` tokens; slot s
of a cache is row s % page_size of page s // page_size.  One step, for prompts
and generated tokens alike:

1. ``paged_kv_plan``: pages for the new tokens, block tables, slots, positions;
2. ``qk_norm_rope`` and ``write_paged_kv`` for prompts, whose attention
   (``VecAttention_prefill``) wants the keys too, or ``qk_norm_rope_to_cache``
   for generated tokens;
3. ``paged_decode_attention``: one new token of every request over its pages.
   No operator attends from several new tokens of a request over its pages.

A cache is (num_pages, page_size, num_kv_heads, head_dim) with kv_layout "NHD",
(num_pages, num_kv_heads, page_size, head_dim) with "HND"; any strides with
contiguous features.  Nothing waits for the GPU or is kept between calls, so the
calls can be captured into a graph.
"""
from typing import NamedTuple

import torch

from . import _native as nat


class PagedStep(NamedTuple):
    """What a step needs to know, on the GPU (``paged_kv_plan``).  The tensors of
    the requests share one allocation, those of the tokens another."""
    kv_lens: torch.Tensor       # (N,) int32: lengths after the step
    qo_indptr: torch.Tensor     # (N + 1,) int32: first token of each request
    slot_mapping: torch.Tensor  # (num_tokens,) int64: slot of each token, -1 for none
    positions: torch.Tensor     # (num_tokens,) int64: its place among its request's tokens
    request_ids: torch.Tensor   # (num_tokens,) int32: its request, -1 for padding
    pages_taken: torch.Tensor   # (1,) int64: pages asked for


def paged_kv_plan(kv_lens, new_lens, block_tables, free_pages, page_size, num_tokens,
                  free_head=None):
    """Block tables, slots and positions of a step from the request lengths.

    kv_lens, new_lens: (N,) int32, tokens that each request holds and adds
    (either may be 0).  block_tables: (N, M) int32, updated in place: behind the
    ceil(kv_lens / page_size) pages that a row lists come the pages its new
    tokens need, taken from ``free_pages`` ((F,) int32) in the order of the
    requests, from entry ``free_head`` on (a one-element int32 tensor; None: 0).
    num_tokens: rows of the per-token outputs, at least sum(new_lens); further
    rows are padding (request -1, position 0, slot -1).  ``positions`` count a
    request's tokens; where the model's positions do not (the tokens of an image
    cover fewer of them than their number), the rotation takes ``positions`` plus
    the request's offset, indexed by ``request_ids``.

    Pages that the list no longer has give -1 entries and slots; then
    free_head + pages_taken exceeds F.  A token past the table's M pages has
    slot -1.  The operators below skip such slots, and ``paged_decode_attention``
    answers NaN for a request that cannot be read.
    """
    return PagedStep._make(nat.host_call("plan", block_tables, kv_lens, new_lens, block_tables,
                                         free_pages, page_size, num_tokens, free_head))


def write_paged_kv(k, v, k_cache, v_cache, slot_mapping, kv_layout="NHD"):
    """Keys and values of a step's tokens to their slots, in place.

    k, v: (T, num_kv_heads, head_dim) in the cache's dtype, any strides with
    contiguous features (a (1, Hk, S, D) prefill tensor: ``k[0].transpose(0,
    1)``).  slot_mapping: (T,) int64; a slot outside the cache (-1) takes
    nothing, the others must be distinct.
    """
    nat.host_call("write_kv", k, k, v, k_cache, v_cache, slot_mapping, kv_layout)


def qk_norm_rope_to_cache(q, k, v, k_cache, v_cache, slot_mapping, positions, inv_freq,
                          q_weight=None, k_weight=None, eps=1e-6, mrope_section=None,
                          interleaved=False, attention_scaling=1.0, kv_layout="NHD"):
    """``qk_norm_rope`` for a step's tokens, with the keys and values going to
    their slots of the caches in the same launch.

    q: (T, Hq, D); k, v: (T, Hk, D); positions (T,), or with ``mrope_section``
    (axes, T) ((T,): the same on every axis, as generated text has it; the
    positions of the model, which behind an image are not the plan's);
    slot_mapping and caches as in ``write_paged_kv``.  Returns the rotated queries
    (T, Hq, D); those of tokens without a slot too.
    """
    return nat.host_call("rope_to_cache", q, q, k, v, k_cache, v_cache, slot_mapping, positions,
                         inv_freq, q_weight, k_weight, eps, mrope_section, interleaved,
                         attention_scaling, kv_layout)


def paged_decode_attention(q, k_cache, v_cache, block_tables, kv_lens, kv_layout="NHD",
                           sm_scale=None):
    """Attention of one new token of every request over its pages.

    q: (N, num_qo_heads, head_dim); the caches in q's dtype (bf16/fp16/fp32,
    head_dim up to 256); block_tables: (N, M) int32; kv_lens: (N,) int32, the
    keys that each request's token sees (the new token's own among them).
    Returns (N, num_qo_heads, head_dim) in q's dtype: for each query head h the
    softmax(q . K_g^T * sm_scale) V_g of kv head g = h // (num_qo_heads //
    num_kv_heads), zeros where kv_lens is 0 (or less).

    A request whose length exceeds its table's M pages, or whose table names a
    page that the cache does not have, gives NaN.  Which form of the kernel runs
    goes by M: tables cut to the step's longest request (``block_tables[:, :m]``)
    are the faster ones for short requests.
    """
    return nat.host_call("decode", q, q, k_cache, v_cache, block_tables, kv_lens, kv_layout,
                         sm_scale)


__all__ = ["PagedStep", "paged_kv_plan", "write_paged_kv", "qk_norm_rope_to_cache",
           "paged_decode_attention"]

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

Rows of the batch may hold the same pages: several answers to one prompt, the
beams of a search.  Between two steps ``paged_kv_fork`` makes the next rows from
the present ones (rows go on, are forked, cut back or dropped) and
``copy_paged_kv`` copies what it lists in all layers; ``paged_kv_prefix`` finds
what rows begin with in common, once a step, and then
``paged_prefix_decode_attention`` reads it once for all of them.
``paged_kv_compact`` moves the pages in use together.

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


class PagedFork(NamedTuple):
    """The next step's rows (``paged_kv_fork``).  The tensors of the rows share one
    allocation, those of the pages another."""
    kv_lens: torch.Tensor       # (R,) int32
    block_tables: torch.Tensor  # (R, M) int32, -1 behind a row's pages
    page_shares: torch.Tensor   # (num_pages,) int32
    free_pages: torch.Tensor    # (F,) int32
    free_head: torch.Tensor     # (1,) int32: its first free entry
    copy_src: torch.Tensor      # (R,) int32: page that the row's last tokens are in, -1 for no copy
    copy_dst: torch.Tensor      # (R,) int32: page that they are to be in, -1 for no copy
    copy_rows: torch.Tensor     # (R,) int32: how many of them


def paged_kv_fork(kv_lens, parents, block_tables, page_shares, free_pages, page_size,
                  free_head=None, keep_lens=None):
    """The rows of the next step from those of this one, with the pages they share.

    kv_lens (N,), block_tables (N, M): the rows as they are.  parents: (R,), the row
    that each new row goes on from; one that several name is forked, one that none
    names is dropped, and a parent outside [0, N) (-1) makes an empty row.
    keep_lens: (R,), tokens that a new row keeps at most (None: all of them).
    page_shares: (num_pages,), the rows that hold each page beyond the first; zeros
    to begin with.  free_pages and free_head: the list that ``paged_kv_plan`` takes
    from.  All int32.  Nothing is written in place: the results replace them.

    Pages are shared, not copied, but for the one that a row's next tokens go into:
    where rows would share a page that is not full, each but one gets its own
    (``copy_src``, ``copy_dst``, ``copy_rows`` are what ``copy_paged_kv`` then copies
    in every layer).  Pages that no row holds any more return to the free list, in
    front of ``free_head`` and in ascending order, and the copies take theirs from
    there.  Where the list ends they get -1 (``paged_decode_attention`` answers NaN
    for such a row) and the new ``free_head`` exceeds the list; a list with an entry
    for every page of the cache has room for all that return.  At most 65536 rows, each
    of which looks at all before it: 33 us for 512 of long prompts, 0.1 ms for 8192 short
    ones, 2 ms for 65536.
    """
    return PagedFork._make(nat.host_call("fork", block_tables, kv_lens, parents, block_tables,
                                         page_shares, free_pages, page_size, free_head,
                                         keep_lens))


class PagedCompaction(NamedTuple):
    """Pages moved together (``paged_kv_compact``)."""
    block_tables: torch.Tensor  # (N, M) int32
    page_shares: torch.Tensor   # (num_pages,) int32
    free_pages: torch.Tensor    # (F,) int32: the free ones at its end, in ascending order
    free_head: torch.Tensor     # (1,) int32: its first free entry
    copy_src: torch.Tensor      # (num_pages // 2,) int32: pages to move, -1 behind them
    copy_dst: torch.Tensor      # (num_pages // 2,) int32: where to
    num_moves: torch.Tensor     # (1,) int32


def paged_kv_compact(kv_lens, block_tables, page_shares, free_pages, page_size, free_head=None):
    """The pages of the tables to the lowest numbers of those pages and the free ones.

    Arguments as for ``paged_kv_fork``.  Pages that are neither in the tables' rows
    nor in the list from ``free_head`` on stay where they are and keep their numbers,
    so the tables have to be all that may be renumbered.  ``copy_paged_kv(k_caches,
    v_caches, c.copy_src, c.copy_dst)`` moves the rows of every layer.
    """
    return PagedCompaction._make(nat.host_call("compact", block_tables, kv_lens, block_tables,
                                               page_shares, free_pages, page_size, free_head))


def copy_paged_kv(k_caches, v_caches, src_pages, dst_pages, rows=None, kv_layout="NHD"):
    """Pages to other pages of the same caches, in place, up to 32 layers a launch.

    k_caches, v_caches: the cache of one layer, or lists of those of all layers (one
    shape, type and strides).  src_pages, dst_pages: (C,) int32; an entry with a page
    outside the cache (-1) copies nothing.  The pages copied to must be distinct, and
    none of them copied from.  rows: (C,) int32, the tokens at the beginning of each
    page that are copied (None: all); the rows behind them stay.

    An empty entry takes time, a little of it: a list of 50000 that are all -1 takes
    44 us for 4 layers, 280 for 28.  A program that knows how many moves a compaction
    can have at most (its requests' pages) passes that much of the lists.
    """
    one = k_caches[0] if isinstance(k_caches, (list, tuple)) and k_caches else k_caches
    nat.host_call("copy", one, k_caches, v_caches, src_pages, dst_pages, rows, kv_layout)


class SharedPrefix(NamedTuple):
    """What neighbouring rows begin with in common (``paged_kv_prefix``)."""
    prefix_lens: torch.Tensor  # (N,) int32: tokens that the row's group shares, in whole pages
    group_rows: torch.Tensor   # (N,) int32: rows of the group that begins here, else 0


def paged_kv_prefix(kv_lens, block_tables, page_size, group_ids=None):
    """Which rows begin with the same pages, for ``paged_prefix_decode_attention``.

    Rows that follow each other, hold tokens and have the same group_ids ((N,) int32)
    are a group; without group_ids, rows whose first page is the same (a system
    prompt that all requests begin with makes one group of them: ids say which larger
    parts to share instead).  ``prefix_lens`` are the tokens of the whole pages that
    all rows of a group begin with, 0 where a row is alone.  What it finds stays true
    while rows grow; after a fork or a compaction it has to be found anew.  At most 65536
    rows, each of which looks at all before it: 10 us for 256, 0.2 ms for 8192, 10 ms
    for 65536.
    """
    return SharedPrefix._make(nat.host_call("prefix", block_tables, kv_lens, block_tables,
                                            page_size, group_ids))


def paged_prefix_decode_attention(q, k_cache, v_cache, block_tables, kv_lens, prefix,
                                  kv_layout="NHD", sm_scale=None):
    """``paged_decode_attention`` for rows that share the beginnings of their pages.

    prefix: ``paged_kv_prefix`` of these rows (a pair of prefix_lens and group_rows).
    The keys and values of a group's prefix are read once, for the query heads of all
    of its rows together, and every row's own keys after them; otherwise arguments and
    result are those of ``paged_decode_attention``, up to rounding: in 16-bit types a
    shared key's weight is rounded to the type's bits once, where the other keeps two
    parts, so an output is off by about its own rounding more (in bf16 2.3e-3 in the
    norm against 1.7e-3, in fp16 2.9e-4 against 2.1e-4).  Rows of a group hold at least
    prefix_lens tokens, and list the same pages for them.

    Batches too small to gain, by the tables' width, take ``paged_decode_attention``'s
    own path.  Past that, a batch that shares little takes longer here than there: by up
    to 12% with 28 + 4 heads of 128 and 30% with 16 + 16 of 64 where at most 64 tokens are
    shared, and by 3 to 9 us where tables have room for far more than the rows hold.
    """
    prefix_lens, group_rows = prefix
    return nat.host_call("prefix_decode", q, q, k_cache, v_cache, block_tables, kv_lens,
                         prefix_lens, group_rows, kv_layout, sm_scale)


__all__ = ["PagedStep", "paged_kv_plan", "write_paged_kv", "qk_norm_rope_to_cache",
           "paged_decode_attention", "PagedFork", "paged_kv_fork", "PagedCompaction",
           "paged_kv_compact", "copy_paged_kv", "SharedPrefix", "paged_kv_prefix",
           "paged_prefix_decode_attention"]

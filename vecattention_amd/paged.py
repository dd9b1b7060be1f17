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

A cache is (num_pages, page_size, num_kv_heads, head_dim) with kv_layout "NHD",
(num_pages, num_kv_heads, page_size, head_dim) with "HND"; any strides with
contiguous features.  Nothing waits for the GPU or is kept between calls, so the
calls can be captured into a graph.
"""
import functools
import math
import operator
from typing import NamedTuple

import torch

from . import _native as nat
from .rotary import refuse_devices, refuse_grad, rotation_args, rows_like


class PagedStep(NamedTuple):
    """What a step needs to know, on the GPU (``paged_kv_plan``)."""
    kv_lens: torch.Tensor       # (N,) int32: lengths after the step
    qo_indptr: torch.Tensor     # (N + 1,) int32: first token of each request
    slot_mapping: torch.Tensor  # (num_tokens,) int64: slot of each token, -1 for none
    positions: torch.Tensor     # (num_tokens,) int64: position in its request
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
    rows are padding (request -1, position 0, slot -1).

    Pages that the list no longer has give -1 entries and slots; then
    free_head + pages_taken exceeds F.  A token past the table's M pages has
    slot -1.  The operators below skip such slots, and ``paged_decode_attention``
    answers NaN for a request that cannot be read.
    """
    if kv_lens.dim() != 1 or kv_lens.shape != new_lens.shape:
        raise ValueError("kv_lens and new_lens must be vectors of one length")
    if block_tables.dim() != 2 or block_tables.shape[0] != kv_lens.shape[0]:
        raise ValueError(f"block_tables {tuple(block_tables.shape)}: expected "
                         f"({kv_lens.shape[0]}, pages)")
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be a vector")
    if free_head is not None and free_head.numel() != 1:
        raise ValueError("free_head must have one element")
    if not (kv_lens.dtype == new_lens.dtype == block_tables.dtype == free_pages.dtype
            == torch.int32) or free_head is not None and free_head.dtype != torch.int32:
        raise TypeError("lengths, block_tables, free_pages and free_head must be int32")
    page_size, num_tokens = operator.index(page_size), operator.index(num_tokens)
    if page_size <= 0:
        raise ValueError(f"page_size {page_size}")
    if num_tokens < 0:
        raise ValueError(f"num_tokens {num_tokens}")
    N, M = block_tables.shape
    row, entry = block_tables.stride()
    if M > 1 and entry != 1 or N > 1 and row < M:
        raise ValueError("block_tables needs contiguous rows of its own")
    dev = block_tables.get_device()
    if not (0 <= dev == kv_lens.get_device() == new_lens.get_device() == free_pages.get_device()
            and (free_head is None or free_head.get_device() == dev)):
        refuse_devices("paged_kv_plan", block_tables, kv_lens, new_lens, free_pages, free_head)
    device, empty = block_tables.device, torch.empty
    kv_lens, new_lens = kv_lens.contiguous(), new_lens.contiguous()
    free_pages = free_pages.contiguous()
    out = PagedStep(empty(N, dtype=torch.int32, device=device),
                    empty(N + 1, dtype=torch.int32, device=device),
                    empty(num_tokens, dtype=torch.int64, device=device),
                    empty(num_tokens, dtype=torch.int64, device=device),
                    empty(num_tokens, dtype=torch.int32, device=device),
                    empty(1, dtype=torch.int64, device=device))
    bytes_ = _plan_workspace(N)
    work = empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None
    with nat.on_device(device):
        rc = nat.lib().va_paged_plan(
            kv_lens.data_ptr(), new_lens.data_ptr(), N, block_tables.data_ptr(), row, M,
            free_pages.data_ptr(), free_pages.shape[0], nat.addr(free_head), page_size, num_tokens,
            *[t.data_ptr() for t in out], nat.addr(work), bytes_, nat.stream_addr(device))
    nat.check("va_paged_plan", rc)
    return out


# Workspace queries, which depend on their arguments alone.
@functools.lru_cache(maxsize=1024)
def _plan_workspace(N):
    return nat.lib().va_paged_plan_workspace_size(N)


@functools.lru_cache(maxsize=1024)
def _decode_workspace(*sizes):
    return max(nat.lib().va_paged_decode_workspace_size(*sizes), 16)


def _cache(k_cache, v_cache, kv_layout, D, dtype):
    """(num_pages, page_size, heads, page/row/head strides of K, those of V) of a checked cache."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must "
                         "be 4-dimensional and alike")
    kp, k1, k2, kd = k_cache.stride()
    vp, v1, v2, vd = v_cache.stride()
    if kv_layout == "NHD":
        pages, page, heads, width = k_cache.shape
        ks, vs = (kp, k1, k2), (vp, v1, v2)
    elif kv_layout == "HND":
        pages, heads, page, width = k_cache.shape
        ks, vs = (kp, k2, k1), (vp, v2, v1)
    else:
        raise KeyError(f"Invalid kv_layout {kv_layout}")
    if width != D:
        raise ValueError(f"a cache of shape {tuple(k_cache.shape)} does not hold rows of {D}")
    if not k_cache.dtype == v_cache.dtype == dtype:
        raise ValueError("the caches and the rows must share a dtype")
    if pages == 0 or page == 0:
        raise ValueError("the cache has no pages")
    if (kd != 1 or vd != 1) and D > 1:
        raise ValueError("k_cache and v_cache need contiguous head_dim")
    return pages, page, heads, ks, vs


def _tokens(k, v, slot_mapping):
    """k, v (features contiguous), slots, and k's shape, of a step's checked tokens."""
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be "
                         "(tokens, num_kv_heads, head_dim)")
    if v.dtype != k.dtype:
        raise ValueError(f"k ({k.dtype}) and v ({v.dtype}) must share a dtype")
    T, Hk, D = k.shape
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (T,):
        raise ValueError(f"slot_mapping must be int64 of ({T},)")
    return (k if k.stride(2) == 1 else k.contiguous(), v if v.stride(2) == 1 else v.contiguous(),
            slot_mapping.contiguous(), T, Hk, D)


def write_paged_kv(k, v, k_cache, v_cache, slot_mapping, kv_layout="NHD"):
    """Keys and values of a step's tokens to their slots, in place.

    k, v: (T, num_kv_heads, head_dim) in the cache's dtype, any strides with
    contiguous features (a (1, Hk, S, D) prefill tensor: ``k[0].transpose(0,
    1)``).  slot_mapping: (T,) int64; a slot outside the cache (-1) takes
    nothing, the others must be distinct.
    """
    k, v, slot_mapping, T, Hk, D = _tokens(k, v, slot_mapping)
    dtype = nat.dtype_code(k)
    pages, page, heads, ks, vs = _cache(k_cache, v_cache, kv_layout, D, k.dtype)
    if heads != Hk:
        raise ValueError(f"a cache of {heads} heads for keys of {Hk}")
    if not (0 <= k.get_device() == v.get_device() == k_cache.get_device() == v_cache.get_device()
            == slot_mapping.get_device()):
        refuse_devices("write_paged_kv", k, v, k_cache, v_cache, slot_mapping)
    refuse_grad("write_paged_kv", k, v, k_cache, v_cache)
    if T == 0 or Hk == 0 or D == 0:
        return
    device = k.device
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    with nat.on_device(device):
        rc = nat.lib().va_write_paged_kv(
            dtype, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, k_cache.data_ptr(), *ks,
            v_cache.data_ptr(), *vs, pages, page, slot_mapping.data_ptr(), T, Hk, D,
            nat.stream_addr(device))
    nat.check("va_write_paged_kv", rc)


def qk_norm_rope_to_cache(q, k, v, k_cache, v_cache, slot_mapping, positions, inv_freq,
                          q_weight=None, k_weight=None, eps=1e-6, mrope_section=None,
                          interleaved=False, attention_scaling=1.0, kv_layout="NHD"):
    """``qk_norm_rope`` for a step's tokens, with the keys and values going to
    their slots of the caches in the same launch.

    q: (T, Hq, D); k, v: (T, Hk, D); positions (T,), or with ``mrope_section``
    (axes, T) ((T,): the same on every axis, as generated text has it);
    slot_mapping and caches as in ``write_paged_kv``.  Returns the rotated queries
    (T, Hq, D); those of tokens without a slot too.
    """
    k, v, slot_mapping, T, Hk, D = _tokens(k, v, slot_mapping)
    if q.dim() != 3 or q.shape[0] != T or q.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)} must be (tokens, num_qo_heads, head_dim), with k's "
                         "tokens and head_dim")
    if q.dtype != k.dtype:
        raise ValueError(f"q ({q.dtype}) and k ({k.dtype}) must share a dtype")
    Hq = q.shape[1]
    dtype = nat.dtype_code(q)
    positions, spa, axes, sections, rot, wtype = rotation_args(
        D, q.dtype, positions, inv_freq, q_weight, k_weight, mrope_section, (T,))
    pages, page, heads, ks, vs = _cache(k_cache, v_cache, kv_layout, D, k.dtype)
    if heads != Hk:
        raise ValueError(f"a cache of {heads} heads for keys of {Hk}")
    dev = q.get_device()
    if not (0 <= dev == k.get_device() == v.get_device() == k_cache.get_device()
            == v_cache.get_device() == slot_mapping.get_device() == positions.get_device()
            == inv_freq.get_device()
            and (q_weight is None or q_weight.get_device() == dev)
            and (k_weight is None or k_weight.get_device() == dev)):
        refuse_devices("qk_norm_rope_to_cache", q, k, v, k_cache, v_cache, slot_mapping, positions,
                       inv_freq, q_weight, k_weight)
    refuse_grad("qk_norm_rope_to_cache", q, k, v, k_cache, v_cache, inv_freq, q_weight, k_weight)
    if q.stride(2) != 1:
        q = q.contiguous()
    out = rows_like(q)
    if T == 0 or Hq == 0 or Hk == 0:
        return out
    device = q.device
    qt, qh, _ = q.stride()
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    ot, oh, _ = out.stride()
    with nat.on_device(device):
        rc = nat.lib().va_qk_norm_rope_to_cache(
            dtype, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
            out.data_ptr(), ot, oh, k_cache.data_ptr(), *ks, v_cache.data_ptr(), *vs, pages, page,
            slot_mapping.data_ptr(), T, Hq, Hk, D, positions.data_ptr(), spa, axes, sections,
            inv_freq.data_ptr(), rot, nat.addr(q_weight), nat.addr(k_weight), wtype,
            float(eps), float(attention_scaling), 1 if interleaved else 0, nat.stream_addr(device))
    nat.check("va_qk_norm_rope_to_cache", rc)
    return out


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
    page that the cache does not have, gives NaN.
    """
    if q.dim() != 3:
        raise ValueError("q must be (requests, num_qo_heads, head_dim)")
    N, Hq, D = q.shape
    dtype = nat.dtype_code(q)
    pages, page, Hk, ks, vs = _cache(k_cache, v_cache, kv_layout, D, q.dtype)
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"num_qo_heads {Hq} is not a multiple of num_kv_heads {Hk}")
    if block_tables.dim() != 2 or block_tables.shape[0] != N or kv_lens.shape != (N,):
        raise ValueError(f"block_tables {tuple(block_tables.shape)} and kv_lens "
                         f"{tuple(kv_lens.shape)} do not fit {N} requests")
    if not block_tables.dtype == kv_lens.dtype == torch.int32:
        raise TypeError("block_tables and kv_lens must be int32")
    if not (0 <= q.get_device() == k_cache.get_device() == v_cache.get_device()
            == block_tables.get_device() == kv_lens.get_device()):
        refuse_devices("paged_decode_attention", q, k_cache, v_cache, block_tables, kv_lens)
    refuse_grad("paged_decode_attention", q, k_cache, v_cache)
    M = block_tables.shape[1]
    qn, qh, qd = q.stride()
    if qd != 1:
        q = q.contiguous()
        qn, qh, qd = q.stride()
    row, entry = block_tables.stride()
    if M > 1 and entry != 1:
        block_tables = block_tables.contiguous()
        row = M
    kv_lens = kv_lens.contiguous()
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    device = q.device
    out = torch.empty((N, Hq, D), dtype=q.dtype, device=device)
    if N * Hq * D == 0:
        return out
    bytes_ = _decode_workspace(dtype, N, Hq, Hk, D, M, page)
    work = torch.empty(bytes_, dtype=torch.uint8, device=device)
    with nat.on_device(device):
        rc = nat.lib().va_paged_decode_attn(
            dtype, q.data_ptr(), qn, qh, k_cache.data_ptr(), *ks, v_cache.data_ptr(), *vs,
            out.data_ptr(), Hq * D, D, block_tables.data_ptr(), row, M, kv_lens.data_ptr(), N, Hq,
            Hk, D, page, pages, float(sm_scale), work.data_ptr(), bytes_, nat.stream_addr(device))
    nat.check("va_paged_decode_attn", rc)
    return out


__all__ = ["PagedStep", "paged_kv_plan", "write_paged_kv", "qk_norm_rope_to_cache",
           "paged_decode_attention"]

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
import math
from typing import NamedTuple

import torch

from . import _native as nat
from .rotary import refuse_grad, rotation_args, rows_like, same_device


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
    for name, t in (("kv_lens", kv_lens), ("new_lens", new_lens), ("block_tables", block_tables),
                    ("free_pages", free_pages), ("free_head", free_head)):
        if t is not None and t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, not {t.dtype}")
    if page_size <= 0:
        raise ValueError(f"page_size {page_size}")
    if num_tokens < 0:
        raise ValueError(f"num_tokens {num_tokens}")
    N, M = block_tables.shape
    if M > 1 and block_tables.stride(1) != 1 or N > 1 and block_tables.stride(0) < M:
        raise ValueError("block_tables needs contiguous rows of its own")
    device = block_tables.device
    if not block_tables.is_cuda:
        raise RuntimeError("paged_kv_plan runs on the GPU")
    same_device("paged_kv_plan", device, kv_lens, new_lens, free_pages, free_head)
    kv_lens, new_lens, free_pages = (t.contiguous() for t in (kv_lens, new_lens, free_pages))
    out = PagedStep(torch.empty(N, dtype=torch.int32, device=device),
                    torch.empty(N + 1, dtype=torch.int32, device=device),
                    torch.empty(num_tokens, dtype=torch.int64, device=device),
                    torch.empty(num_tokens, dtype=torch.int64, device=device),
                    torch.empty(num_tokens, dtype=torch.int32, device=device),
                    torch.empty(1, dtype=torch.int64, device=device))
    lib = nat.lib()
    bytes_ = lib.va_paged_plan_workspace_size(N)
    work = torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None
    with nat.on_device(device):
        rc = lib.va_paged_plan(
            nat.addr(kv_lens), nat.addr(new_lens), N, nat.addr(block_tables),
            block_tables.stride(0), M, nat.addr(free_pages), free_pages.shape[0],
            nat.addr(free_head), page_size, num_tokens, nat.addr(out.kv_lens),
            nat.addr(out.qo_indptr), nat.addr(out.slot_mapping), nat.addr(out.positions),
            nat.addr(out.request_ids), nat.addr(out.pages_taken), nat.addr(work), bytes_,
            nat.stream_addr(device))
    nat.check("va_paged_plan", rc)
    return out


def _cache(k_cache, v_cache, kv_layout, Hk, D, dtype):
    """(num_pages, page_size, page/row/head strides of K, those of V) of a checked cache."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must "
                         "be 4-dimensional and alike")
    if kv_layout == "NHD":
        row, head = 1, 2
    elif kv_layout == "HND":
        row, head = 2, 1
    else:
        raise KeyError(f"Invalid kv_layout {kv_layout}")
    if k_cache.shape[head] != Hk or k_cache.shape[3] != D:
        raise ValueError(f"a {kv_layout} cache of shape {tuple(k_cache.shape)} does not hold "
                         f"{Hk} heads of {D}")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError("the caches and the rows must share a dtype")
    if k_cache.shape[0] == 0 or k_cache.shape[row] == 0:
        raise ValueError("the cache has no pages")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and D > 1:
        raise ValueError("k_cache and v_cache need contiguous head_dim")
    return (k_cache.shape[0], k_cache.shape[row], (ks[0], ks[row], ks[head]),
            (vs[0], vs[row], vs[head]))


def _tokens(k, v, slot_mapping):
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be "
                         "(tokens, num_kv_heads, head_dim)")
    if v.dtype != k.dtype:
        raise ValueError(f"k ({k.dtype}) and v ({v.dtype}) must share a dtype")
    if tuple(slot_mapping.shape) != (k.shape[0],) or slot_mapping.dtype != torch.int64:
        raise ValueError(f"slot_mapping must be int64 of ({k.shape[0]},)")
    return (k if k.stride(2) == 1 else k.contiguous(), v if v.stride(2) == 1 else v.contiguous(),
            slot_mapping.contiguous())


def write_paged_kv(k, v, k_cache, v_cache, slot_mapping, kv_layout="NHD"):
    """Keys and values of a step's tokens to their slots, in place.

    k, v: (T, num_kv_heads, head_dim) in the cache's dtype, any strides with
    contiguous features (a (1, Hk, S, D) prefill tensor: ``k[0].transpose(0,
    1)``).  slot_mapping: (T,) int64; a slot outside the cache (-1) takes
    nothing, the others must be distinct.
    """
    k, v, slot_mapping = _tokens(k, v, slot_mapping)
    T, Hk, D = k.shape
    dtype = nat.dtype_code(k)
    pages, page, ks, vs = _cache(k_cache, v_cache, kv_layout, Hk, D, k.dtype)
    if not k.is_cuda:
        raise RuntimeError("write_paged_kv runs on the GPU")
    same_device("write_paged_kv", k.device, v, k_cache, v_cache, slot_mapping)
    refuse_grad("write_paged_kv", k, v, k_cache, v_cache)
    if k.numel() == 0:
        return
    with nat.on_device(k.device):
        rc = nat.lib().va_write_paged_kv(
            dtype, nat.addr(k), k.stride(0), k.stride(1), nat.addr(v), v.stride(0), v.stride(1),
            nat.addr(k_cache), *ks, nat.addr(v_cache), *vs, pages, page, nat.addr(slot_mapping),
            T, Hk, D, nat.stream_addr(k.device))
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
    if q.dim() != 3 or q.shape[0] != k.shape[0]:
        raise ValueError(f"q {tuple(q.shape)} must be (tokens, num_qo_heads, head_dim), with k's "
                         "tokens")
    k, v, slot_mapping = _tokens(k, v, slot_mapping)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    dtype = nat.dtype_code(q)
    positions, spa, axes, sections, rot, wtype = rotation_args(
        q, k, positions, inv_freq, q_weight, k_weight, mrope_section, (T,))
    pages, page, ks, vs = _cache(k_cache, v_cache, kv_layout, Hk, D, k.dtype)
    if not q.is_cuda:
        raise RuntimeError("qk_norm_rope_to_cache runs on the GPU")
    same_device("qk_norm_rope_to_cache", q.device, k, v, k_cache, v_cache, slot_mapping, positions,
                inv_freq, q_weight, k_weight)
    refuse_grad("qk_norm_rope_to_cache", q, k, v, k_cache, v_cache, inv_freq, q_weight, k_weight)
    if q.stride(2) != 1:
        q = q.contiguous()
    out = rows_like(q)
    if T == 0 or Hq == 0 or Hk == 0:
        return out
    with nat.on_device(q.device):
        rc = nat.lib().va_qk_norm_rope_to_cache(
            dtype, nat.addr(q), q.stride(0), q.stride(1), nat.addr(k), k.stride(0), k.stride(1),
            nat.addr(v), v.stride(0), v.stride(1), nat.addr(out), out.stride(0), out.stride(1),
            nat.addr(k_cache), *ks, nat.addr(v_cache), *vs, pages, page, nat.addr(slot_mapping),
            T, Hq, Hk, D, nat.addr(positions), spa, axes, sections, nat.addr(inv_freq), rot,
            nat.addr(q_weight), nat.addr(k_weight), wtype, eps, attention_scaling,
            int(interleaved), nat.stream_addr(q.device))
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
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be 4-dimensional")
    Hk = k_cache.shape[1 if kv_layout == "HND" else 2]
    dtype = nat.dtype_code(q)
    pages, page, ks, vs = _cache(k_cache, v_cache, kv_layout, Hk, D, q.dtype)
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"num_qo_heads {Hq} is not a multiple of num_kv_heads {Hk}")
    if block_tables.dim() != 2 or block_tables.shape[0] != N or tuple(kv_lens.shape) != (N,):
        raise ValueError(f"block_tables {tuple(block_tables.shape)} and kv_lens "
                         f"{tuple(kv_lens.shape)} do not fit {N} requests")
    if block_tables.dtype != torch.int32 or kv_lens.dtype != torch.int32:
        raise TypeError("block_tables and kv_lens must be int32")
    if not q.is_cuda:
        raise RuntimeError("paged_decode_attention runs on the GPU")
    same_device("paged_decode_attention", q.device, k_cache, v_cache, block_tables, kv_lens)
    refuse_grad("paged_decode_attention", q, k_cache, v_cache)
    M = block_tables.shape[1]
    if q.stride(2) != 1:
        q = q.contiguous()
    if M > 1 and block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    kv_lens = kv_lens.contiguous()
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    out = torch.empty(N, Hq, D, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    lib = nat.lib()
    bytes_ = max(lib.va_paged_decode_workspace_size(dtype, N, Hq, Hk, D, M, page), 16)
    work = torch.empty(bytes_, dtype=torch.uint8, device=q.device)
    with nat.on_device(q.device):
        rc = lib.va_paged_decode_attn(
            dtype, nat.addr(q), q.stride(0), q.stride(1), nat.addr(k_cache), *ks,
            nat.addr(v_cache), *vs, nat.addr(out), Hq * D, D, nat.addr(block_tables),
            block_tables.stride(0), M, nat.addr(kv_lens), N, Hq, Hk, D, page, pages,
            float(sm_scale), nat.addr(work), bytes_, nat.stream_addr(q.device))
    nat.check("va_paged_decode_attn", rc)
    return out


__all__ = ["PagedStep", "paged_kv_plan", "write_paged_kv", "qk_norm_rope_to_cache",
           "paged_decode_attention"]

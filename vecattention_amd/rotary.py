"""Norms of queries and keys for each head with the position rotation, in one
pass, on the MI355X kernels.

What a patched attention forward does between its projections and
``VecAttention_prefill`` (rotary embedding, over one position axis or the three
of a vision-language model: spattn/src/models/load_qwen2p5_vl.py:42-45), with
the per-head RMS norms that some models put before it.  Everything is computed
in fp32 from angles reduced in 64 bits, and rounded once.
"""
import ctypes

import torch

from . import _native as nat


def refuse_grad(what, *tensors):
    """These operators have no backward pass: say so rather than cut a graph."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError(
                    f"{what} has no backward pass: call it under torch.no_grad()")


def same_device(what, device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")


def _sections(mrope_section, half):
    if mrope_section is None:
        return 1, None
    axes = len(mrope_section)
    if not 1 <= axes <= 4:
        raise ValueError(f"mrope_section has {axes} entries; 1 to 4 position axes are supported")
    if any(n < 0 for n in mrope_section) or sum(mrope_section) != half:
        raise ValueError(f"mrope_section {list(mrope_section)} does not add up to {half}")
    return axes, (ctypes.c_int64 * axes)(*mrope_section)


def rotation_args(q, k, positions, inv_freq, q_weight, k_weight, mrope_section, tokens):
    """Checked arguments that both forms share: (positions, its axis stride, number of axes,
    sections, rotary_dim, weight type).  tokens: the shape of one axis' positions."""
    D = q.shape[-1]
    if k.shape[-1] != D:
        raise ValueError(f"head_dim of q ({D}) and k ({k.shape[-1]}) differ")
    if q.dtype != k.dtype:
        raise ValueError(f"q ({q.dtype}) and k ({k.dtype}) must share a dtype")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 vector")
    rot = 2 * inv_freq.shape[0]
    if not 0 < rot <= D:
        raise ValueError(f"inv_freq has {rot // 2} frequencies for a head_dim of {D}")
    axes, sections = _sections(mrope_section, rot // 2)
    if positions.dtype != torch.int64:
        if positions.dtype != torch.int32:
            raise TypeError(f"positions must be int64 or int32, not {positions.dtype}")
        positions = positions.long()
    shape = tuple(tokens) if mrope_section is None else (axes, *tokens)
    if tuple(positions.shape) != shape:
        # (S,) for every row of the batch; (T,) of a step's tokens for every axis.
        if tuple(positions.shape) != shape[:-2] + shape[-1:]:
            raise ValueError(f"positions {tuple(positions.shape)}: expected {shape}")
        positions = positions.unsqueeze(-2).expand(shape)
    if shape[-1] > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    weight_type = q.dtype
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if tuple(w.shape) != (D,) or not w.is_contiguous():
            raise ValueError(f"norm weights must be contiguous, of {D} values")
        if w.dtype not in (q.dtype, torch.float32):
            raise ValueError(f"norm weights of {w.dtype} for rows of {q.dtype}")
        weight_type = w.dtype
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must share a dtype")
    return (positions, positions.stride(0) if mrope_section is not None else 0, axes, sections,
            rot, nat.VA_F32 if weight_type == torch.float32 else nat.dtype_code(q))


def rows_like(x):
    """An output of x's shape with x's order of dimensions and contiguous features."""
    out = torch.empty_like(x)
    return out if out.stride(-1) == 1 or out.shape[-1] == 1 else torch.empty(
        x.shape, dtype=x.dtype, device=x.device)


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6,
                 mrope_section=None, interleaved=False, attention_scaling=1.0):
    """Per-head RMS norms and rotation of a prefill's queries and keys.

    q: (B, Hq, S, D), k: (B, Hk, S, D), bf16/fp16/fp32, any strides with
    contiguous features (others are copied); D up to 512.  Returns (q, k) as new
    tensors in the same order of dimensions.

    q_weight, k_weight: (D,) norm weights in q's dtype or fp32 (None: no norm):
    x * rsqrt(mean(x^2) + eps) * w over each head's row.
    positions: integers (B, S) or (S,), or with ``mrope_section`` (its entries
    are the frequencies that each position axis turns, at most four axes)
    (axes, B, S) or (axes, S).  inv_freq: fp32 (rotary_dim / 2,); features from
    rotary_dim on are left alone.  Pairs are (f, f + rotary_dim / 2), or
    ``interleaved`` (2f, 2f + 1).  attention_scaling multiplies cos and sin.
    """
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be (batch, heads, seq, head_dim)")
    B, Hq, S, D = q.shape
    if (k.shape[0], k.shape[2]) != (B, S):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or length")
    dtype = nat.dtype_code(q)
    positions, spa, axes, sections, rot, wtype = rotation_args(
        q, k, positions, inv_freq, q_weight, k_weight, mrope_section, (B, S))
    if not q.is_cuda:
        raise RuntimeError("qk_norm_rope runs on the GPU")
    same_device("qk_norm_rope", q.device, k, positions, inv_freq, q_weight, k_weight)
    refuse_grad("qk_norm_rope", q, k, inv_freq, q_weight, k_weight)
    if q.stride(3) != 1:
        q = q.contiguous()
    if k.stride(3) != 1:
        k = k.contiguous()
    qo, ko = rows_like(q), rows_like(k)
    if B * S == 0 or Hq == 0 or k.shape[1] == 0:
        return qo, ko
    with nat.on_device(q.device):
        rc = nat.lib().va_qk_norm_rope(
            dtype, nat.addr(q), *q.stride()[:3], nat.addr(k), *k.stride()[:3], nat.addr(qo),
            *qo.stride()[:3], nat.addr(ko), *ko.stride()[:3], B, Hq, k.shape[1], S, D,
            nat.addr(positions), spa, positions.stride(-2), axes, sections, nat.addr(inv_freq),
            rot, nat.addr(q_weight), nat.addr(k_weight), wtype, eps, attention_scaling,
            int(interleaved), nat.stream_addr(q.device))
    nat.check("va_qk_norm_rope", rc)
    return qo, ko


__all__ = ["qk_norm_rope"]

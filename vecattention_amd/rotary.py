"""Norms of queries and keys for each head with the position rotation, in one
pass, on the MI355X kernels.

What a patched attention forward does between its projections and
``VecAttention_prefill`` (rotary embedding, over one position axis or the three
of a vision-language model: spattn/src/models/load_qwen2p5_vl.py:42-45), with
the per-head RMS norms that some models put before it.  Everything is computed
in fp32 from angles reduced in 64 bits, and rounded once.
"""
import ctypes
import functools

import torch

from . import _native as nat


def refuse_grad(what, *tensors):
    """These operators have no backward pass: say so rather than cut a graph."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError(
                    f"{what} has no backward pass: call it under torch.no_grad()")


def refuse_devices(what, *tensors):
    """The error for tensors that are not all on one GPU."""
    if not tensors[0].is_cuda:
        raise RuntimeError(f"{what} runs on the GPU")
    for t in tensors:
        if t is not None and t.device != tensors[0].device:
            raise ValueError(f"{what}: tensors on {tensors[0].device} and {t.device}")


@functools.lru_cache(maxsize=256)
def _sections(section, half):
    """(axes, their sections for the C call)."""
    axes = len(section)
    if not 1 <= axes <= 4:
        raise ValueError(f"mrope_section has {axes} entries; 1 to 4 position axes are supported")
    if any(n < 0 for n in section) or sum(section) != half:
        raise ValueError(f"mrope_section {list(section)} does not add up to {half}")
    return axes, (ctypes.c_int64 * axes)(*section)


def rotation_args(D, dtype, positions, inv_freq, q_weight, k_weight, mrope_section, tokens):
    """Checked arguments that both forms share: (positions, its axis stride, number of axes,
    sections, rotary_dim, weight type).  tokens: the shape of one axis' positions."""
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 vector")
    half = inv_freq.shape[0]
    if not 0 < 2 * half <= D:
        raise ValueError(f"inv_freq has {half} frequencies for a head_dim of {D}")
    if mrope_section is None:
        axes, sections, shape = 1, None, tokens
    else:
        axes, sections = _sections(tuple(mrope_section), half)
        shape = (axes, *tokens)
    if positions.dtype != torch.int64:
        if positions.dtype != torch.int32:
            raise TypeError(f"positions must be int64 or int32, not {positions.dtype}")
        positions = positions.long()
    if positions.shape != shape:
        # (S,) for every row of the batch; (T,) of a step's tokens for every axis.
        if positions.shape != shape[:-2] + shape[-1:]:
            raise ValueError(f"positions {tuple(positions.shape)}: expected {shape}")
        positions = positions.unsqueeze(-2).expand(shape)
    if shape[-1] > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    weight_type = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.shape != (D,) or not w.is_contiguous():
            raise ValueError(f"norm weights must be contiguous, of {D} values")
        if w.dtype != dtype and w.dtype != torch.float32:
            raise ValueError(f"norm weights of {w.dtype} for rows of {dtype}")
        if weight_type is not None and w.dtype != weight_type:
            raise ValueError("q_weight and k_weight must share a dtype")
        weight_type = w.dtype
    return (positions, 0 if sections is None else positions.stride(0), axes, sections, 2 * half,
            nat.VA_F32 if weight_type == torch.float32 else nat.DTYPES[dtype])


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
    Bk, Hk, Sk, Dk = k.shape
    if Bk != B or Sk != S or Dk != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, length or "
                         "head_dim")
    if q.dtype != k.dtype:
        raise ValueError(f"q ({q.dtype}) and k ({k.dtype}) must share a dtype")
    dtype = nat.dtype_code(q)
    positions, spa, axes, sections, rot, wtype = rotation_args(
        D, q.dtype, positions, inv_freq, q_weight, k_weight, mrope_section, (B, S))
    dev = q.get_device()
    if not (0 <= dev == k.get_device() == positions.get_device() == inv_freq.get_device()
            and (q_weight is None or q_weight.get_device() == dev)
            and (k_weight is None or k_weight.get_device() == dev)):
        refuse_devices("qk_norm_rope", q, k, positions, inv_freq, q_weight, k_weight)
    refuse_grad("qk_norm_rope", q, k, inv_freq, q_weight, k_weight)
    qb, qh, qs, qd = q.stride()
    if qd != 1:
        q = q.contiguous()
        qb, qh, qs, qd = q.stride()
    kb, kh, ks, kd = k.stride()
    if kd != 1:
        k = k.contiguous()
        kb, kh, ks, kd = k.stride()
    qo, ko = rows_like(q), rows_like(k)
    if B * S == 0 or Hq == 0 or Hk == 0:
        return qo, ko
    qob, qoh, qos, _ = qo.stride()
    kob, koh, kos, _ = ko.stride()
    device = q.device
    with nat.on_device(device):
        rc = nat.lib().va_qk_norm_rope(
            dtype, q.data_ptr(), qb, qh, qs, k.data_ptr(), kb, kh, ks, qo.data_ptr(), qob, qoh,
            qos, ko.data_ptr(), kob, koh, kos, B, Hq, Hk, S, D, positions.data_ptr(), spa,
            positions.stride(-2), axes, sections, inv_freq.data_ptr(), rot, nat.addr(q_weight),
            nat.addr(k_weight), wtype, float(eps), float(attention_scaling),
            1 if interleaved else 0,
            nat.stream_addr(device))
    nat.check("va_qk_norm_rope", rc)
    return qo, ko


__all__ = ["qk_norm_rope"]

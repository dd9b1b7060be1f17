"""Norms of queries and keys for each head with the position rotation, in one
pass, on the MI355X kernels.

What a patched attention forward does between its projections and
``VecAttention_prefill`` (rotary embedding, over one position axis or the three
of a vision-language model: spattn/src/models/load_qwen2p5_vl.py:42-45), with
the per-head RMS norms that some models put before it.  Everything is computed
in fp32 from angles reduced in 64 bits, and rounded once.
"""
from . import _native as nat


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6,
                 mrope_section=None, interleaved=False, attention_scaling=1.0):
    """Per-head RMS norms and rotation of a prefill's queries and keys.

    q: (B, Hq, S, D), k: (B, Hk, S, D), bf16/fp16/fp32, any strides with
    contiguous features (others are copied); D up to 512.  Returns (q, k) as new
    tensors in the same order of dimensions.

    q_weight, k_weight: (D,) norm weights in q's dtype or fp32 (None: no norm):
    x * rsqrt(mean(x^2) + eps) * w over each head's row (a norm over the features of
    all heads together is the caller's, who then passes no weights).
    positions: integers (B, S) or (S,), or with ``mrope_section`` (its entries
    are the frequencies that each position axis turns, at most four axes)
    (axes, B, S) or (axes, S).  inv_freq: fp32 (rotary_dim / 2,); features from
    rotary_dim on are left alone.  Pairs are (f, f + rotary_dim / 2), or
    ``interleaved`` (2f, 2f + 1).  attention_scaling multiplies cos and sin.
    """
    return nat.host_call("rope", q, q, k, positions, inv_freq, q_weight, k_weight, eps,
                         mrope_section, interleaved, attention_scaling)


__all__ = ["qk_norm_rope"]

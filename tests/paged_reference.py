"""Plain 64-bit forms of the paged-cache operators, and what their fp32 kernels
may differ from them by."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# A value below the smallest normal number is rounded to a fixed step.
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def plan(kv_lens, new_lens, table, free, page, num_tokens, head=0):
    """(table, kv_lens, indptr, slots, positions, requests, taken), request by request."""
    table = [list(map(int, r)) for r in table]
    free, width = list(map(int, free)), len(table[0]) if table else 0
    at, lens, indptr, slots, pos, req = head, [], [0], [], [], []
    for i, (l, n) in enumerate(zip(map(int, kv_lens), map(int, new_lens))):
        l, n = max(l, 0), max(n, 0)
        for p in range(-(-l // page), min(-(-(l + n) // page), width)):
            table[i][p] = free[at] if 0 <= at < len(free) else -1
            at += 1
        for t in range(l, l + n):
            p = t // page
            ok = p < width and table[i][p] >= 0
            slots.append(table[i][p] * page + t % page if ok else -1)
            pos.append(t)
            req.append(i)
        lens.append(min(l + n, 2 ** 31 - 1))
        indptr.append(indptr[-1] + n)
    pad = num_tokens - len(slots)
    if pad > 0:
        slots, pos, req = slots + [-1] * pad, pos + [0] * pad, req + [-1] * pad
    return (table, lens, indptr, slots[:num_tokens], pos[:num_tokens], req[:num_tokens], at - head)


def rotate(x, positions, inv_freq, weight=None, eps=1e-6, sections=None, interleaved=False,
           scaling=1.0):
    """x (..., D) in 64 bits; positions (...) or (axes, ...) broadcast to x's rows.
    Returns the result and what its fp32 evaluation may be off by."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    rot = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    if sections is not None:
        parts = torch.split(angle, sections, -1)
        angle = torch.cat([p[a] for a, p in enumerate(parts)], -1)
    cos, sin = angle.cos() * scaling, angle.sin() * scaling
    y, size = x.clone(), x.abs()
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * max(1.0, abs(scaling))
    # Roundings to fp32 on the way, each at most 2^-24 of the sizes that meet there: the squares'
    # sum (at most D/64 + 7 terms after one another, halved by the root), mean, eps, root,
    # quotient and two products (14); the part of a turn (2^-25 of half a turn, times pi: 2), the
    # sine and cosine (4, their stated error) and scaling; two products and a sum: 24 in all.
    return y, 32 * 2.0 ** -24 * size


def rounded(want, slack, dtype):
    """The slack with the one rounding of the output added."""
    return slack + HALF_STEP[dtype] * (want.abs() + slack) + SMALLEST[dtype]


def cache_rows(cache, layout):
    """(num_pages * page_size, Hk, D) of a cache."""
    x = cache if layout == "NHD" else cache.transpose(1, 2)
    return x.reshape(-1, x.shape[2], x.shape[3])


def decode(q, k_cache, v_cache, table, lens, layout, scale=None):
    """(want, slack) of decode attention, request by request in 64 bits."""
    N, Hq, D = q.shape
    page = k_cache.shape[1 if layout == "NHD" else 2]
    k_rows, v_rows = cache_rows(k_cache, layout), cache_rows(v_cache, layout)
    Hk = k_rows.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    want, slack = torch.zeros(N, Hq, D).double(), torch.zeros(N, Hq, D).double()
    for n in range(N):
        L = int(lens[n])
        if L <= 0:
            continue
        t = torch.arange(L)
        at = table[n].long()[t // page] * page + t % page
        k = k_rows[at].double().repeat_interleave(Hq // Hk, 1)
        v = v_rows[at].double().repeat_interleave(Hq // Hk, 1)
        x = q[n].double()
        s = (k * x).sum(-1) * scale
        p = torch.softmax(s, 0)
        want[n] = (p[..., None] * v).sum(0)
        # A score is a sum of D products (D + 1 roundings of at most 2^-24 of the sum of the
        # products' sizes), scaled (2 roundings); the exponent's argument is a difference of
        # scaled scores (1) and exp2 is good to 2^-23: each weight is off by that factor, and so
        # is the weights' sum, which adds at most L roundings, as does the sum of the values.
        # 16-bit types hold a weight in two parts, to 2^-16.
        off = ((k * x).abs().sum(-1) * abs(scale) * (D + 1)).max() + 4 * s.abs().max() + 4
        part = 0.0 if q.dtype == torch.float32 else 2.0 ** -16
        rel = 2 * (off + 2 * L) * 2.0 ** -24 + 2 * part
        slack[n] = rel * (p[..., None] * v.abs()).sum(0)
    return want, slack

"""Workloads of the operators of a decode step over a paged key-value cache.

A program that prefills prompts and then generates for several requests at once keeps keys and
values in pages of a few tokens.  Each step plans where its tokens go, rotates queries and keys,
writes keys and values to their slots, and attends from every request's new token:

- ``plan``: block tables, slots and positions of a step from the request lengths
  (``paged_kv_plan``).
- ``rope``: norms of queries and keys for each head and the position rotation, on a prefill's
  (B, H, S, D) tensors (``qk_norm_rope``).
- ``store``: the same for a step's tokens, with keys and values going straight to their slots
  (``qk_norm_rope_to_cache``).
- ``write``: a prompt's keys and values to their slots (``write_paged_kv``).
- ``decode``: attention of one new token for each request over its pages
  (``paged_decode_attention``).

Each has its plain form in elementary torch operations, which runs where ``own`` is false.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA, EPS = 1e6, 1e-6


def listed():
    return [
        # One token for each of 32 requests: the smallest plan, once for every generated token.
        {"name": "plan-decode-32", "kind": "plan", "N": 32, "page": 16, "longest": 4096,
         "prompts": 0, "prompt": 0},
        # A step that takes up 96 new prompts of up to 4096 tokens beside 400 running requests.
        {"name": "plan-mixed-496", "kind": "plan", "N": 496, "page": 16, "longest": 32768,
         "prompts": 96, "prompt": 4096},
        # A short image prompt of a vision-language model: rotation over three position axes, no
        # norms, on the projections' (B, S, H, D) memory; a ragged length.
        {"name": "rope-vlm-2333", "kind": "rope", "B": 1, "S": 2333, "Hq": 28, "Hk": 4, "D": 128,
         "rot": 128, "norm": False, "axes": 3, "pairs": "half", "bshd": True, "dtype": "bf16"},
        # One layer of a video DiT: norms of each head, neighbouring features rotated, contiguous
        # (B, H, S, D), in fp16.
        {"name": "rope-dit-32760", "kind": "rope", "B": 1, "S": 32760, "Hq": 12, "Hk": 12,
         "D": 128, "rot": 128, "norm": True, "axes": 3, "pairs": "adjacent", "bshd": False,
         "dtype": "fp16"},
        # The next token of one request: latency counts.
        {"name": "store-1", "kind": "store", "T": 1, "Hq": 28, "Hk": 4, "D": 128, "rot": 128,
         "norm": True, "axes": 1, "pairs": "half", "page": 16, "layout": "NHD", "dtype": "bf16"},
        # One chunk of prompts in a step, heads outermost in a page.
        {"name": "store-8192", "kind": "store", "T": 8192, "Hq": 32, "Hk": 8, "D": 128,
         "rot": 128, "norm": True, "axes": 1, "pairs": "half", "page": 64, "layout": "HND",
         "dtype": "bf16"},
        # The keys and values of a short prompt, of odd length, in fp32.
        {"name": "write-613", "kind": "write", "T": 613, "Hk": 4, "D": 64, "page": 16,
         "layout": "NHD", "dtype": "fp32"},
        # Those of a 128K video prompt.
        {"name": "write-131072", "kind": "write", "T": 131072, "Hk": 4, "D": 128, "page": 16,
         "layout": "NHD", "dtype": "bf16"},
        # The next token of a chat of two thousand tokens.
        {"name": "decode-1-2081", "kind": "decode", "N": 1, "longest": 2081, "Hq": 28, "Hk": 4,
         "D": 128, "page": 16, "layout": "NHD", "dtype": "bf16"},
        # The next token after a 128K prompt: the cache's bytes count.
        {"name": "decode-1-131072", "kind": "decode", "N": 1, "longest": 131072, "Hq": 28,
         "Hk": 4, "D": 128, "page": 16, "layout": "NHD", "dtype": "bf16"},
        # A step of 64 requests whose lengths lie between a hundred and sixteen thousand tokens.
        {"name": "decode-64-16384", "kind": "decode", "N": 64, "longest": 16384, "Hq": 28,
         "Hk": 4, "D": 128, "page": 16, "layout": "NHD", "dtype": "bf16"},
        # fp32, a key head for each query head, pages of 24 tokens with the heads outermost.
        {"name": "decode-19-3001-fp32", "kind": "decode", "N": 19, "longest": 3001, "Hq": 8,
         "Hk": 8, "D": 64, "page": 24, "layout": "HND", "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "store", "write", "decode", "decode", "decode"])
    Hq, Hk = rng.choice([(28, 4), (28, 4), (32, 8), (16, 16), (12, 2), (8, 1), (40, 2)])
    D = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    page = rng.choice([16, 16, 16, 32, 64, 128, 1, 12, 24])
    layout = rng.choice(["NHD", "NHD", "HND"])
    if kind == "plan":
        N = _log(rng, 1, 2000)
        prompts = rng.choice([0, 0, rng.randint(0, min(N, 120))])
        return {"kind": "plan", "N": N, "page": page,
                "longest": _log(rng, 64, max(64, min(32768, page * (1 << 20) // N))),
                "prompts": prompts, "prompt": _log(rng, 16, 4096) if prompts else 0}
    cost = Hk * D * (4 if dtype == "fp32" else 2)  # bytes of a token's keys
    if kind == "write":
        return {"kind": "write", "T": _log(rng, 1, (1 << 27) // cost), "Hk": Hk, "D": D,
                "page": page, "layout": layout, "dtype": dtype}
    if kind == "decode":
        N = _log(rng, 1, 256)
        longest = _log(rng, 1, min(131072, (1 << 30) // (N * cost)))
        return {"kind": "decode", "N": N, "longest": longest, "Hq": Hq, "Hk": Hk, "D": D,
                "page": page, "layout": layout, "dtype": dtype}
    more = {"Hq": Hq, "Hk": Hk, "D": D, "rot": rng.choice([D, D, D, D // 2]),
            "norm": rng.random() < 0.6, "axes": rng.choice([1, 1, 3]),
            "pairs": rng.choice(["half", "half", "adjacent"]), "dtype": dtype}
    if kind == "store":
        return {"kind": "store", "T": _log(rng, 1, 8192), "page": page, "layout": layout, **more}
    B = rng.choice([1, 1, 2, 3])
    most = (24 << 15) // ((Hq + Hk) * B) // (2 if dtype == "fp32" else 1)
    return {"kind": "rope", "B": B, "S": _log(rng, 1, most), "bshd": rng.random() < 0.6, **more}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _rotation(case, g, tokens):
    """Positions, inverse frequencies, axes' sections and norm weights."""
    dev, rot, axes = _device(), case["rot"], case["axes"]
    st = {"inv_freq": (THETA ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64)
                                 / rot)).float(),
          "sections": None, "qw": None, "kw": None}
    shape = tuple(tokens) if axes == 1 else (axes, *tokens)
    start = torch.randint(0, 4096, (axes, 1, 1), generator=g, device=dev)
    if case["kind"] == "store":  # one row of each of several requests, or chunks of them
        st["positions"] = torch.randint(0, 131072, shape, generator=g, device=dev)
    else:
        at = start + torch.arange(tokens[1], device=dev) // torch.tensor(
            [1, 7, 3], device=dev)[:axes, None, None]
        st["positions"] = at.expand(axes, *tokens).contiguous().reshape(shape)
    if axes == 3:
        third = rot // 2 * 3 // 8
        st["sections"] = [rot // 2 - 2 * third, third, third]
    if case["norm"]:
        dtype = DTYPES[case["dtype"]]
        st["qw"], st["kw"] = ((1 + 0.2 * torch.randn(case["D"], generator=g, device=dev)).to(dtype)
                              for _ in range(2))
    return st


def _cache(case, g, pages):
    dev, dtype = _device(), DTYPES[case["dtype"]]
    shape = ((pages, case["page"], case["Hk"], case["D"]) if case["layout"] == "NHD"
             else (pages, case["Hk"], case["page"], case["D"]))
    return tuple(torch.randn(shape, generator=g, device=dev, dtype=dtype) for _ in range(2))


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(dev).manual_seed(seed)
    kind = case["kind"]
    st = {"case": dict(case)}
    if kind == "plan":
        N, page = case["N"], case["page"]
        host = torch.Generator().manual_seed(seed)
        lens = torch.randint(1, case["longest"] + 1, (N,), generator=host)
        new, order = torch.ones(N, dtype=torch.int64), torch.randperm(N, generator=host)
        at, out = order[:case["prompts"]], order[case["prompts"]:][:N // 16]
        lens[at] = 0  # prompts of every length up to the longest, in any order
        new[at] = torch.linspace(1, max(1, case["prompt"]), len(at)).round().long()
        new[out] = 0  # requests that sit this step out
        width = -(-(case["longest"] + case["prompt"] + 1) // page)
        held, total = -(-lens // page), -(-(lens + new) // page)
        ids = torch.randperm(int(total.sum()) + 64, generator=host).to(torch.int32)
        table = torch.full((N, width), -1, dtype=torch.int32)
        inside = torch.arange(width)[None] < held[:, None]
        table[inside] = ids[:int(held.sum())]
        st.update(lens=lens.int().to(dev), new=new.int().to(dev), table=table.to(dev),
                  free=ids[int(held.sum()):].contiguous().to(dev),
                  tokens=-(-max(1, int(new.sum())) // 64) * 64)  # padded for a captured graph
        return st
    dtype = DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    if kind == "rope":
        B, S, D = case["B"], case["S"], case["D"]
        for name, H in (("q", case["Hq"]), ("k", case["Hk"])):
            st[name] = rand(B, S, H, D).transpose(1, 2) if case["bshd"] else rand(B, H, S, D)
        st.update(_rotation(case, g, (B, S)))
        return st
    if kind in ("store", "write"):
        T, Hk, D = case["T"], case["Hk"], case["D"]
        pages = -(-T // case["page"]) + 64
        st["k"], st["v"] = rand(T, Hk, D), rand(T, Hk, D)
        st["kc"], st["vc"] = _cache(case, g, pages)
        slots = torch.randperm(pages, generator=g, device=dev)[:, None] * case["page"]
        st["slots"] = (slots + torch.arange(case["page"], device=dev)).reshape(-1)[:T].contiguous()
        if T > 8:
            st["slots"][-(T // 64 + 1):] = -1  # padding of the step
        if kind == "store":
            st["q"] = rand(T, case["Hq"], D)
            st.update(_rotation(case, g, (T,)))
        return st
    N, longest, page = case["N"], case["longest"], case["page"]
    low = math.log(min(longest, 100))
    lens = torch.exp(low + (math.log(longest) - low) * torch.rand(
        N, generator=g, device=dev, dtype=torch.float64)).round().long()
    lens[0] = longest
    if N > 8:
        lens[3] = 0  # a row of the batch without a request
    width = -(-longest // page) + 3
    held = -(-lens // page)
    pages = int(held.sum()) + 8
    ids = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(N, width, dtype=torch.int32, device=dev)
    inside = torch.arange(width, device=dev)[None] < held[:, None]
    table[inside] = ids[:int(held.sum())]
    st["q"] = rand(N, case["Hq"], case["D"])
    st["kc"], st["vc"] = _cache(case, g, pages)
    st.update(table=table, lens=lens.int())
    return st


def _rotate(x, weight, cos, sin, case):
    """x (..., D) in 32 bits: the norm, then the rotation of its first rot features."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    rot = case["rot"]
    y, rest = x[..., :rot], x[..., rot:]
    if case["pairs"] == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _angles(st):
    """(tokens..., rot/2) cosines and sines: the angles in 64 bits, each frequency's own axis."""
    at = st["positions"].double()[..., None] * st["inv_freq"].double()
    if st["sections"] is not None:
        parts = torch.split(at, st["sections"], -1)
        at = torch.cat([part[axis] for axis, part in enumerate(parts)], -1)
    return at.cos().float(), at.sin().float()


def _scatter(cache, x, slots, case):
    """x (T, Hk, D) to the cache's slots; a slot of -1 takes nothing."""
    page, keep = case["page"], slots >= 0
    x, slots = x.to(cache.dtype)[keep], slots[keep]
    if case["layout"] == "NHD":
        cache[slots // page, slots % page] = x
    else:
        cache[slots // page, :, slots % page] = x


def _plan(st):
    page, table, free = st["case"]["page"], st["table"], st["free"]
    lens, new, T = st["lens"].long(), st["new"].long(), st["tokens"]
    N, held = lens.numel(), (lens + page - 1) // page
    need = (lens + new + page - 1) // page - held
    first = need.cumsum(0) - need
    ends = new.cumsum(0)
    t = torch.arange(T, device=lens.device)
    real = t < ends[-1]
    r = torch.searchsorted(ends, t, right=True).clamp(max=N - 1)
    pos = torch.where(real, lens[r] + t - (ends - new)[r], 0)
    p = pos // page
    fresh = real & (p >= held[r])
    taken = free[(first[r] + p - held[r]).clamp(0, free.numel() - 1)]
    ids = torch.where(fresh, taken, table[r, p])
    wide = torch.cat([table, table[:1]])  # tokens without a new page write to a row of their own
    wide[torch.where(fresh, r, N), torch.where(fresh, p, 0)] = ids
    table.copy_(wide[:N])
    slots = torch.where(real, ids.long() * page + pos % page, -1)
    starts = torch.cat([ends.new_zeros(1), ends])
    return (table, (lens + new).int(), starts.int(), slots, pos,
            torch.where(real, r, -1).int(), need.sum()[None])


def _decode(st):
    case, table, lens = st["case"], st["table"].long(), st["lens"].long()
    q, (N, Hq, D), Hk = st["q"].float(), st["q"].shape, case["Hk"]
    order = (0, 3, 1, 2, 4) if case["layout"] == "NHD" else (0, 2, 1, 3, 4)
    k, v = (st[c][table].permute(*order).reshape(N, Hk, -1, D).float() for c in ("kc", "vc"))
    s = torch.matmul(k, q.view(N, Hk, Hq // Hk, D).transpose(2, 3).contiguous()) / math.sqrt(D)
    seen = (torch.arange(k.shape[2], device=q.device) < lens[:, None])[:, None, :, None]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(2, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(2, keepdim=True)
    e = e / torch.where(total == 0, 1.0, total)
    o = torch.matmul(e.transpose(2, 3).contiguous(), v)
    return o.reshape(N, Hq, D).to(st["q"].dtype)


def run(state):
    st, case = state, state["case"]
    kind = case["kind"]
    if own:
        import vecattention_amd as va
        if kind == "plan":
            return (st["table"], *va.paged_kv_plan(st["lens"], st["new"], st["table"], st["free"],
                                                   case["page"], st["tokens"]))
        if kind == "decode":
            return va.paged_decode_attention(st["q"], st["kc"], st["vc"], st["table"], st["lens"],
                                             kv_layout=case["layout"])
        if kind == "write":
            va.write_paged_kv(st["k"], st["v"], st["kc"], st["vc"], st["slots"],
                              kv_layout=case["layout"])
            return st["kc"], st["vc"]
        how = dict(q_weight=st["qw"], k_weight=st["kw"], eps=EPS, mrope_section=st["sections"],
                   interleaved=case["pairs"] == "adjacent")
        if kind == "rope":
            return va.qk_norm_rope(st["q"], st["k"], st["positions"], st["inv_freq"], **how)
        q = va.qk_norm_rope_to_cache(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["slots"],
                                     st["positions"], st["inv_freq"], kv_layout=case["layout"],
                                     **how)
        return q, st["kc"], st["vc"]
    if kind == "plan":
        return _plan(st)
    if kind == "decode":
        return _decode(st)
    if kind == "write":
        _scatter(st["kc"], st["k"], st["slots"], case)
        _scatter(st["vc"], st["v"], st["slots"], case)
        return st["kc"], st["vc"]
    heads = 1 if kind == "rope" else -2  # the axis of the heads
    cos, sin = (x.unsqueeze(heads) for x in _angles(st))
    q, k = (_rotate(st[x], st[w], cos, sin, case).to(st[x].dtype)
            for x, w in (("q", "qw"), ("k", "kw")))
    if kind == "rope":
        return q, k
    _scatter(st["kc"], k, st["slots"], case)
    _scatter(st["vc"], st["v"], st["slots"], case)
    return q, st["kc"], st["vc"]


def work(case):
    kind = case["kind"]
    if kind == "plan":
        # Lengths in, lengths and row starts out; slot, position and request of every token; every
        # new page's id in and out.  Half the prompts' and almost every other request's tokens.
        tokens = case["N"] - case["prompts"] + case["prompts"] * (case["prompt"] + 1) / 2
        pages = tokens / case["page"] + case["prompts"] / 2
        return {"bytes": 16 * case["N"] + 20 * tokens + 8 * pages, "flops": 0}
    es = 4 if case["dtype"] == "fp32" else 2
    D, Hk = case["D"], case["Hk"]
    if kind == "write":
        return {"bytes": case["T"] * (4 * Hk * D * es + 8), "flops": 0}
    if kind == "decode":
        low, high = min(case["longest"], 100), case["longest"]
        mean = (high - low) / math.log(high / low) if high > low else high
        keys = high + (case["N"] - 1) * mean
        return {"bytes": es * D * (2 * Hk * keys + 2 * case["Hq"] * case["N"]),
                "flops": 4 * D * case["Hq"] * keys}
    tokens = case["T"] if kind == "store" else case["B"] * case["S"]
    rows = tokens * (case["Hq"] + Hk)
    moved = 2 * rows * D * es + 8 * case["axes"] * tokens
    if kind == "store":
        moved += tokens * (2 * Hk * D * es + 8)
    return {"bytes": moved, "flops": rows * D * (7 if case["norm"] else 3)}


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers
    st = prepare(case, seed)
    if kind == "decode":
        rows, lens = [], st["lens"].tolist()
        for n, length in enumerate(lens):
            q = st["q"][n].double()
            if length == 0:
                rows.append(torch.zeros_like(q))
                continue
            ids = st["table"][n, :-(-length // case["page"])].long()
            k, v = st["kc"][ids].double(), st["vc"][ids].double()
            if case["layout"] == "HND":
                k, v = k.transpose(1, 2), v.transpose(1, 2)
            k, v = (x.flatten(0, 1)[:length].repeat_interleave(case["Hq"] // case["Hk"], 1)
                    for x in (k, v))
            p = ((k * q).sum(-1) * case["D"] ** -0.5).softmax(0)
            rows.append((p[..., None] * v).sum(0))
        return torch.stack(rows)

    def stored(cache, x):
        cache = cache.double()
        flat = cache if case["layout"] == "NHD" else cache.transpose(1, 2).contiguous()
        flat = flat.reshape(-1, *x.shape[1:])
        at = torch.nonzero(st["slots"] >= 0)[:, 0]
        flat.index_copy_(0, st["slots"][at], x.double()[at])
        flat = flat.reshape(-1, case["page"], *x.shape[1:])
        return flat if case["layout"] == "NHD" else flat.transpose(1, 2)

    if kind == "write":
        return stored(st["kc"], st["k"]), stored(st["vc"], st["v"])
    rot, axes = case["rot"], case["axes"]
    axis = torch.zeros(rot // 2, dtype=torch.long, device=st["k"].device)
    if axes > 1:
        axis = torch.repeat_interleave(torch.arange(axes, device=axis.device),
                                       torch.tensor(st["sections"], device=axis.device))
    at = st["positions"] if axes > 1 else st["positions"][None]
    angle = at.movedim(0, -1)[..., axis].double() * st["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        y = x[..., :rot].unflatten(-1, (2, -1) if case["pairs"] == "half" else (-1, 2))
        y = y.transpose(-1, -2) if case["pairs"] == "half" else y
        y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * turn)
        y = y.transpose(-1, -2) if case["pairs"] == "half" else y
        return torch.cat([y.flatten(-2), x[..., rot:]], -1)

    q, k = turned(st["q"], st["qw"]), turned(st["k"], st["kw"])
    if kind == "rope":
        return q, k
    return q, stored(st["kc"], k), stored(st["vc"], st["v"])

"""Workloads of the operators that let the requests of a paged key-value cache share pages.

Several answers to one prompt, the beams of a search, several questions about one long video: their
requests begin with the same tokens, and a cache in pages holds those once.  Beside the plan, the
writes and the attention of a step, a program then needs:

- ``fork``: the next step's rows from this one's: rows go on, are forked, cut back or dropped, pages
  nobody holds any more return to the free list, and a row that goes on inside a page it shares
  gets one of its own (``paged_kv_fork``).
- ``copy``: pages to other places of the caches of all layers, those of the rows above or of the
  compaction (``copy_paged_kv``).
- ``compact``: the pages in use moved to the lowest numbers (``paged_kv_compact``).
- ``prefix``: which rows begin with the same pages, and how many (``paged_kv_prefix``).
- ``attend``: attention of one new token of each request, with the keys that requests share read
  and multiplied once for all of them (``paged_prefix_decode_attention``).

Each has its plain form in elementary torch operations, which runs where ``own`` is false.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST = 2 ** 31 - 1


def listed():
    return [
        # A step of a beam search over one chat: eight beams, once for every generated token.
        {"name": "fork-8", "kind": "fork", "N": 8, "groups": 1, "longest": 2081, "tail": 100,
         "page": 16, "drop": 0.0, "trim": False},
        # A server's step: 64 prompts of up to 32768 tokens with eight answers each, some of them
        # done, some with their last tokens taken back.
        {"name": "fork-512", "kind": "fork", "N": 512, "groups": 64, "longest": 32768, "tail": 700,
         "page": 16, "drop": 0.1, "trim": True},
        # The last pages of forked beams, in part, in a few layers: latency counts.
        {"name": "copy-tails-8", "kind": "copy", "C": 8, "moves": 5, "layers": 4, "pages": 512,
         "page": 16, "Hk": 4, "D": 128, "tails": True, "layout": "NHD", "dtype": "bf16"},
        # A compaction's moves: whole pages, heads outermost, most of the list empty.
        {"name": "copy-moves-1500", "kind": "copy", "C": 4096, "moves": 1500, "layers": 4,
         "pages": 8192, "page": 16, "Hk": 8, "D": 128, "tails": False, "layout": "HND",
         "dtype": "bf16"},
        # A small cache after some requests ended.
        {"name": "compact-12", "kind": "compact", "N": 12, "groups": 5, "longest": 3001,
         "tail": 60, "page": 24, "used": 0.5},
        # That of a server with long prompts, a third in use.
        {"name": "compact-256", "kind": "compact", "N": 256, "groups": 64, "longest": 32768,
         "tail": 700, "page": 16, "used": 0.35},
        # Eight beams of one chat.
        {"name": "prefix-8", "kind": "prefix", "N": 8, "groups": 1, "longest": 2081, "tail": 100,
         "page": 16, "ids": False},
        # 64 questions about each of four videos of up to 128K tokens.
        {"name": "prefix-256", "kind": "prefix", "N": 256, "groups": 4, "longest": 131072,
         "tail": 700, "page": 16, "ids": True},
        # Four answers to a short prompt: the smallest attention, once for each layer and token.
        {"name": "attend-4-1000", "kind": "attend", "N": 4, "groups": 1, "longest": 1000,
         "tail": 40, "Hq": 28, "Hk": 4, "D": 128, "page": 16, "layout": "NHD", "dtype": "bf16"},
        # Eight beams behind an image prompt, fp16, pages of 24 tokens with the heads outermost.
        {"name": "attend-8-16000", "kind": "attend", "N": 8, "groups": 1, "longest": 16000,
         "tail": 300, "Hq": 16, "Hk": 16, "D": 64, "page": 24, "layout": "HND", "dtype": "fp16"},
        # Six prompts with up to seven answers each, of different lengths.
        {"name": "attend-40-6x8192", "kind": "attend", "N": 40, "groups": 6, "longest": 8192,
         "tail": 1024, "Hq": 32, "Hk": 8, "D": 128, "page": 64, "layout": "NHD", "dtype": "bf16"},
        # 64 questions about one video of 128K tokens: the matrix products count.
        {"name": "attend-64-131072", "kind": "attend", "N": 64, "groups": 1, "longest": 131072,
         "tail": 1024, "Hq": 28, "Hk": 4, "D": 128, "page": 16, "layout": "NHD", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["fork", "fork", "copy", "compact", "prefix", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 16, 32, 64, 128, 1, 12, 24])
    Hq, Hk = rng.choice([(28, 4), (28, 4), (32, 8), (16, 16), (12, 2), (8, 1), (40, 2)])
    D = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    layout = rng.choice(["NHD", "NHD", "HND"])
    cost = 2 * Hk * D * (4 if dtype == "fp32" else 2)  # bytes of a token's keys and values
    if kind == "copy":
        layers = rng.randint(1, 6)
        pages = _log(rng, 4, min(8192, (1 << 29) // (layers * page * cost)))
        C = rng.randint(1, max(1, pages // 2))
        return {"kind": "copy", "C": C, "moves": rng.randint(0, C), "layers": layers,
                "pages": pages, "page": page, "Hk": Hk, "D": D, "tails": rng.random() < 0.5,
                "layout": layout, "dtype": dtype}
    if kind == "attend":
        N = _log(rng, 2, 96)
        groups = rng.choice([1, 1, rng.randint(1, N)])
        own_tokens = _log(rng, 1, 1024)
        most = min(131072, (1 << 28) // (groups * cost),  # the cache, and the products
                   64 * 28 * 131072 * 128 // (N * Hq * D))
        return {"kind": "attend", "N": N, "groups": groups, "longest": _log(rng, 1, most),
                "tail": own_tokens, "Hq": Hq, "Hk": Hk, "D": D, "page": page, "layout": layout,
                "dtype": dtype}
    N = _log(rng, 2 if kind == "prefix" else 1, 512)
    groups = rng.randint(1, N // 2 if kind == "prefix" else N)
    tail = _log(rng, 1, 700)
    longest = _log(rng, 64 * page if kind == "prefix" else 1,
                   min(131072, page * (1 << 17) // groups, page * (1 << 21) // N))
    more = {"N": N, "groups": groups, "longest": longest, "tail": tail, "page": page}
    if kind == "fork":
        return {"kind": "fork", **more, "drop": rng.choice([0.0, 0.05, 0.3]),
                "trim": rng.random() < 0.3}
    if kind == "compact":
        return {"kind": "compact", **more, "used": rng.uniform(0.05, 0.95)}
    return {"kind": "prefix", **more, "ids": rng.random() < 0.5}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _first(case, dev):
    """First row of each group, and N: row n belongs to group n * groups // N."""
    at = torch.arange(case["groups"] + 1, device=dev)
    return (at * case["N"] + case["groups"] - 1) // case["groups"]


def _width(case):
    return -(-(case["longest"] + case["tail"]) // case["page"]) + 2


def _most_pages(case):
    """Pages of a pool for the longest prompts and answers."""
    N, G, page = case["N"], case["groups"], case["page"]
    return G * (case["longest"] // page) + N * (-(-case["tail"] // page) + 1)


def _tail(case):
    """Pages of a row's own keys at most: all that it has where it shares none."""
    N, G, page = case["N"], case["groups"], case["page"]
    smallest = min(N // G, N - -(-(G - 1) * N // G) - (N > 8))
    own_tokens = case["tail"] + (case["longest"] if smallest < 2 else page)
    return -(-own_tokens // page)


def _rows(case, host, spare):
    """Lengths, prompts and tables of N rows in groups, on the host.  A group's rows share the
    whole pages of its prompt and, some of them, of the answer's beginning; the pool could hold the
    longest prompts and answers, and `spare` times as many pages more."""
    N, G, page = case["N"], case["groups"], case["page"]
    group = torch.arange(N) * G // N
    low = math.log(min(case["longest"], 100))
    prompt = torch.exp(low + (math.log(case["longest"]) - low) * torch.rand(
        G, generator=host, dtype=torch.float64)).round().long().clamp(1, case["longest"])
    prompt[0] = case["longest"]
    if case["kind"] == "prefix":
        prompt[0] -= torch.randint(0, case["longest"] // 4 + 1, (1,), generator=host)[0]
    if case["kind"] == "fork":  # the beams of a prompt are all of one length
        tail = torch.randint(1, case["tail"] + 1, (G,), generator=host)[group]
    else:
        tail = torch.exp(math.log(case["tail"]) * torch.rand(
            N, generator=host, dtype=torch.float64)).round().long().clamp(1, case["tail"])
    lens = prompt[group] + tail
    common = prompt // page  # whole pages of each prompt
    held = -(-lens // page)
    width = _width(case)
    leads = torch.ones(N, dtype=torch.bool)
    leads[1:] = group[1:] != group[:-1]
    # Whole pages that a row has from the first row of its group.
    same = common[group]
    if case["kind"] in ("fork", "compact"):
        more = torch.minimum(lens // page, (lens // page)[leads][group]) - same
        same = same + (more.clamp(min=0) * torch.rand(N, generator=host)).long()
    same[leads] = 0
    cols = torch.arange(width)
    fresh = (cols < held[:, None]) & (cols >= same[:, None])
    count, pages = int(fresh.sum()), int(_most_pages(case) * (1 + spare)) + 4
    ids = torch.randperm(pages, generator=host).to(torch.int32)
    table = torch.full((N, width), -1, dtype=torch.int32)
    table[fresh] = ids[:count]
    shared = cols < same[:, None]
    table = torch.where(shared, table[leads][group], table)
    return lens, prompt, group, table, ids[count:], pages, leads


def _cache(case, g, pages):
    dev, dtype = _device(), DTYPES[case["dtype"]]
    shape = ((pages, case["page"], case["Hk"], case["D"]) if case["layout"] == "NHD"
             else (pages, case["Hk"], case["page"], case["D"]))
    return tuple(torch.randn(shape, generator=g, device=dev, dtype=dtype) for _ in range(2))


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kind, page = case["kind"], case["page"]
    st = {"case": dict(case)}
    if kind == "copy":
        C, pages = case["C"], case["pages"]
        layers = [_cache(case, g, pages) for _ in range(case["layers"])]
        order = torch.randperm(pages, generator=host).to(torch.int32)
        at = (torch.sort(torch.randperm(C, generator=host)[:case["moves"]])[0] if case["tails"]
              else torch.arange(case["moves"]))  # rows that need none lie between, or all behind
        src, dst = torch.full((2, C), -1, dtype=torch.int32)
        src[at], dst[at] = order[:case["moves"]], order[pages // 2:][:case["moves"]]
        rows = None
        if case["tails"]:
            rows = torch.zeros(C, dtype=torch.int32)
            rows[at] = torch.randint(1, page + 1, (case["moves"],), generator=host).int()
            rows = rows.to(dev)
        st.update(k=[x[0] for x in layers], v=[x[1] for x in layers], src=src.to(dev),
                  dst=dst.to(dev), rows=rows)
        return st
    spare = 1 / case["used"] - 1 if kind == "compact" else 0
    lens, prompt, group, table, free, pages, leads = _rows(case, host, spare)
    N = case["N"]
    if kind in ("fork", "compact"):
        held = torch.arange(table.shape[1]) < (-(-lens // page))[:, None]
        shares = torch.bincount(table[held].long(), minlength=pages).int() - 1
        shares = shares.clamp(min=0)
        stack = torch.full((pages,), -1, dtype=torch.int32)  # taken pages leave their entries
        stack[pages - len(free):] = free
        head = torch.tensor([pages - len(free)], dtype=torch.int32)
        st.update(lens=lens.int().to(dev), table=table.to(dev), shares=shares.to(dev),
                  free=stack.to(dev), head=head.to(dev))
        if kind == "fork":
            first = torch.nonzero(leads)[:, 0]
            size = torch.diff(first, append=torch.tensor([N]))
            # Every row goes on from a row of its group, better ones more often.
            luck = torch.rand(N, generator=host) ** 1.5
            parents = (first[group] + (luck * size[group]).long()).int()
            parents[torch.rand(N, generator=host) < case["drop"]] = -1
            keep = None
            if case["trim"]:
                keep = torch.full((N,), MOST, dtype=torch.int32)
                back = torch.rand(N, generator=host) < 0.2
                cut = torch.randint(1, 9, (N,), generator=host)
                keep[back] = (lens - cut).clamp(min=0).int()[back]
                keep = keep.to(dev)
            st.update(parents=parents.to(dev), keep=keep)
        return st
    if N > 8:
        lens[-1] = 0  # a row of the batch without a request
    st.update(lens=lens.int().to(dev), table=table.to(dev))
    if kind == "prefix":
        st["ids"] = group.int().to(dev) if case["ids"] else None
        return st
    # The plan of the step, which every layer's attention is given.
    present = lens > 0
    size = torch.bincount(group[present], minlength=case["groups"])
    both = (size > 1)[group] & present
    shared = torch.where(both, (prompt // page * page)[group], 0)
    st["prefix"] = shared.int().to(dev)
    st["group_rows"] = torch.where(leads & (shared > 0), size[group], 0).int().to(dev)
    st["q"] = torch.randn((N, case["Hq"], case["D"]), generator=g, device=dev,
                          dtype=DTYPES[case["dtype"]])
    st["kc"], st["vc"] = _cache(case, g, pages)
    return st


def _fork(st):
    page, table, lens = st["case"]["page"], st["table"], st["lens"].long()
    free, parents = st["free"], st["parents"].long()
    (N, M), P, F, R = table.shape, st["shares"].numel(), free.numel(), parents.numel()
    dev = table.device
    cols, rows = torch.arange(M, device=dev), torch.arange(R, device=dev)
    named = (parents >= 0) & (parents < N)
    a = parents.clamp(0, N - 1)
    new_lens = torch.where(named, lens[a], 0)
    if st["keep"] is not None:
        new_lens = torch.minimum(new_lens, st["keep"].long())
    held = torch.clamp((lens + page - 1) // page, max=M)
    new_held = torch.clamp((new_lens + page - 1) // page, max=M)
    new = table[a]
    # Rows that hold each page, less one.
    count = st["shares"].long()
    count = count + torch.bincount(new[cols < new_held[:, None]], minlength=P)
    count = count - torch.bincount(table[cols < held[:, None]], minlength=P)
    # Rows whose next token goes into a page that holds some of theirs already.
    last = torch.where((new_lens % page != 0) & (new_held > 0), new_held - 1, 0)
    ends = torch.where(new_lens % page != 0, new.gather(1, last[:, None])[:, 0].long(), P)
    writers = torch.zeros(P + 1, dtype=torch.long, device=dev)
    writers.index_add_(0, ends, torch.ones_like(ends))
    least = torch.full((P + 1,), R, dtype=torch.long, device=dev)
    least.scatter_reduce_(0, ends, rows, "amin")
    at = ends.clamp(max=P - 1)
    copies = (ends < P) & ((least[ends] != rows) | (count[at] + 1 > writers[ends]))
    # Freed pages lie on top of the free ones; copies take from the top.
    gone = count < 0
    freed, taken = gone.long().cumsum(0), copies.long().cumsum(0)
    nf, nt = freed[-1], taken[-1]
    head = st["head"].long().clamp(0, F)
    stack = torch.cat([free.new_zeros(P), free, free.new_full((R,), -1)])
    top = P + head - nf
    spot = torch.where(gone, top + freed - 1, P + F + R - 1)
    stack.scatter_(0, spot, torch.where(gone, torch.arange(P, device=dev), -1).int())
    given = stack[torch.where(copies, top + taken - 1, 0)]
    kept = torch.arange(F, device=dev) + P
    new_free = torch.where((kept >= top + nt) & (kept < P + head), stack[P:P + F], free)
    new_shares = count.clone()
    new_shares.index_add_(0, at, -copies.long())
    new_shares = torch.where(gone, 0, new_shares.clamp(min=0))
    out = torch.where(cols < new_held[:, None], new, -1)
    out = torch.where(copies[:, None] & (cols == last[:, None]), given[:, None], out)
    return (new_lens.int(), out, new_shares.int(), new_free,
            torch.clamp(head - nf + nt, min=0).int(),
            torch.where(copies, ends, -1).int(), torch.where(copies, given, -1),
            torch.where(copies, new_lens % page, 0).int())


def _compact(st):
    page, table, lens, free = st["case"]["page"], st["table"], st["lens"].long(), st["free"]
    M, P, F = table.shape[1], st["shares"].numel(), free.numel()
    dev = table.device
    held = torch.clamp((lens + page - 1) // page, max=M)
    inside = torch.arange(M, device=dev) < held[:, None]
    used = torch.zeros(P + 1, dtype=torch.bool, device=dev)
    used[torch.where(inside, table.long(), P).reshape(-1)] = True
    used = used[:P]
    open_ = torch.zeros(P + 1, dtype=torch.bool, device=dev)
    open_[torch.where(torch.arange(F, device=dev) >= st["head"], free.long(), P)] = True
    open_ = open_[:P] & ~used
    rank = (used | open_).long().cumsum(0) - 1
    total = used.long().sum()
    moves, holes = used & (rank >= total), open_ & (rank < total)
    k, h = moves.long().cumsum(0) - 1, holes.long().cumsum(0) - 1
    ids = torch.arange(P, device=dev)
    half = P // 2
    src = torch.full((half + 1,), -1, dtype=torch.long, device=dev)
    dst = src.clone()
    src[torch.where(moves, k, half)] = torch.where(moves, ids, -1)
    dst[torch.where(holes, h, half)] = torch.where(holes, ids, -1)
    place = torch.where(moves, dst[k.clamp(min=0)], ids)
    out = torch.where(inside & (table >= 0), place[table.clamp(min=0).long()].int(), table)
    shares = torch.cat([torch.where(moves, 0, st["shares"]), free.new_zeros(1)])
    shares.scatter_(0, torch.where(moves, place, P), torch.where(moves, st["shares"], 0))
    behind = (used | open_) & (rank >= total)
    left = behind.long().sum()
    new_free = torch.cat([free, free.new_zeros(1)])
    new_free[torch.where(behind, F - left + rank - total, F)] = ids.int()
    return (out, shares[:P], new_free[:F], (F - left).int()[None], src[:half].int(),
            dst[:half].int(), moves.long().sum().int()[None])


def _copy_rows(caches, st):
    """Rows of whole pages, or the first of them, from page to page of each cache."""
    page, nhd = st["case"]["page"], st["case"]["layout"] == "NHD"
    keep = st["src"] >= 0
    src, dst = st["src"][keep].long(), st["dst"][keep].long()
    if st["rows"] is None:
        return [c.index_copy_(0, dst, c[src]) for c in caches]
    take = torch.arange(page, device=src.device) < st["rows"][keep][:, None]
    take = take[:, :, None, None] if nhd else take[:, None, :, None]
    return [c.index_copy_(0, dst, torch.where(take, c[src], c[dst])) for c in caches]


def _prefix(st):
    page, table, lens = st["case"]["page"], st["table"], st["lens"].long()
    N, M = table.shape
    dev = table.device
    here = lens > 0
    ids = table[:, 0] if st["ids"] is None else st["ids"]
    joins = torch.zeros(N, dtype=torch.bool, device=dev)
    joins[1:] = (ids[1:] == ids[:-1]) & here[1:] & here[:-1]
    if st["ids"] is None:
        joins &= ids >= 0
    first = torch.where(joins, 0, torch.arange(N, device=dev)).cummax(0)[0]
    whole = torch.clamp(lens // page, 0, M)
    same = (table == table[first]) & (table >= 0) & (torch.arange(M, device=dev) < whole[:, None])
    pages = same.long().cumprod(1).sum(1)
    least = torch.full((N,), M, dtype=torch.long, device=dev)
    least = least.scatter_reduce(0, first, pages, "amin")
    size = torch.zeros(N, dtype=torch.long, device=dev).index_add(0, first, torch.ones_like(first))
    shared = torch.where(size[first] > 1, least[first] * page, 0)
    return shared.int(), torch.where(~joins & (shared > 0), size, 0).int()


def _attend(st):
    case, table, lens = st["case"], st["table"].long(), st["lens"].long()
    q, (N, Hq, D), Hk, page = st["q"].float(), st["q"].shape, case["Hk"], case["page"]
    rep, dev = Hq // Hk, q.device
    order = (0, 3, 1, 2, 4) if case["layout"] == "NHD" else (0, 2, 1, 3, 4)

    def rows_of(cache, ids):
        return cache[ids.clamp(min=0)].permute(*order).reshape(ids.shape[0], Hk, -1, D).float()

    # The prompts' keys once for a group, all rows of the group behind one another.
    first = _first(case, dev)[:-1]
    group = torch.arange(N, device=dev) * case["groups"] // N
    place = torch.arange(N, device=dev) - first[group]
    G, B, wide = case["groups"], -(-N // case["groups"]), max(1, case["longest"] // page)
    least = st["prefix"].long()
    qg = q.new_zeros(G, B, Hk, rep, D)
    qg[group, place] = q.view(N, Hk, rep, D) / math.sqrt(D)
    qg = qg.permute(0, 2, 1, 3, 4).reshape(G, Hk, B * rep, D)
    s = torch.matmul(qg, rows_of(st["kc"], table[first, :wide]).transpose(2, 3).contiguous())
    seen = least.new_zeros(G, B)
    seen[group, place] = least
    mask = torch.arange(wide * page, device=dev) < seen[:, :, None]
    s = torch.where(mask[:, None, :, None], s.view(G, Hk, B, rep, -1), -math.inf)
    # Their own keys.
    cols = (least // page)[:, None] + torch.arange(_tail(case), device=dev)
    ids = table.gather(1, cols.clamp(max=table.shape[1] - 1))
    t = torch.matmul(q.view(N, Hk, rep, D) / math.sqrt(D),
                     rows_of(st["kc"], ids).transpose(2, 3).contiguous())
    own_at = torch.arange(t.shape[-1], device=dev)
    t = torch.where((own_at < (lens - least)[:, None])[:, None, None], t, -math.inf)
    top = torch.maximum(t.amax(-1, keepdim=True), s[group, :, place].amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    high = q.new_zeros(G, B, Hk, rep, 1)
    high[group, place] = top
    t, e = torch.exp(t - top), torch.exp(s - high.permute(0, 2, 1, 3, 4))
    total = t.sum(-1, keepdim=True) + e.sum(-1, keepdim=True)[group, :, place]
    e = torch.matmul(e.view(G, Hk, B * rep, -1), rows_of(st["vc"], table[first, :wide]))
    o = torch.matmul(t, rows_of(st["vc"], ids)) + e.view(G, Hk, B, rep, D)[group, :, place]
    o = o / torch.where(total == 0, 1.0, total)
    return o.reshape(N, Hq, D).to(st["q"].dtype)


def run(state):
    st, case = state, state["case"]
    kind, page = case["kind"], case["page"]
    if own:
        import vecattention_amd as va
        if kind == "fork":
            f = va.paged_kv_fork(st["lens"], st["parents"], st["table"], st["shares"], st["free"],
                                 page, free_head=st["head"], keep_lens=st["keep"])
            return (f.kv_lens, f.block_tables, f.page_shares, f.free_pages, f.free_head,
                    f.copy_src, f.copy_dst, f.copy_rows)
        if kind == "compact":
            c = va.paged_kv_compact(st["lens"], st["table"], st["shares"], st["free"], page,
                                    free_head=st["head"])
            return (c.block_tables, c.page_shares, c.free_pages, c.free_head, c.copy_src,
                    c.copy_dst, c.num_moves)
        if kind == "copy":
            va.copy_paged_kv(st["k"], st["v"], st["src"], st["dst"], rows=st["rows"],
                             kv_layout=case["layout"])
            return st["k"], st["v"]
        if kind == "prefix":
            return tuple(va.paged_kv_prefix(st["lens"], st["table"], page, group_ids=st["ids"]))
        return va.paged_prefix_decode_attention(
            st["q"], st["kc"], st["vc"], st["table"], st["lens"], (st["prefix"], st["group_rows"]),
            kv_layout=case["layout"])
    if kind == "fork":
        return _fork(st)
    if kind == "compact":
        return _compact(st)
    if kind == "copy":
        return _copy_rows(st["k"], st), _copy_rows(st["v"], st)
    return _prefix(st) if kind == "prefix" else _attend(st)


def _mean(low, high):
    """Of a value spread evenly over its logarithm."""
    return (high - low) / math.log(high / low) if high > low else high


def work(case):
    page = case["page"]
    if case["kind"] == "copy":
        es = 4 if case["dtype"] == "fp32" else 2
        tokens = case["moves"] * ((page + 1) / 2 if case["tails"] else page)
        return {"bytes": 4 * tokens * case["layers"] * case["Hk"] * case["D"] * es + 8 * case["C"],
                "flops": 0}
    N, G = case["N"], case["groups"]
    prompts = case["longest"] + (G - 1) * _mean(min(case["longest"], 100), case["longest"])
    if case["kind"] == "attend":
        es, D, Hq, Hk = 4 if case["dtype"] == "fp32" else 2, case["D"], case["Hq"], case["Hk"]
        tails = N * _mean(1, case["tail"])
        return {"bytes": es * D * (2 * Hk * (prompts + tails) + 2 * Hq * N),
                "flops": 4 * D * Hq * (prompts / G * N + tails)}
    entries = N * (prompts / G + case["tail"] / 2) / page  # of tables that are in use
    if case["kind"] == "prefix":
        return {"bytes": 4 * N * prompts / G / page + 16 * N, "flops": 0}
    pages = _most_pages(case) / (case["used"] if case["kind"] == "compact" else 1)
    return {"bytes": 4 * entries + 4 * N * _width(case) + 16 * pages + 32 * N, "flops": 0}


def exact(case, seed):
    kind = case["kind"]
    if kind not in ("copy", "attend"):
        return None  # whole numbers
    st = prepare(case, seed)
    page, nhd = case["page"], case["layout"] == "NHD"
    if kind == "copy":
        src, dst = st["src"].tolist(), st["dst"].tolist()
        count = [page] * len(src) if st["rows"] is None else st["rows"].tolist()

        def moved(cache):
            flat = cache.double() if nhd else cache.double().transpose(1, 2).contiguous()
            before = flat.clone()
            at = [(s, d, n) for s, d, n in zip(src, dst, count) if s >= 0]
            if at:
                move = torch.tensor(at, device=flat.device)
                for n in sorted({n for _, _, n in at}):
                    these = move[move[:, 2] == n]
                    flat[these[:, 1], :n] = before[these[:, 0], :n]
            return flat if nhd else flat.transpose(1, 2)

        return [moved(c) for c in st["k"]], [moved(c) for c in st["v"]]
    Hq, Hk = case["Hq"], case["Hk"]
    outs = []
    for n, length in enumerate(st["lens"].tolist()):
        q = st["q"][n].double().unflatten(0, (Hk, Hq // Hk))
        if length == 0:
            outs.append(torch.zeros_like(q).flatten(0, 1))
            continue
        ids = st["table"][n, :-(-length // page)].long()
        k, v = (c[ids].double() if nhd else c[ids].double().transpose(1, 2)
                for c in (st["kc"], st["vc"]))
        k, v = (x.flatten(0, 1)[:length].transpose(0, 1).contiguous() for x in (k, v))
        p = torch.softmax(torch.matmul(k, q.transpose(1, 2).contiguous()) * case["D"] ** -0.5, 1)
        outs.append(torch.matmul(p.transpose(1, 2).contiguous(), v).flatten(0, 1))
    return torch.stack(outs)

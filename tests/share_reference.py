"""Plain forms of the operators on pages that rows share, entry by entry."""


def pages_of(length, page, width):
    return min(-(-max(length, 0) // page), width)


def fork(lens, parents, table, shares, free, page, head=0, keep=None):
    """(lens, table, shares, free, head, src, dst, rows)."""
    N, width, P, F = len(lens), len(table[0]) if table else 0, len(shares), len(free)
    count = list(shares)
    for n in range(N):
        for p in table[n][:pages_of(lens[n], page, width)]:
            if 0 <= p < P:
                count[p] -= 1
    out_lens, out, ends = [], [], []
    for r, a in enumerate(parents):
        length = max(lens[a], 0) if 0 <= a < N else 0
        if keep is not None:
            length = min(length, max(keep[r], 0))
        held = pages_of(length, page, width)
        row = (table[a][:held] if held else []) + [-1] * (width - held)
        for p in row[:held]:
            if 0 <= p < P:
                count[p] += 1
        at = length // page
        open_ = length % page and at < width and 0 <= row[at] < P
        ends.append(row[at] if open_ else None)
        out_lens.append(length)
        out.append(row)
    freed = [p for p in range(P) if count[p] < 0]
    count = [max(c, 0) for c in count]
    head = min(max(head, 0), F)
    src, dst, rows = [-1] * len(parents), [-1] * len(parents), [0] * len(parents)
    copies = []
    for r, p in enumerate(ends):
        if p is not None:
            writers = [i for i, e in enumerate(ends) if e == p]
            if r != writers[0] or count[p] + 1 > len(writers):
                copies.append(r)
    given = (freed + list(free[head:]) + [-1] * len(copies))[:len(copies)]
    for r, new in zip(copies, given):
        at = out_lens[r] // page
        src[r], dst[r], rows[r] = ends[r], new, out_lens[r] % page
        out[r][at] = new
    left = list(free)
    top = head - len(freed)
    for j, p in enumerate(freed):
        if j >= len(copies) and top + j >= 0:
            left[top + j] = p
    for p in {src[r] for r in copies}:
        count[p] = max(count[p] - src.count(p), 0)
    return out_lens, out, count, left, max(top + len(copies), 0), src, dst, rows


def compact(lens, table, shares, free, page, head=0):
    """(table, shares, free, head, src, dst, moves)."""
    P, F, width = len(shares), len(free), len(table[0]) if table else 0
    used = {p for n, row in enumerate(table) for p in row[:pages_of(lens[n], page, width)]
            if 0 <= p < P}
    open_ = {p for p in free[min(max(head, 0), F):] if 0 <= p < P} - used
    both = sorted(used | open_)
    low = both[:len(used)]
    movers, holes = sorted(used - set(low)), sorted(set(low) - used)
    to = dict(zip(movers, holes))
    out = [[to.get(p, p) if k < pages_of(lens[n], page, width) else p for k, p in enumerate(row)]
           for n, row in enumerate(table)]
    count = list(shares)
    for a, b in to.items():
        count[b] = shares[a]
    for a in to:
        count[a] = 0
    behind = both[len(used):]
    left = list(free)
    left[F - len(behind):] = behind
    pad = [-1] * (P // 2 - len(to))
    return out, count, left, F - len(behind), movers + pad, holes + pad, len(to)


def prefix(lens, table, page, ids=None):
    """(prefix_lens, group_rows)."""
    N = len(lens)
    shared, sizes, n = [0] * N, [0] * N, 0
    while n < N:
        end = n + 1

        def alike(i):
            if lens[i] <= 0 or lens[i - 1] <= 0:
                return False
            if ids is not None:
                return ids[i] == ids[i - 1]
            return bool(table[i]) and table[i][0] >= 0 and table[i][0] == table[i - 1][0]
        while end < N and alike(end):
            end += 1
        common = 0
        if end - n > 1:
            most = min(min(lens[n:end]) // page, len(table[n]))
            while common < most and table[n][common] >= 0 and all(
                    table[i][common] == table[n][common] for i in range(n, end)):
                common += 1
        for i in range(n, end):
            shared[i] = common * page
        if common:
            sizes[n] = end - n
        n = end
    return shared, sizes

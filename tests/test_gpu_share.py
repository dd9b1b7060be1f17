"""The operators on pages that rows share against their plain forms
(tests/share_reference.py, tests/paged_reference.py), on an MI355X."""
import random

import pytest
import torch

import share_reference as ref
from vecattention_amd import copy_paged_kv, paged_kv_compact, paged_kv_fork, paged_kv_prefix

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def note(*a):
    print("[case]", *a, flush=True)


def ints(x, dev=DEV):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def table_of(table):
    return ints(table).reshape(len(table), len(table[0]) if table else 0)


def check(got, want):
    torch.cuda.synchronize()
    for name, a, b in zip(got._fields, got, want):
        assert a.dtype == torch.int32 and a.is_cuda
        b = [b] if isinstance(b, int) else b
        assert a.flatten().tolist() == [
            y for x in b for y in (x if isinstance(x, list) else [x])], name


def random_state(r, N, page, width, P, share=0.5):
    """Rows as steps of forks and plans leave them: (lens, table, shares, free, head)."""
    ids = list(range(P))
    r.shuffle(ids)
    lens, table, taken = [], [], 0
    for n in range(N):
        length = r.choice([0, 1, page, r.randint(0, page * width), r.randint(0, page * width)])
        held = ref.pages_of(length, page, width)
        row = []
        if table and r.random() < share:
            other = r.randrange(n)
            whole = min(lens[other] // page, length // page, width)
            row = table[other][:r.randint(0, whole)]
        need = held - len(row)
        need = min(need, P - taken)
        row = row + ids[taken:taken + need]
        taken += need
        row += [-1] * (width - len(row))
        lens.append(length)
        table.append(row)
    shares = [0] * P
    for n in range(N):
        for p in table[n][:ref.pages_of(lens[n], page, width)]:
            if p >= 0:
                shares[p] += 1
    shares = [max(s - 1, 0) for s in shares]
    free = [-1] * taken + ids[taken:]
    return lens, table, shares, free, taken


def fork_case(lens, parents, table, shares, free, page, head=None, keep=None):
    note("fork", len(lens), "to", len(parents), "rows, page", page, "of", len(shares), "pages")
    want = ref.fork(lens, parents, table, shares, free, page, head or 0, keep)
    given = [ints(lens), ints(parents), table_of(table), ints(shares),
             ints(free)]
    before = [t.clone() for t in given]
    got = paged_kv_fork(*given, page, None if head is None else ints([head]),
                        None if keep is None else ints(keep))
    check(got, want)
    assert got.block_tables.shape == (len(parents), given[2].shape[1])
    assert all(torch.equal(a, b) for a, b in zip(given, before))
    return got


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("N,R,width,P", [
    (1, 1, 3, 8), (4, 7, 9, 60), (9, 4, 5, 30), (64, 64, 12, 900), (300, 500, 7, 5000),
    (12, 30, 1500, 20000), (600, 70, 3, 9000)])
def test_fork_matches_the_plain_form(N, R, width, P, page):
    r = random.Random(N * 1000 + page)
    for trial in range(3):
        state = random_state(r, N, page, width, P)
        lens, table, shares, free, head = state
        parents = [r.choice([-1, r.randrange(N), r.randrange(N), r.randrange(min(N, 3))])
                   for _ in range(R)]
        keep = None
        if trial:
            keep = [r.choice([0, 2 ** 31 - 1, r.randint(0, page * width)]) for _ in range(R)]
        fork_case(lens, parents, table, shares, free, page, head, keep)


def test_fork_edges():
    fork_case([5], [], [[1, 2]], [0] * 4, [0, 3], 4, 0)                     # all rows dropped
    fork_case([], [-1, 0], [], [0] * 4, [0, 3], 4)                          # none to begin with
    fork_case([5], [0], [[1, 2]], [0] * 4, [], 4)  # nothing free, nothing needed
    fork_case([5], [0, 0, 0], [[1, 2]], [0] * 4, [0], 4)                    # the list ends
    fork_case([5], [0, 0, 0], [[1, 2]], [0] * 4, [0, 3], 4, 9)              # a head past the list
    fork_case([5], [0, 0, 0], [[1, 2]], [0] * 4, [0, 3], 4, -7)
    fork_case([5, 6], [0, 0, 0], [[1, 2], [0, 3]], [0] * 4, [], 4)  # freed pages go to the copies
    fork_case([5, 6], [-1, -5, 2, 99], [[1, 2], [0, 3]], [0] * 4, [7, 7, 7], 4, 2)  # no room
    fork_case([-3, 9], [0, 1, 1], [[1, 2], [0, 3]], [0] * 4, [2], 4)  # negative, and past the table
    fork_case([9, 9], [0, 1, 0], [[1, -1, 70], [-4, 3, 0]], [0] * 4, [2], 4)  # no pages
    fork_case([6, 7], [0, 1], [[3, 5], [3, 6]], [0, 0, 0, 1, 0, 0, 0], [9, 4], 4, 1, [2, 3])
    fork_case([6, 7], [1, 0], [[3, 5], [3, 6]], [0, 0, 0, 4, 0, 0, 0], [9, 4], 4, 1, [2, 3])
    fork_case([4, 4], [0, 1], [[3], [3]], [0, 0, 0, 1], [0, 1], 4, 0, [4, 2])
    fork_case([4, 4], [0, 1], [[3], [3]], [0, 0, 0, 1], [0, 1], 4, 0, [-1, 2])
    fork_case([2 ** 31 - 1], [0, 0], [[1, 2]], [0] * 4, [0, 3], 1 << 30, 0)
    fork_case([2 ** 31 - 1], [0, 0], [[1, 2]], [0] * 4, [0, 3], 2 ** 31 - 1, 0)
    fork_case([3], [0, 0], [[]], [0] * 4, [0, 3], 4, 0)                     # tables of no width
    fork_case([3], [0, 0], [[1]], [], [0, 3], 4, 0)                         # a cache of no pages


def test_fork_wide_tables_and_many_pages():
    r = random.Random(8)
    for P in (4096, 4097, 70001):
        lens, table, shares, free, head = random_state(r, 6, 2, 3000, P, 0.9)
        fork_case(lens, [0, 0, 3, -1, 5], table, shares, free, 2, head)


def test_fork_strided_arguments_and_devices():
    r = random.Random(2)
    lens, table, shares, free, head = random_state(r, 7, 4, 9, 80)
    parents = [3, 3, 0, 6, 6, 6]
    want = ref.fork(lens, parents, table, shares, free, 4, head)
    wide = torch.full((7, 20), 77, dtype=torch.int32, device=DEV)
    wide[:, :9] = ints(table)
    every = [torch.stack([ints(x), ints(x) + 1], 1)[:, 0] for x in (lens, parents, shares, free)]
    got = paged_kv_fork(every[0], every[1], wide[:, :9], every[2], every[3], 4, ints([head]))
    check(got, want)
    got = paged_kv_fork(every[0], every[1], ints(table).t().contiguous().t(), every[2], every[3], 4,
                        ints([[head]]))
    check(got, want)
    with pytest.raises(ValueError, match="tensors on"):
        paged_kv_fork(ints(lens), ints(parents, "cpu"), ints(table), ints(shares), ints(free), 4)


def compact_case(lens, table, shares, free, page, head=None):
    note("compact", len(lens), "rows, page", page, "of", len(shares), "pages")
    want = ref.compact(lens, table, shares, free, page, head or 0)
    given = [ints(lens), table_of(table), ints(shares), ints(free)]
    before = [t.clone() for t in given]
    got = paged_kv_compact(*given, page, None if head is None else ints([head]))
    check(got, want)
    assert all(torch.equal(a, b) for a, b in zip(given, before))


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("N,width,P", [(1, 3, 8), (9, 5, 33), (64, 12, 900), (40, 1500, 70001),
                                       (300, 7, 4096)])
def test_compact_matches_the_plain_form(N, width, P, page):
    r = random.Random(N * 1000 + page)
    for trial in range(3):
        lens, table, shares, free, head = random_state(r, N, page, width, P)
        if trial == 2:  # some pages belong to somebody else
            free = [p if p < 0 or r.random() < 0.5 else -1 for p in free]
        compact_case(lens, table, shares, free, page, head)


def test_compact_edges():
    compact_case([], [], [0] * 5, [4, 2], 4)
    compact_case([0, 0], [[1], [2]], [0] * 5, [4, 2], 4)                 # no page in use
    compact_case([4], [[4]], [0] * 5, [], 4)                             # none free
    compact_case([4], [[4]], [0] * 5, [3, 3, 3, 0, 0], 4)                # the same page twice
    compact_case([4], [[4]], [0] * 5, [4, 1, -1, 9], 4)                  # free and in use: in use
    compact_case([8, 4], [[-1, 4], [9, 3]], [0, 0, 0, 0, 7], [0, 1], 4, 1)
    compact_case([8, 4], [[2, 4], [1, 3]], [0] * 5, [0], 4, 77)          # a head past the list
    compact_case([8, 4], [[2, 4], [1, 3]], [0] * 5, [0], 4, -2)
    compact_case([3], [[0]], [0], [], 4)
    compact_case([3], [[0]], [], [1], 4)                                 # a cache of no pages
    compact_case([3], [[]], [0] * 3, [1], 4)
    compact_case([128], [list(range(64, 128))], [0] * 128, list(range(64)), 2)
    compact_case([128], [list(range(127, 63, -1))], [0] * 128, list(range(63, -1, -1)), 2)


def prefix_case(lens, table, page, ids=None):
    note("prefix", len(lens), "rows, page", page)
    got = paged_kv_prefix(ints(lens), table_of(table), page,
                          None if ids is None else ints(ids))
    check(got, ref.prefix(lens, table, page, ids))


@pytest.mark.parametrize("N,width,page", [(1, 4, 4), (2, 5, 1), (9, 9, 4), (70, 3, 16),
                                          (300, 40, 2), (24, 3000, 1), (1000, 2, 3)])
def test_prefix_matches_the_plain_form(N, width, page):
    r = random.Random(N + width)
    for trial in range(4):
        base = [[r.randint(0, 9999) for _ in range(width)] for _ in range(3)]
        lens, table, ids, at = [], [], [], 0
        for n in range(N):
            if r.random() < 0.2:
                at = r.randrange(3)
            row = list(base[at])
            cut = r.choice([width, width, r.randint(0, width), max(width - r.randint(0, 3), 0)])
            row[cut:] = [r.choice([-1, r.randint(0, 9999)]) for _ in range(width - cut)]
            table.append(row)
            lens.append(r.choice([0, -1, r.randint(1, width * page), width * page, width * page + 9,
                                  width * page]) if r.random() < 0.3 else width * page)
            ids.append(r.choice([at, at, at, -1]))
        prefix_case(lens, table, page, ids if trial % 2 else None)


def test_prefix_edges():
    prefix_case([], [], 4)
    prefix_case([4, 4], [[], []], 4)                       # tables of no width
    prefix_case([4, 4], [[], []], 4, [1, 1])
    prefix_case([8, 8], [[5, 6], [5, 6]], 4)               # the whole of both
    prefix_case([3, 3], [[5, 6], [5, 6]], 4)               # no whole page
    prefix_case([8, 8], [[-1, 6], [-1, 6]], 4, [0, 0])     # no page
    prefix_case([8, 8, 8], [[5, 6], [5, 7], [5, 6]], 4)
    prefix_case([2 ** 31 - 1] * 2, [[5, 6], [5, 6]], 2 ** 30)
    prefix_case([8] * 200, [[5, 6]] * 200, 4)
    prefix_case([8] * 130, [[n // 65, 6] for n in range(130)], 4)
    note("prefix empty")
    assert paged_kv_prefix(ints([]), ints([]).reshape(0, 4), 4).prefix_lens.numel() == 0


# ---------------------------------------------------------------- copies

def copy_case(layers, P, page, Hk, D, layout, dtype, C, seed, rows=True, view=None):
    note("copy", layers, P, page, Hk, D, layout, dtype, C)
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    shape = (P, page, Hk, D) if layout == "NHD" else (P, Hk, page, D)
    view = view or (lambda t: t)
    caches = [[torch.randn(shape, generator=g).to(dtype) for _ in range(layers)] for _ in range(2)]
    order = list(range(P))
    r.shuffle(order)
    src, dst = order[:P // 2], order[P // 2:]
    src, dst = [r.choice(src) for _ in range(C)], (dst + [-1] * C)[:C]  # a page may be copied twice
    for i in range(C):
        if r.random() < 0.3:
            src[i], dst[i] = r.choice([(-1, dst[i]), (src[i], -1), (P, dst[i]), (src[i], P + 7),
                                       (src[i], src[i]), (2 ** 31 - 1, -2 ** 31)])
    count = [r.choice([0, page, -2, page + 5, r.randint(0, page)]) for _ in range(C)]
    want = [[t.clone() for t in kind] for kind in caches]
    for kind, old in zip(want, caches):
        for new, t in zip(kind, old):
            for s, d, n in zip(src, dst, count):
                n = max(min(n, page), 0) if rows else page
                if 0 <= s < P and 0 <= d < P:
                    if layout == "NHD":
                        new[d, :n] = t[s, :n]
                    else:
                        new[d, :, :n] = t[s, :, :n]
    dev = [[view(t.to(DEV)) for t in kind] for kind in caches]
    versions = [t._version for kind in dev for t in kind]
    copy_paged_kv(dev[0] if layers > 1 else dev[0][0], tuple(dev[1]) if layers > 1 else dev[1][0],
                  ints(src), ints(dst), ints(count) if rows else None, kv_layout=layout)
    torch.cuda.synchronize()
    for kind, old in zip(dev, want):
        for t, w in zip(kind, old):
            assert torch.equal(t.cpu(), w)
    assert all(t._version > v for t, v in zip((t for kind in dev for t in kind), versions))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layers,P,page,Hk,D,layout,C", [
    (1, 2, 1, 1, 64, "NHD", 1), (3, 40, 16, 4, 128, "NHD", 20), (2, 30, 24, 3, 64, "HND", 15),
    (33, 9, 5, 2, 72, "NHD", 4), (2, 12, 300, 2, 128, "HND", 6), (1, 20, 16, 4, 7, "NHD", 9),
    (2, 700, 1, 1, 20, "HND", 350), (70, 4, 2, 1, 8, "NHD", 2)])
@pytest.mark.parametrize("rows", [True, False])
def test_copy_matches_the_plain_form(layers, P, page, Hk, D, layout, C, rows, dtype):
    copy_case(layers, P, page, Hk, D, layout, dtype, C, P + page, rows)


def test_copy_of_views():
    def padded(t):  # rows of a wider cache, 16-byte aligned
        wide = torch.zeros(*t.shape[:3], 2 * t.shape[3], dtype=t.dtype, device=t.device)
        wide[..., :t.shape[3]] = t
        return wide[..., :t.shape[3]]

    def odd(t):     # rows that start at any element
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def turned(t):  # pages innermost but for the features
        return t.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)

    for view in (padded, odd, turned):
        for layout in ("NHD", "HND"):
            copy_case(2, 24, 12, 3, 64, layout, BF16, 12, 4, True, view)
    # The neighbours of the rows stay.
    note("copy neighbours")
    wide = torch.arange(6 * 4 * 2 * 16, device=DEV).view(6, 4, 2, 16).float()
    old = wide.clone()
    copy_paged_kv(wide[..., 4:12], wide[..., 4:12], ints([1]), ints([5]), ints([3]))
    old[5, :3, :, 4:12] = old[1, :3, :, 4:12]
    assert torch.equal(wide, old)


def test_copy_nothing():
    note("copy nothing")
    k = torch.ones(3, 4, 2, 8, device=DEV)
    copy_paged_kv(k, k, ints([]), ints([]))
    copy_paged_kv(k[:, :, :0], k[:, :, :0], ints([0]), ints([1]))
    assert bool((k == 1).all())


def test_copy_refusals_on_the_gpu():
    k = torch.ones(3, 4, 2, 8, device=DEV)
    with pytest.raises(ValueError, match="tensors on"):
        copy_paged_kv(k, k, ints([0]), ints([1], "cpu"))
    with pytest.raises(ValueError, match="tensors on"):
        copy_paged_kv([k, k.cpu()], [k, k], ints([0]), ints([1]))
    with pytest.raises(NotImplementedError, match="no backward"):
        copy_paged_kv([k, k], [k, k.clone().requires_grad_()], ints([0]), ints([1]))


def test_copy_offsets_past_32_bits():
    note("copy far")
    P, page = 70000, 16
    k = torch.zeros(P, page, 4, 128, dtype=BF16, device=DEV)  # 1.1 GB, 2^29 elements
    k[7] = 3
    v = torch.zeros(P * 5, page, 4, 128, dtype=BF16, device=DEV)[::5]  # 2^31 elements apart
    v[P - 2] = 5
    copy_paged_kv(k, v, ints([7, P - 2]), ints([P - 1, 3]))
    assert bool((k[P - 1] == 3).all()) and bool((v[3] == 5).all()) and bool((v[P - 1] == 0).all())


# ---------------------------------------------------------------- streams and graphs

def test_share_streams_and_graph():
    """Fork, copies, compaction and prefix in one graph, replayed with other inputs and beside
    eager calls."""
    note("share graph")
    r = random.Random(5)
    N, R, page, width, P = 12, 12, 4, 20, 400
    k = torch.randn(P, page, 2, 64, device=DEV)
    states = [random_state(r, N, page, width, P) for _ in range(4)]
    parents = [[r.randint(-1, N - 1) for _ in range(R)] for _ in range(4)]
    static = [ints(x) for x in (states[0][0], parents[0], states[0][1], states[0][2], states[0][3],
                                [states[0][4]])]

    def step():
        f = paged_kv_fork(static[0], static[1], static[2], static[3], static[4], page, static[5])
        copy_paged_kv(k, k, f.copy_src, f.copy_dst, f.copy_rows)
        c = paged_kv_compact(f.kv_lens, f.block_tables, f.page_shares, f.free_pages, page,
                             f.free_head)
        copy_paged_kv(k, k, c.copy_src, c.copy_dst)
        return (*f, *c, *paged_kv_prefix(f.kv_lens, c.block_tables, page))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    start = torch.randn(P, page, 2, 64, device=DEV)
    for trial in (1, 2, 3, 1, 0):
        lens, table, shares, free, head = states[trial]
        for t, x in zip(static, (lens, parents[trial], table, shares, free, [head])):
            t.copy_(ints(x))
        k.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        after = k.clone()
        k.copy_(start)
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)) and torch.equal(after, k)
        f = ref.fork(lens, parents[trial], table, shares, free, page, head)
        c = ref.compact(f[0], f[1], f[2], f[3], page, f[4])
        assert out[8].tolist() == c[0] and out[12].tolist() == c[4]
        assert out[15].tolist() == ref.prefix(f[0], c[0], page)[0]

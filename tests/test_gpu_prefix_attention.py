"""Attention of rows that share the beginnings of their pages, against the plain 64-bit form
(tests/paged_reference.py), on an MI355X."""
import math

import pytest
import torch

import paged_reference as ref
from vecattention_amd import (paged_decode_attention, paged_kv_prefix,
                              paged_prefix_decode_attention)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def note(*a):
    print("[case]", *a, flush=True)


def make(groups, Hq, Hk, D, page, layout, dtype, seed=0):
    """Rows in groups [(prefix tokens, [own tokens of each row])]: the prefix's whole pages are
    shared, the rest of it is each row's own copy, as a fork leaves it.  Returns q, caches, tables
    and lengths on the CPU."""
    g = torch.Generator().manual_seed(seed)
    lens, rows, used = [], [], 0
    for prefix, owns in groups:
        whole = prefix // page
        base = list(range(used, used + whole))
        used += whole
        for own in owns:
            length = prefix + own if own >= 0 else 0
            held = -(-length // page)
            more = max(held - whole, 0)
            rows.append((base + list(range(used, used + more)))[:held])
            used += more
            lens.append(length)
    width = max([len(r) for r in rows] + [1])
    pages = used + 3
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(rows), width), -1, dtype=torch.int32)
    for n, r in enumerate(rows):
        table[n, :len(r)] = order[torch.tensor(r, dtype=torch.long)].int()
    shape = (pages, page, Hk, D) if layout == "NHD" else (pages, Hk, page, D)
    kc, vc = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(len(rows), Hq, D, generator=g).to(dtype)
    return q, kc, vc, table, torch.tensor(lens, dtype=torch.int32)


def widened(table, kc, layout="NHD"):
    """The same table with room for longer requests: so much that the prefix is computed once (the
    form goes by the tables' width), however few keys there are."""
    page, Hk = (kc.shape[1], kc.shape[2]) if layout == "NHD" else (kc.shape[2], kc.shape[1])
    D = kc.shape[3]
    most = (260 if kc.dtype == F32 and D == 128 else 130) << 20
    width = -(-most // (4 * len(table) * page * Hk * D))
    more = torch.full((len(table), max(width - table.shape[1], 0)), -1, dtype=torch.int32)
    return torch.cat([table, more.to(table.device)], 1)


def room(q, kc, vc, table, lens, layout, scale=None):
    """(want, slack): the plain form's slack, and the rounding of the shared keys' weights to 16
    bits: by half a step each, in the sum of the values and in the weights' sum.  fp16 holds
    weights to 2^-25 of 2^-7 of the greatest."""
    want, slack = ref.decode(q, kc, vc, table, lens, layout, scale)
    if q.dtype != F32:
        size, _ = ref.decode(q, kc, vc.abs(), table, lens, layout, scale)
        slack = slack + 2 * ref.HALF_STEP[q.dtype] * size
        if q.dtype == F16:
            slack = slack + 2.0 ** -31 * int(lens.max()) * float(vc.abs().max())
    return want, slack


def run(q, kc, vc, table, lens, layout="NHD", ids=None, scale=None, wide=True):
    page = kc.shape[1 if layout == "NHD" else 2]
    d_table, d_lens = (widened(table, kc, layout) if wide else table).to(DEV), lens.to(DEV)
    prefix = paged_kv_prefix(d_lens, d_table, page, None if ids is None else ids.to(DEV))
    out = paged_prefix_decode_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), d_table, d_lens, prefix,
                                        kv_layout=layout, sm_scale=scale)
    torch.cuda.synchronize()
    return out, prefix


def check(case, layout="NHD", ids=None, scale=None, wide=True):
    q, kc, vc, table, lens = case
    note("attend", list(q.shape), list(kc.shape), layout, q.dtype, "rows", len(lens))
    out, prefix = run(q, kc, vc, table, lens, layout, ids, scale, wide)
    want, slack = room(q, kc, vc, table, lens, layout, scale)
    assert out.dtype == q.dtype and out.shape == want.shape
    off = (out.double().cpu() - want).abs()
    most = ref.rounded(want, slack, q.dtype)
    assert bool((off <= most).all()), (float((off - most).max()), float(off.max()))
    assert bool((out[lens.to(DEV) <= 0] == 0).all())
    return out, prefix


CASES = [
    ([(130, [1, 5, 40])], 4, 2, 128, 16, "NHD"),
    ([(64, [0, 0])], 4, 4, 64, 16, "HND"),                       # nothing of their own
    ([(63, [1, 2, 3])], 28, 4, 128, 16, "NHD"),                  # less than a tile
    ([(1000, [3] * 8)], 28, 4, 128, 16, "NHD"),
    ([(512, list(range(40)))], 28, 4, 128, 64, "HND"),           # three tiles of rows
    ([(777, [9, 300, 2]), (200, [1, 1]), (0, [50, 70]), (640, [5] * 5)], 8, 2, 64, 16, "NHD"),
    ([(300, [4, 5]), (0, [-1, -1, 33]), (300, [9]), (131, [0, 1, 2])], 6, 3, 128, 24, "NHD"),
    ([(2000, [7, 1])], 40, 2, 64, 1, "HND"),
    ([(1500, [17, 90, 3])], 16, 16, 64, 5, "NHD"),
    ([(900, [1, 1]), (900, [2, 2])], 12, 2, 128, 12, "HND"),
    ([(700, [30] * 3)], 8, 1, 128, 128, "NHD"),
    ([(4000, [100, 1])], 300, 2, 64, 16, "NHD"),                 # a request's heads fill a tile
    ([(260, [2, 2])], 4, 4, 128, 48, "NHD"),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("groups,Hq,Hk,D,page,layout", CASES)
def test_matches_the_plain_form(groups, Hq, Hk, D, page, layout, dtype):
    case = make(groups, Hq, Hk, D, page, layout, dtype, len(groups) + Hq)
    check(case, layout)
    check(case, layout, wide=False)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 40, 256])
def test_any_head_dim(D, dtype):
    check(make([(200, [4, 9]), (0, [3])], 6, 2, D, 16, "NHD", dtype, D))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 24)])
def test_long_prefixes_in_many_shares(D, page, dtype):
    check(make([(20011, [33, 5, 1, 800]), (6000, [1, 2])], 8, 2, D, page, "NHD", dtype, D + page))


def test_many_rows_and_groups():
    check(make([(100 + 64 * (i % 5), [i % 7] * (1 + i % 4)) for i in range(90)], 4, 2, 64, 16,
               "NHD", BF16, 1))
    check(make([(320, [n % 50 for n in range(300)])], 4, 1, 128, 16, "NHD", F16, 2))


def test_ids_choose_the_groups():
    case = make([(640, [5, 6, 7, 8, 9, 1])], 8, 2, 128, 16, "NHD", BF16, 3)
    ids = torch.tensor([3, 3, 9, 9, 9, 3], dtype=torch.int32)
    a, prefix = check(case, ids=ids)
    assert prefix.group_rows.tolist() == [2, 0, 3, 0, 0, 0]
    assert prefix.prefix_lens.tolist() == [640] * 5 + [0]
    b, prefix = check(case)
    assert prefix.group_rows.tolist() == [6, 0, 0, 0, 0, 0]


def test_agrees_with_the_unshared_form():
    note("unshared")
    q, kc, vc, table, lens = (t.to(DEV) for t in make([(5000, [60, 7, 900, 1]), (64, [3, 3])], 28,
                                                      4, 128, 16, "NHD", BF16, 5))
    table = widened(table, kc)
    shared = paged_prefix_decode_attention(q, kc, vc, table, lens, paged_kv_prefix(lens, table, 16))
    plain = paged_decode_attention(q, kc, vc, table, lens)
    assert float((shared.double() - plain.double()).norm() / plain.double().norm()) < 2.0 ** -8
    none = torch.zeros_like(lens)
    alone = paged_prefix_decode_attention(q, kc, vc, table, lens, (none, none))
    assert float((alone.double() - plain.double()).norm() / plain.double().norm()) < 2.0 ** -10


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-4])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scales(scale, dtype):
    check(make([(400, [1, 20])], 4, 2, 64, 16, "NHD", dtype, 6), scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_small_weights_beside_a_great_one(dtype):
    """One shared key far above the others, or one own key: the others' sum counts."""
    for at in (3, 700, 4090, 4100):
        q, kc, vc, table, lens = make([(4096, [9, 30])], 2, 1, 64, 16, "NHD", dtype, at)
        q[:] = 0.5
        kc[:] = 0
        page, row = int(table[0, min(at, 4104) // 16]), at % 16
        kc[page, row] = 0.25                      # a score of 8 * scale 1 = 8 nats more
        kc[int(table[1, min(at, 4104) // 16]), row] = 0.25
        vc[page, row] = 0
        check((q, kc, vc, table, lens), scale=1.0)


def test_scores_whose_steps_are_large():
    """Scores of 2^27 and more, where m + 8 is not a number: no weight overflows fp16."""
    for top in (2.0 ** 20, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28, 2.0 ** 30):
        q, kc, vc, table, lens = make([(640, [3, 3])], 2, 1, 64, 16, "NHD", F16, 9)
        g = torch.Generator().manual_seed(int(top) % 1000)
        q[:] = 256
        kc[:] = (1 + torch.randint(0, 64, kc.shape[:-1] + (1,), generator=g) / 64).half() * 64
        out, _ = run(q, kc, vc, table, lens, scale=top / 2.0 ** 20)
        assert bool(torch.isfinite(out).all()), top
        # The greatest scores are exact ties here, so the weights are those of the maximum.
        want, _ = ref.decode(q, kc, vc, table, lens, "NHD", top / 2.0 ** 20)
        assert float((out.double().cpu() - want).abs().max()) < 2.0 ** -8


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_pages_that_cannot_be_read(dtype):
    note("bad pages", dtype)
    case = make([(640, [5, 6, 7]), (128, [3, 3]), (0, [20])], 4, 2, 64, 16, "NHD", dtype, 11)
    q, kc, vc, table, lens = case
    want, slack = room(*case, "NHD")
    for n, k, bad in ((0, 3, 10 ** 6), (3, 7, kc.shape[0]), (1, 40, -1), (5, 0, -7)):
        broken = widened(table, kc)
        rows = [n]
        if n in (0, 3) and k < (40 if n == 0 else 8):  # a page that the whole group shares
            rows = [0, 1, 2] if n == 0 else [3, 4]
        for r in rows:
            broken[r, k] = bad
        d = [t.to(DEV) for t in (q, kc, vc, broken, lens)]
        prefix = paged_kv_prefix(d[4], table.to(DEV), 16)  # as it was found before
        out = paged_prefix_decode_attention(*d[:5], prefix).double().cpu()
        for r in range(len(lens)):
            if r in rows:
                assert bool(torch.isnan(out[r]).all()), (n, r)
            else:
                assert bool(((out[r] - want[r]).abs()
                             <= ref.rounded(want, slack, dtype)[r]).all()), (n, r)
    short = table[:, :30].contiguous()  # tables narrower than the lengths
    out, _ = run(q, kc, vc, short, lens, wide=False)
    assert bool(torch.isnan(out[:3]).all()) and bool(torch.isfinite(out[3:]).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 24)])
def test_values_that_are_not_finite(D, page, dtype):
    """They reach the outputs of their own feature and rows, whatever their key's weight is."""
    for at, value in ((5, math.inf), (500, -math.inf), (37, math.nan), (610, math.inf)):
        note("values", D, page, dtype, at, value)
        q, kc, vc, table, lens = make([(600, [20, 30, 1]), (70, [4, 4])], 8, 2, D, page, "NHD",
                                      dtype, at)
        whole = 600 // page * page
        far = at == 500
        if far:  # a key whose weight is too small for any type
            q[:, :, 0] = 8
            kc[..., 0] = 0
            kc[int(table[0, at // page]), at % page, :, 0] = -240
        vc[int(table[0, at // page]), at % page, 1, 3] = value
        out, _ = run(q, kc, vc, table, lens, scale=1.0)
        out = out.double().cpu()
        clean = vc.clone()
        clean[int(table[0, at // page]), at % page, 1, 3] = 0
        want, slack = room(q, kc, clean, table, lens, "NHD", 1.0)
        touched = torch.zeros_like(want, dtype=torch.bool)
        for n in range(3 if at < whole else 1):
            if at < int(lens[n]):
                touched[n, 4:, 3] = True
        if math.isnan(value):
            assert bool(torch.isnan(out[touched]).all())
        else:
            assert bool((out[touched] == value).all())
        room_ = ref.rounded(want, slack, dtype)
        assert bool(((out - want).abs() <= room_)[~touched].all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_keys_that_are_not_finite(dtype):
    for value in (math.inf, math.nan):
        note("keys", dtype, value)
        q, kc, vc, table, lens = make([(320, [20, 30]), (320, [4, 4])], 8, 2, 64, 16, "NHD", dtype)
        kc[int(table[0, 3]), 2, 1, 5] = value
        out, _ = run(q, kc, vc, table, lens)
        q[:, :, 5] = q[:, :, 5].abs() + 1
        assert bool(torch.isnan(run(q, kc, vc, table, lens)[0][:2, 4:]).all())
        want, slack = room(q, torch.where(torch.isfinite(kc), kc, 0), vc, table, lens, "NHD")
        off = (run(q, kc, vc, table, lens)[0].double().cpu() - want).abs()
        fine = off <= ref.rounded(want, slack, dtype)
        assert bool(fine[2:].all()) and bool(fine[:2, :4].all())
    # A key of weight 0 (a score of -infinity), and rows of such keys alone: 0 / 0.
    q, kc, vc, table, lens = make([(320, [20, 30]), (320, [0, 0])], 2, 1, 64, 16, "NHD", dtype)
    q[:, :, 5] = 1
    kc[int(table[0, 3]), 2, 0, 5] = -math.inf
    for p in table[2, :20].tolist():
        kc[p, :, 0, 5] = -math.inf
    out, _ = run(q, kc, vc, table, lens)
    assert bool(torch.isnan(out[2:]).all())
    kc[int(table[0, 3]), 2, 0] = 0
    kc[int(table[0, 3]), 2, 0, 5] = -30000  # a weight of 0 in any type
    want, slack = room(q[:2], kc, vc, table[:2], lens[:2], "NHD")
    assert bool(((out[:2].double().cpu() - want).abs() <= ref.rounded(want, slack, dtype)).all())


def test_strided_views():
    q, kc, vc, table, lens = make([(600, [20, 30, 1]), (70, [4, 4])], 8, 2, 64, 16, "NHD", BF16, 4)
    want, slack = room(q, kc, vc, table, lens, "NHD")
    d_q = torch.zeros(5, 8, 100, dtype=BF16, device=DEV)[:, :, 8:72]
    d_q.copy_(q)
    wide = torch.zeros(kc.shape[0], 16, 5, 72, dtype=BF16, device=DEV)
    wide[:, :, 1:5:2, :64] = vc.to(DEV)
    tall = torch.zeros(kc.shape[0] * 2, 16, 2, 64, dtype=BF16, device=DEV)
    tall[::2] = kc.to(DEV)
    odd = torch.zeros(kc.numel() + 1, dtype=BF16, device=DEV)[1:].view(kc.shape)
    odd.copy_(kc)
    d_table = widened(table, kc).to(DEV)
    pairs = torch.stack([lens, lens + 1], 1).to(DEV)
    prefix = paged_kv_prefix(pairs[:, 0], d_table, 16)
    doubled = [torch.stack([t, t], 1)[:, 0] for t in prefix]
    for k in (tall[::2], odd):
        for t in (d_table, d_table.t().contiguous().t()):
            note("strided")
            out = paged_prefix_decode_attention(d_q, k, wide[:, :, 1:5:2, :64], t, pairs[:, 0],
                                                doubled)
            off = (out.double().cpu() - want).abs()
            assert bool((off <= ref.rounded(want, slack, BF16)).all())


def test_offsets_past_32_bits():
    note("far pages")
    q, kc, vc, table, lens = make([(640, [20, 30])], 8, 2, 128, 16, "NHD", BF16, 4)
    P = kc.shape[0]
    big_k = torch.zeros(400000, 16, 2, 128, dtype=BF16, device=DEV)  # 3.3 GB
    big_v = torch.zeros(400000, 16, 2, 128, dtype=BF16, device=DEV)
    at = 400000 - P
    big_k[at:], big_v[at:] = kc.to(DEV), vc.to(DEV)
    far = widened(torch.where(table >= 0, table + at, table), kc).to(DEV)
    d_lens = lens.to(DEV)
    out = paged_prefix_decode_attention(q.to(DEV), big_k, big_v, far, d_lens,
                                        paged_kv_prefix(d_lens, far, 16))
    near = run(q, kc, vc, table, lens)[0]
    assert torch.equal(out, near)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("more", [0, 30])
def test_fp32_tiles_of_every_height(D, more):
    """8, 48 and 160 rows a kv head: one, two and four waves take turns at a tile's keys; `more`
    rows that share nothing take the batch past the 64 that a wave counts by itself."""
    check(make([(700, [3, 1]), (1030, [5] * 12), (390, [2] * 40)] + [(0, [20])] * more, 8, 2, D, 16,
               "NHD", F32, 11))


def test_streams_and_two_graphs():
    """Two captured graphs and eager calls on another stream, each with a workspace of its own."""
    note("graphs")
    cases = [[t.to(DEV) for t in make([(3000 + 100 * s, [60, 7, 300, 1]), (640, [3, 3])], 8, 2, 128,
                                      16, "NHD", BF16, s)] for s in (0, 1)]
    for case in cases:
        case[3] = widened(case[3], case[1])
    want = []
    for q, kc, vc, table, lens in cases:
        want.append(paged_prefix_decode_attention(q, kc, vc, table, lens,
                                                  paged_kv_prefix(lens, table, 16)))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, kc, vc, table, lens in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            prefix = paged_kv_prefix(lens, table, 16)
            outs.append(paged_prefix_decode_attention(q, kc, vc, table, lens, prefix))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for trial in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
            graphs[1].replay()
        q, kc, vc, table, lens = cases[trial % 2]
        eager = paged_prefix_decode_attention(q, kc, vc, table, lens,
                                              paged_kv_prefix(lens, table, 16))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(eager, want[trial % 2])


def test_same_bits_every_time():
    note("same bits")
    q, kc, vc, table, lens = (t.to(DEV) for t in make([(9000, [60, 7, 300, 1]), (640, [3, 3])], 28,
                                                      4, 128, 16, "NHD", BF16, 3))
    table = widened(table, kc)
    prefix = paged_kv_prefix(lens, table, 16)
    want = paged_prefix_decode_attention(q, kc, vc, table, lens, prefix)
    for _ in range(5):
        assert torch.equal(paged_prefix_decode_attention(q, kc, vc, table, lens, prefix), want)


def test_no_backward():
    q, kc, vc, table, lens = (t.to(DEV) for t in make([(64, [1, 1])], 2, 1, 64, 16, "NHD", F32))
    prefix = paged_kv_prefix(lens, table, 16)
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, kc, vc))]
        with pytest.raises(NotImplementedError, match="no backward"):
            paged_prefix_decode_attention(*args, table, lens, prefix)
    with torch.no_grad():
        paged_prefix_decode_attention(*args, table, lens, prefix)

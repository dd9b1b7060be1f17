"""Attention of rows that share the beginnings of their pages where its arithmetic is at its ends:
scores whose steps are large, weights far below the greatest one, infinities and NaN, in every type
and with one, two and four waves at a tile's rows, on an MI355X."""
import math

import pytest
import torch

import paged_reference as ref
from test_gpu_prefix_attention import check, make, note, room, run, widened
from vecattention_amd import (paged_decode_attention, paged_kv_prefix,
                              paged_prefix_decode_attention)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# (groups, query heads, kv heads, head_dim, page size): 2 and 4 rows, 48 rows, 160 rows a kv head,
# in one piece of work or several, in pages of whole tiles and of any size.
SHAPES = [([(4096, [9, 30])], 2, 1, 64, 16),
          ([(700, [3, 1])], 4, 2, 128, 24),
          ([(640, [2] * 12)], 8, 2, 64, 24),
          ([(256, [2] * 40)], 8, 2, 128, 16)]


def row_of(c, table, n, t, page):
    return c[int(table[n, t // page]), t % page]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("own", [[3, 3], [0, 0]])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_scores_of_large_steps_of_either_sign(dtype, D, own, sign):
    """Equal scores of 2^24 to 2^31 in size, whatever their scaled value rounds to: every key has
    the same weight, and the output is the values' mean."""
    q, kc, vc, table, lens = make([(640, own)], 2, 1, D, 16, "NHD", dtype, 9)
    vc = vc.abs()
    want = torch.stack([torch.stack([row_of(vc, table, n, t, 16)[0].double()
                                     for t in range(int(lens[n]))]).mean(0) for n in range(2)])
    want = want[:, None].expand(2, 2, D)
    q[:], kc[:] = 0, 0
    q[:, :, 0] = 2048.0
    for num in (33, 37, 41, 48, 55, 61, 63):      # of 32: not powers of two
        for exponent in (4, 9, 10):
            kc[..., 0] = sign * 512.0 * num / 32  # scores of 2^20 * num / 32, exactly
            out, _ = run(q, kc, vc, table, lens, scale=2.0 ** exponent)
            # The weights are one power of two for all keys, exactly: 2^0 of a whole exponent.
            # Both sums have at most 643 terms, and the quotient one rounding.
            slack = 2 * 644 * 2.0 ** -24 * want
            off = (out.double().cpu() - want).abs()
            assert bool((off <= ref.rounded(want, slack, dtype)).all()), (num, exponent,
                                                                          float(off.max()))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("groups,Hq,Hk,D,page", SHAPES)
def test_small_weights_beside_a_sink(groups, Hq, Hk, D, page, dtype):
    """One key 12 to 24 nats above the others whose value is 0, among the shared keys or a row's
    own: what the others' small weights add up to is all of the output."""
    note("sink", groups[0][0], Hq, Hk, D, page, dtype)
    g = torch.Generator().manual_seed(D + page)
    q, kc, vc, table, lens = make(groups, Hq, Hk, D, page, "NHD", dtype, D)
    shared, L = groups[0][0], int(lens.max())
    q[:] = 0
    q[:, :, 0] = 1.0                       # a score is feature 0 of its key, exactly
    kc[..., 0] = (0.3 * torch.randn(kc.shape[:-1], generator=g)).to(dtype)
    for at in (shared // 3, shared - page - 1, shared + 1):
        for gap, size in ((12.0, 1.0), (16.0, 1.0), (18.0, 1.0), (24.0, 500.0)):
            k, v = kc.clone(), (size * (vc.abs() + 0.125)).to(dtype)
            for n in range(len(lens)):
                if at < int(lens[n]):
                    row_of(k, table, n, at, page)[:, 0] = gap
                    row_of(v, table, n, at, page)[:] = 0
            out, _ = run(q, k, v, table, lens, scale=1.0)
            for n in sorted({0, 1, len(lens) - 1}):
                t = torch.arange(int(lens[n]))
                rows = table[n].long()[t // page] * page + t % page
                K, V = (ref.cache_rows(c, "NHD")[rows].double().repeat_interleave(Hq // Hk, 1)
                        for c in (k, v))
                want = (torch.softmax(K[..., 0], 0)[..., None] * V).sum(0)
                # Roundings of 2^-24 each: scores of size below 37 in units of log2(e) (three for
                # the scaled score, one for the difference, one step of exp2: below 250 in a
                # weight and in the weights' sum together), and the two sums of L terms.  Shared
                # keys' weights of 16 bits: half a step of each, in the values' sum and in the
                # weights' own.  fp16's end 2^-44 below the greatest one.
                slack = (2 * L + 250) * 2.0 ** -24 * want
                if dtype != F32:
                    slack = slack + 2 * ref.HALF_STEP[dtype] * want
                if dtype == F16:
                    slack = slack + L * 2.0 ** -44 * V.max()
                off = (out[n].double().cpu() - want).abs()
                assert bool((off <= ref.rounded(want, slack, dtype)).all()), (
                    at, gap, n, float((off / want.abs().clamp_min(1e-30)).max()))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("groups,Hq,Hk,D,page", SHAPES)
def test_finite_outputs_beside_others(groups, Hq, Hk, D, page, dtype):
    """An infinite value or a NaN among the shared values, or in a query, reaches the outputs that
    the formula has it in; all others stay as they are, bit for bit."""
    note("beside others", groups[0][0], Hq, Hk, D, page, dtype)
    q, kc, vc, table, lens = make(groups, Hq, Hk, D, page, "NHD", dtype, D)
    G, shared = Hq // Hk, groups[0][0] // page * page
    clean, _ = run(q, kc, vc, table, lens)
    assert bool(torch.isfinite(clean).all())
    v = vc.clone()
    row_of(v, table, 0, shared // 2, page)[0, 3] = math.inf
    row_of(v, table, 0, 1, page)[0, 9] = -math.inf
    row_of(v, table, 0, shared // 3, page)[Hk - 1, 5] = math.nan
    want = clean.clone()
    want[:, :G, 3], want[:, :G, 9] = math.inf, -math.inf
    out, _ = run(q, kc, v, table, lens)
    assert bool(torch.isnan(out[:, Hq - G:, 5]).all())
    out[:, Hq - G:, 5] = want[:, Hq - G:, 5]
    assert torch.equal(out, want)
    q[1, 1, 7] = math.nan
    out, _ = run(q, kc, vc, table, lens)
    assert bool(torch.isnan(out[1, 1]).all())
    out[1, 1] = clean[1, 1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("page", [16, 24])
def test_finite_outputs_beside_others_of_many_rows(page, dtype):
    """The same of more rows than a wave counts by itself, in groups of one row to four."""
    note("beside others, many rows", page, dtype)
    groups = [(100 + 64 * (i % 5), [i % 7] * (1 + i % 4)) for i in range(90)]
    q, kc, vc, table, lens = make(groups, 4, 2, 64, page, "NHD", dtype, 1)
    clean, _ = run(q, kc, vc, table, lens)
    want, n = clean.clone(), 0
    for i, (_, own) in enumerate(groups):
        if i % 3 == 0:
            row_of(vc, table, n, 7, page)[1, 11] = -math.inf
            want[n:n + len(own), 2:, 11] = -math.inf
        n += len(own)
    out, _ = run(q, kc, vc, table, lens)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("groups,Hq,Hk,D,page", SHAPES)
def test_infinite_values_of_tiny_weights(groups, Hq, Hk, D, page, dtype):
    """An infinite value whose weight is too small for fp32, before and behind the key that makes
    it so, is infinite all the same; beside a score of -infinity it is a NaN (0 times infinity)."""
    note("tiny weights", groups[0][0], Hq, Hk, D, page, dtype)
    q, kc, vc, table, lens = make(groups, Hq, Hk, D, page, "NHD", dtype, D)
    shared = groups[0][0] // page * page
    q[:] = 0
    q[:, :, 0] = 1.0
    kc[..., 0] = 0
    row_of(kc, table, 0, shared // 2, page)[:, 0] = 560.0
    row_of(vc, table, 0, 2, page)[0, 3] = math.inf
    row_of(vc, table, 0, shared - 80, page)[0, 5] = -math.inf
    row_of(vc, table, 0, shared // 3, page)[0, 7] = math.inf
    row_of(kc, table, 0, shared // 3, page)[:, 0] = -math.inf
    out, _ = run(q, kc, vc, table, lens, scale=1.0)
    out = out[:, :Hq // Hk].double().cpu()
    assert bool((out[:, :, 3] == math.inf).all()) and bool((out[:, :, 5] == -math.inf).all())
    assert bool(torch.isnan(out[:, :, 7]).all())
    great = row_of(vc, table, 0, shared // 2, page)[0].double()
    others = [i for i in range(D) if i not in (3, 5, 7)]
    # The great key's weight is 1, the others' below 2^-800.
    assert bool((out[:, :, others] == great[others]).all())


@pytest.mark.parametrize("groups,Hq,Hk,D,page", SHAPES)
def test_keys_that_are_not_finite_in_fp32(groups, Hq, Hk, D, page):
    for value in (math.inf, math.nan):
        note("keys", groups[0][0], Hq, Hk, D, page, value)
        q, kc, vc, table, lens = make(groups + [(320, [4, 4])], Hq, Hk, D, page, "NHD", F32)
        rows, G = len(groups[0][1]), Hq // Hk
        q[:, :, 5] = q[:, :, 5].abs() + 1
        kc[int(table[0, 3]), 2, Hk - 1, 5] = value
        out, _ = run(q, kc, vc, table, lens)
        assert bool(torch.isnan(out[:rows, Hq - G:]).all())
        want, slack = room(q, torch.where(torch.isfinite(kc), kc, 0), vc, table, lens, "NHD")
        fine = (out.double().cpu() - want).abs() <= ref.rounded(want, slack, F32)
        assert bool(fine[rows:].all()) and bool(fine[:rows, :Hq - G].all())
        # Scores of -infinity: a weight of 0, and rows of such keys alone 0 / 0.
        q, kc, vc, table, lens = make(groups + [(320, [0, 0])], Hq, Hk, D, page, "NHD", F32)
        q[:, :, 5] = 1
        kc[int(table[0, 3]), 2, :, 5] = -math.inf
        whole = 320 // page * page
        for n in (rows, rows + 1):
            for t in range(int(lens[n])):
                row_of(kc, table, n, t, page)[:, 5] = -math.inf
        assert whole >= 64
        out, _ = run(q, kc, vc, table, lens)
        assert bool(torch.isnan(out[rows:]).all())
        kc[int(table[0, 3]), 2] = 0
        kc[int(table[0, 3]), 2, :, 5] = -30000.0  # a weight of 0 in any type
        want, slack = room(q[:rows], kc, vc, table[:rows], lens[:rows], "NHD")
        assert bool(((out[:rows].double().cpu() - want).abs()
                     <= ref.rounded(want, slack, F32)).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-4])
@pytest.mark.parametrize("groups,Hq,Hk,D,page", SHAPES[1:])
def test_scales_in_fp32(groups, Hq, Hk, D, page, scale):
    check(make(groups, Hq, Hk, D, page, "NHD", F32, 6), scale=scale)


@pytest.mark.parametrize("D,page", [(128, 16), (64, 24)])
def test_long_prefixes_in_many_shares_in_fp32(D, page):
    check(make([(20011, [33, 5, 1, 800]), (6000, [1, 2])], 8, 2, D, page, "NHD", F32, D + page))


def test_prefix_of_30000_keys():
    for dtype in (BF16, F16, F32):
        check(make([(30001, [12, 5])], 4, 2, 64, 16, "HND", dtype, 30), layout="HND")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_same_bits_in_graphs_and_outside(D, dtype):
    """Eager calls, replays and calls on a side stream, of values with an infinity among them."""
    note("graph", D, dtype)
    q, kc, vc, table, lens = make([(5000, [60, 7, 300, 1]), (640, [3] * 12)], 8, 2, D, 16, "NHD",
                                  dtype, 3)
    row_of(vc, table, 0, 77, 16)[0, 3] = math.inf
    q, kc, vc, table, lens = (t.to(DEV) for t in (q, kc, vc, widened(table, kc), lens))
    want = paged_prefix_decode_attention(q, kc, vc, table, lens, paged_kv_prefix(lens, table, 16))
    assert int(torch.isinf(want).sum()) == 4 * 4 and not bool(torch.isnan(want).any())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prefix = paged_kv_prefix(lens, table, 16)
        out = paged_prefix_decode_attention(q, kc, vc, table, lens, prefix)
    side = torch.cuda.Stream()
    for _ in range(4):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        eager = paged_prefix_decode_attention(q, kc, vc, table, lens,
                                              paged_kv_prefix(lens, table, 16))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager, want)


def both(N, shared, Hq, Hk, D, dtype, more=0):
    """(shared form or not, every row for itself) of N rows over the same whole pages of 16, in
    tables with room for `more` keys."""
    g = torch.Generator(device=DEV).manual_seed(N + shared)
    shape = (shared // 16 + 1, 16, Hk, D)
    kc, vc = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn(N, Hq, D, generator=g, device=DEV).to(dtype)
    table = torch.full((N, (shared + more) // 16), -1, dtype=torch.int32, device=DEV)
    table[:, :shared // 16] = torch.arange(shared // 16, device=DEV)
    lens = torch.full((N,), shared, dtype=torch.int32, device=DEV)
    prefix = paged_kv_prefix(lens, table, 16)
    assert prefix.prefix_lens.tolist() == [shared] * N
    return (paged_prefix_decode_attention(q, kc, vc, table, lens, prefix),
            paged_decode_attention(q, kc, vc, table, lens))


def test_batches_that_are_faster_row_by_row():
    """Many rows of short tables, and few rows of few keys, take the form of one row, bit for bit;
    batches past the border the shared one, with the same result to the types' roundings."""
    for N, keys, Hq, Hk, D, dtype in ((200, 256, 16, 16, 64, BF16), (200, 256, 32, 8, 128, BF16),
                                      (64, 512, 32, 8, 128, F16), (64, 1024, 28, 4, 128, BF16),
                                      (8, 4096, 28, 4, 128, F16), (8, 8192, 28, 4, 128, F32),
                                      (2, 2048, 16, 16, 64, F32)):
        note("by rows", N, keys, Hq, Hk, D, dtype)
        assert torch.equal(*both(N, keys, Hq, Hk, D, dtype)), (N, keys)
    for N, keys, Hq, Hk, D, dtype, more in (
            (200, 512, 16, 16, 64, BF16, 0), (64, 1536, 28, 4, 128, BF16, 0),
            (8, 2048, 16, 16, 64, F16, 0), (8, 2048, 16, 16, 64, F32, 0),
            (300, 640, 4, 1, 128, F16, 2000), (8, 6144, 28, 4, 128, BF16, 0)):
        note("shared", N, keys, Hq, Hk, D, dtype)
        out, want = both(N, keys, Hq, Hk, D, dtype, more)
        assert not torch.equal(out, want), (N, keys)
        # Weights rounded by half a step each in both sums, against values of size 1 whose mean
        # over `keys` equal-like weights is about keys^-1/2: in the norm, one step of the type.
        off = float((out.double() - want.double()).norm() / want.double().norm())
        assert off < 2 * ref.HALF_STEP[dtype] if dtype != F32 else off < 2.0 ** -18, (N, off)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("count,Hq,Hk,D,page", [(32, 32, 32, 64, 16), (40, 32, 16, 64, 24)])
def test_more_pieces_than_work_groups(count, Hq, Hk, D, page, dtype):
    """1024 and 640 pieces of work, for 512 work-groups: of up to 64 rows, which a wave counts by
    itself, and of more; with infinite values in some groups, all other outputs bit for bit."""
    note("pieces", count, Hq, Hk, D, page, dtype)
    groups = [(100 + 64 * (i % 4), [i % 5, 3]) for i in range(count)]
    case = make(groups, Hq, Hk, D, page, "NHD", dtype, 7)
    clean, _ = check(case)
    q, kc, vc, table, lens = case
    want = clean.clone()
    for i in range(0, count, 3):
        row_of(vc, table, 2 * i, 5, page)[Hk - 1, 11] = math.inf
        row_of(vc, table, 2 * i, 40, page)[0, 2] = math.nan
        want[2 * i:2 * i + 2, -(Hq // Hk):, 11] = math.inf
    out, _ = run(q, kc, vc, table, lens)
    for i in range(0, count, 3):
        assert bool(torch.isnan(out[2 * i:2 * i + 2, :Hq // Hk, 2]).all())
        out[2 * i:2 * i + 2, :Hq // Hk, 2] = want[2 * i:2 * i + 2, :Hq // Hk, 2]
    assert torch.equal(out, want)

"""The operators over a paged key-value cache against their plain 64-bit forms
(tests/paged_reference.py), on an MI355X."""
import math

import pytest
import torch

import paged_reference as ref
from vecattention_amd import (paged_decode_attention, paged_kv_plan, qk_norm_rope,
                              qk_norm_rope_to_cache, single_decode_with_kv_cache, write_paged_kv)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def note(*a):
    print("[case]", *a, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, slack, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    room = ref.rounded(want, slack, dtype)
    assert bool((off <= room).all()), (float((off - room).max()), float(off.max()))


# ---------------------------------------------------------------- the plan

def plan_case(lens, new, page, width, free, seed=0, head=None, tokens=None, gap=0):
    note("plan", len(lens), "requests, page", page, "width", width, "free", len(free))
    g = gen(seed)
    N = len(lens)
    table = torch.randint(-1, 50000, (N, width + gap), generator=g, dtype=torch.int32)
    lens, new = torch.tensor(lens, dtype=torch.int32), torch.tensor(new, dtype=torch.int32)
    free = torch.as_tensor(free, dtype=torch.int32)
    total = int(new.clamp(min=0).sum())
    tokens = total + 5 if tokens is None else tokens
    want = ref.plan(lens, new, table[:, :width].tolist(), free, page, tokens, head or 0)
    d_table = table.to(DEV)
    got = paged_kv_plan(lens.to(DEV), new.to(DEV), d_table[:, :width], free.to(DEV), page, tokens,
                        None if head is None else torch.tensor([head], dtype=torch.int32,
                                                               device=DEV))
    torch.cuda.synchronize()
    assert d_table[:, :width].tolist() == want[0]
    assert torch.equal(d_table[:, width:].cpu(), table[:, width:])
    for name, a, b in zip(got._fields, got, want[1:]):
        assert a.flatten().tolist() == (b if isinstance(b, list) else [b]), name


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("N", [1, 5, 64, 257, 2048, 2049, 5000])
def test_plan_matches_the_plain_form(N, page):
    g = gen(N + page)
    lens = torch.randint(0, 200, (N,), generator=g).tolist()
    new = torch.randint(0, 4, (N,), generator=g).tolist()
    new[N // 2] = 300
    plan_case(lens, new, page, -(-520 // page), torch.randperm(20000 + N, generator=g), N)


def test_plan_edges():
    plan_case([0], [1], 16, 1, [7])
    plan_case([15, 16, 17, 0], [1, 1, 0, 0], 16, 4, [3, 9])          # a page's last and first row
    plan_case([0, 0, 0], [0, 0, 0], 16, 4, [3], tokens=0)            # nothing to do
    plan_case([0, 0, 0], [0, 0, 0], 16, 4, [3], tokens=9)            # padding only
    plan_case([-3, 5], [2, -1], 4, 3, [1, 2, 3])                     # negative counts as 0
    plan_case([0, 0, 0], [40, 40, 40], 16, 5, [1, 2, 3, 4])          # the list runs out
    plan_case([0, 30], [100, 60], 16, 4, list(range(20)))            # past the table's end
    plan_case([10, 10], [30, 30], 8, 9, list(range(90)), head=80)    # from the list's middle
    plan_case([10, 10], [30, 30], 8, 9, list(range(90)), head=-2)
    plan_case([10, 10], [30, 30], 8, 9, [])                          # no page is free
    plan_case([9, 9, 9], [7, 0, 9], 8, 4, list(range(9)), gap=3)     # rows of a wider table
    plan_case([4] * 6, [3] * 6, 8, 4, list(range(9)), tokens=10)     # more tokens than rows for them
    plan_case([], [], 8, 4, [1], tokens=3)
    plan_case([2 ** 31 - 1, 5], [9, 2], 1 << 20, 2048, [4, 5])       # lengths at the type's end


def test_plan_outputs_are_tensors_of_their_own():
    """Outputs of one allocation: written, copied and used in a graph one by one."""
    note("plan outputs")
    lens, new, table, free = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (
        [3, 0], [2, 9], [[1, 0, 0], [0, 0, 0]], [5, 6, 7, 8]))
    step = paged_kv_plan(lens, new, table, free, 4, 13)
    before = [t.clone() for t in step]
    for i, t in enumerate(step):
        t.add_(1)
        for j, (a, b) in enumerate(zip(step, before)):
            assert torch.equal(a, b + 1 if j <= i else b)
        assert t.is_contiguous() and t._base is None
        assert torch.equal(t.cpu(), (before[i] + 1).cpu()) and torch.equal(t[-1:], t[len(t) - 1:])
    assert (step.positions.float().requires_grad_() * 2).sum().requires_grad


def test_plan_long_prompts_and_replayed_graph():
    note("plan graph")
    g = gen(4)
    N, page, width, tokens = 40, 16, 400, 70000
    lens = torch.randint(0, 300, (N,), generator=g, dtype=torch.int32)
    new = torch.randint(0, 3500, (N,), generator=g, dtype=torch.int32)
    free = torch.randperm(9000, generator=g).int()
    table = torch.full((N, width), -1, dtype=torch.int32)
    d = [t.to(DEV) for t in (lens, new, table, free)]
    head = torch.zeros(1, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        paged_kv_plan(*d, page, tokens, head)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_kv_plan(*d, page, tokens, head)
    for trial in range(4):
        lens = torch.randint(0, 300, (N,), generator=g, dtype=torch.int32)
        new = torch.randint(0, 1500 * trial + 2, (N,), generator=g, dtype=torch.int32)
        d[0].copy_(lens)
        d[1].copy_(new)
        d[2].fill_(7)
        head.fill_(trial * 11)
        graph.replay()
        torch.cuda.synchronize()
        want = ref.plan(lens, new, [[7] * width] * N, free, page, tokens, trial * 11)
        assert d[2].tolist() == want[0]
        for a, b in zip(out, want[1:]):
            assert a.flatten().tolist() == (b if isinstance(b, list) else [b])


# ---------------------------------------------------------------- norms and rotation

def freqs(rot):
    return (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float()


def rope_inputs(B, Hq, Hk, S, D, dtype, seed, bshd=True):
    g = gen(seed)
    shape = (lambda H: (B, S, H, D)) if bshd else (lambda H: (B, H, S, D))
    q, k = (torch.randn(shape(H), generator=g).to(dtype) for H in (Hq, Hk))
    return tuple(x.transpose(1, 2) if bshd else x for x in (q, k))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,Hq,Hk,S,D,rot,axes,norm,bshd", [
    (1, 28, 4, 333, 128, 128, 3, False, True), (2, 4, 4, 37, 64, 64, 1, True, False),
    (1, 1, 1, 1, 128, 128, 1, True, True), (3, 5, 1, 9, 128, 64, 3, True, True),
    (1, 12, 12, 70, 80, 80, 1, True, False), (2, 3, 2, 11, 96, 34, 4, True, True),
    (1, 2, 1, 19, 256, 256, 1, True, True), (1, 40, 2, 130, 64, 32, 3, True, True),
    (1, 1, 3, 5, 2, 2, 1, True, True), (1, 2, 2, 6, 512, 512, 1, False, False),
    (1, 3, 2, 1701, 128, 128, 3, True, True), (2, 5, 1, 801, 64, 48, 1, True, False),
    (1, 1, 1, 1537, 256, 128, 1, False, True)])
def test_rope_matches_the_plain_form(B, Hq, Hk, S, D, rot, axes, norm, bshd, interleaved, dtype):
    note("rope", B, Hq, Hk, S, D, rot, axes, norm, bshd, interleaved, dtype)
    g = gen(S + D)
    q, k = rope_inputs(B, Hq, Hk, S, D, dtype, S, bshd)
    pos = torch.randint(0, 200000, (axes, B, S), generator=g)
    half = rot // 2
    third = half // axes
    sections = [half - (axes - 1) * third] + [third] * (axes - 1) if axes > 1 else None
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None
              for _ in range(2))
    to = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got = qk_norm_rope(to(q), to(k), to(pos if axes > 1 else pos[0]), to(freqs(rot)), to(qw),
                       to(kw), mrope_section=sections, interleaved=interleaved)
    torch.cuda.synchronize()
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        p = (pos if axes > 1 else pos[0]).unsqueeze(-2)
        want, slack = ref.rotate(x, p, freqs(rot), w, sections=sections, interleaved=interleaved)
        within(y, want, slack, dtype)
        assert y.stride() == x.stride() or y.is_contiguous()


def test_rope_options_and_strides():
    """fp32 weights, one norm only, a scaling, int32 positions of one row, tensors cut from a
    joint projection, unaligned rows, and a feature dimension that is not contiguous."""
    note("rope options")
    g = gen(1)
    B, Hq, Hk, S, D = 2, 6, 2, 21, 64
    joint = torch.randn(B, S, Hq + 2 * Hk, D, generator=g).bfloat16()
    q, k = joint[:, :, :Hq].transpose(1, 2), joint[:, :, Hq:Hq + Hk].transpose(1, 2)
    pos = torch.randint(0, 1 << 20, (S,), generator=g, dtype=torch.int32)
    kw = 1 + 0.3 * torch.randn(D, generator=g)
    d = joint.to(DEV)
    qd, kd = d[:, :, :Hq].transpose(1, 2), d[:, :, Hq:Hq + Hk].transpose(1, 2)
    got = qk_norm_rope(qd, kd, pos.to(DEV), freqs(D).to(DEV), None, kw.to(DEV), eps=0.5,
                       attention_scaling=1.25)
    for x, w, y in ((q, None, got[0]), (k, kw, got[1])):
        within(y, *ref.rotate(x, pos.long(), freqs(D), w, eps=0.5, scaling=1.25), BF16)
    # rows that start at odd elements
    flat = torch.randn(B * Hq * S * (D + 1) + 1, generator=g).half()
    q = flat[1:].view(B, Hq, S, D + 1)[..., :D]
    fd = flat.to(DEV)
    qd = fd[1:].view(B, Hq, S, D + 1)[..., :D]
    got = qk_norm_rope(qd, qd[:, :1], pos.to(DEV), freqs(D).to(DEV))
    within(got[0], *ref.rotate(q, pos.long(), freqs(D)), F16)
    within(got[1], *ref.rotate(q[:, :1], pos.long(), freqs(D)), F16)
    # features apart
    q = torch.randn(B, Hq, D, S, generator=g).transpose(2, 3)
    got = qk_norm_rope(q.to(DEV), q.to(DEV), pos.to(DEV), freqs(D).to(DEV))
    within(got[0], *ref.rotate(q, pos.long(), freqs(D)), F32)


def test_rope_more_than_the_cache_holds():
    """Tensors of 278 MB, which go past the Infinity Cache, bit for bit as in two halves."""
    note("rope, 278 MB")
    S = 17001
    q, k = (torch.randn(1, S, H, 128, device=DEV).bfloat16().transpose(1, 2) for H in (28, 4))
    pos = torch.arange(S, device=DEV) + 7
    w = (1 + 0.1 * torch.randn(128, device=DEV)).bfloat16()
    inv = freqs(128).to(DEV)
    whole = qk_norm_rope(q, k, pos, inv, w, w)
    for part in (slice(0, 8000), slice(8000, S)):
        half = qk_norm_rope(q[:, :, part], k[:, :, part], pos[part], inv, w, w)
        for a, b in zip(whole, half):
            assert torch.equal(a[:, :, part], b)


def test_rope_far_positions_and_odd_values():
    """Angles of positions up to 2^31; rows of zeros, infinities and NaN stay where they are."""
    note("rope far")
    q = torch.randn(1, 2, 4, 128, generator=gen(2))
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1])
    got = qk_norm_rope(q.to(DEV), q.to(DEV), pos.to(DEV), freqs(128).to(DEV))
    # fp64 holds these angles to 2^31 * 2^-53 turns: far below fp32's step.
    within(got[0], *ref.rotate(q, pos, freqs(128)), F32)
    q = torch.randn(1, 3, 5, 64, generator=gen(3)).bfloat16()
    q[0, 0, 1] = 0
    q[0, 1, 2, 7] = math.inf
    q[0, 2, 3, 9] = math.nan
    w = torch.ones(64).bfloat16()
    pos = torch.arange(5)
    got = qk_norm_rope(q.to(DEV), q.to(DEV), pos.to(DEV), freqs(64).to(DEV), w.to(DEV))[0].cpu()
    bad = ~torch.isfinite(got.float()).all(-1)
    assert bad.nonzero().tolist() == [[0, 1, 2], [0, 2, 3]]
    assert bool((got[0, 0, 1] == 0).all())


# ---------------------------------------------------------------- writes

def make_cache(pages, page, Hk, D, layout, dtype, g, fill=None):
    shape = (pages, page, Hk, D) if layout == "NHD" else (pages, Hk, page, D)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if fill is not None:
        k.fill_(fill)
        v.fill_(fill)
    return k, v


def stored(cache, rows, slots, layout):
    """The cache with rows at their slots (out of place)."""
    page = cache.shape[1 if layout == "NHD" else 2]
    out = cache.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < cache.shape[0] * page:
            if layout == "NHD":
                out[s // page, s % page] = rows[t]
            else:
                out[s // page, :, s % page] = rows[t]
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("T,Hk,D,page", [(1, 4, 128, 16), (37, 1, 64, 1), (513, 8, 128, 24),
                                         (64, 3, 80, 7), (200, 16, 64, 128), (9, 2, 33, 5)])
def test_write_puts_rows_in_their_slots(T, Hk, D, page, layout, dtype):
    note("write", T, Hk, D, page, layout, dtype)
    g = gen(T)
    pages = -(-T // page) + 3
    k, v = (torch.randn(T, Hk, D, generator=g).to(dtype) for _ in range(2))
    kc, vc = make_cache(pages, page, Hk, D, layout, dtype, g)
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 4:
        slots[1], slots[2], slots[T - 1] = -1, pages * page, -(2 ** 62)
    kd, vd = kc.to(DEV), vc.to(DEV)
    write_paged_kv(k.to(DEV), v.to(DEV), kd, vd, slots.to(DEV), kv_layout=layout)
    torch.cuda.synchronize()
    assert torch.equal(kd.cpu(), stored(kc, k, slots, layout))
    assert torch.equal(vd.cpu(), stored(vc, v, slots, layout))


def test_write_strided_rows_and_caches():
    """A prefill's (1, Hk, S, D) tensors, and caches that share one allocation."""
    note("write strided")
    g = gen(8)
    S, Hk, D, page, pages = 50, 4, 64, 16, 6
    k, v = (torch.randn(1, Hk, S, D, generator=g).bfloat16() for _ in range(2))
    both = torch.randn(pages, 2, page, Hk, D, generator=g).bfloat16()
    slots = torch.randperm(pages * page, generator=g)[:S]
    bd = both.to(DEV)
    write_paged_kv(k.to(DEV)[0].transpose(0, 1), v.to(DEV)[0].transpose(0, 1), bd[:, 0], bd[:, 1],
                   slots.to(DEV))
    assert torch.equal(bd[:, 0].cpu(), stored(both[:, 0], k[0].transpose(0, 1), slots, "NHD"))
    assert torch.equal(bd[:, 1].cpu(), stored(both[:, 1], v[0].transpose(0, 1), slots, "NHD"))
    # rows and caches that start at odd elements
    flat = torch.zeros(pages * page * Hk * D + 1, dtype=BF16, device=DEV)
    kc = flat[1:].view(pages, page, Hk, D)
    vc = torch.zeros(pages, page, Hk, D + 3, dtype=BF16, device=DEV)[..., :D]
    kd, vd = (x.to(DEV)[0].transpose(0, 1) for x in (k, v))
    write_paged_kv(kd, vd, kc, vc, slots.to(DEV))
    zero = torch.zeros(pages, page, Hk, D, dtype=BF16)
    assert torch.equal(kc.cpu(), stored(zero, k[0].transpose(0, 1), slots, "NHD"))
    assert torch.equal(vc.cpu(), stored(zero, v[0].transpose(0, 1), slots, "NHD"))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,Hq,Hk,D,rot,axes,norm,page,layout", [
    (1, 28, 4, 128, 128, 1, True, 16, "NHD"), (130, 32, 8, 128, 128, 1, True, 64, "HND"),
    (33, 8, 1, 64, 64, 3, False, 12, "NHD"), (16, 5, 5, 128, 64, 1, True, 1, "HND"),
    (7, 40, 2, 96, 96, 1, True, 5, "NHD"), (300, 2, 2, 256, 256, 1, True, 32, "NHD"),
    (1538, 3, 2, 128, 128, 3, True, 16, "HND"), (1601, 2, 1, 64, 32, 1, False, 7, "NHD")])
def test_rope_to_cache(T, Hq, Hk, D, rot, axes, norm, page, layout, dtype):
    """Queries and stored keys are those of the plain form, values are copied, other rows stay."""
    note("rope to cache", T, Hq, Hk, D, rot, axes, norm, page, layout, dtype)
    g = gen(T + D)
    q, k, v = (torch.randn(T, H, D, generator=g).to(dtype) for H in (Hq, Hk, Hk))
    pages = -(-T // page) + 2
    kc, vc = make_cache(pages, page, Hk, D, layout, dtype, g)
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 4:
        slots[3], slots[4] = -1, pages * page
    pos = torch.randint(0, 100000, (axes, T), generator=g)
    third = rot // 6
    sections = [rot // 2 - 2 * third, third, third] if axes == 3 else None
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None
              for _ in range(2))
    to = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    kd, vd = to(kc), to(vc)
    got = qk_norm_rope_to_cache(to(q), to(k), to(v), kd, vd, to(slots),
                                to(pos if axes > 1 else pos[0]), to(freqs(rot)), to(qw), to(kw),
                                mrope_section=sections, kv_layout=layout)
    torch.cuda.synchronize()
    p = (pos if axes > 1 else pos[0]).unsqueeze(-1)
    within(got, *ref.rotate(q, p, freqs(rot), qw, sections=sections), dtype)
    assert torch.equal(vd.cpu(), stored(vc, v, slots, layout))
    want, slack = ref.rotate(k, p, freqs(rot), kw, sections=sections)
    rows, before = ref.cache_rows(kd.cpu(), layout), ref.cache_rows(kc, layout)
    real = (slots >= 0) & (slots < pages * page)
    within(rows[slots[real]], want[real], slack[real], dtype)
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[real]] = False
    assert torch.equal(rows[rest], before[rest])


def test_rope_to_cache_same_position_on_every_axis():
    note("rope to cache, one position")
    g = gen(12)
    q, k, v = (torch.randn(4, 2, 64, generator=g).to(DEV) for _ in range(3))
    caches = [torch.zeros(1, 16, 2, 64, device=DEV) for _ in range(4)]
    slots, pos = torch.arange(4, device=DEV), torch.tensor([5, 900, 31, 7], device=DEV)
    a = qk_norm_rope_to_cache(q, k, v, *caches[:2], slots, pos, freqs(64).to(DEV))
    b = qk_norm_rope_to_cache(q, k, v, *caches[2:], slots, pos, freqs(64).to(DEV),
                              mrope_section=[16, 8, 8])
    assert torch.equal(a, b) and torch.equal(caches[0], caches[2])


# ---------------------------------------------------------------- decode attention

def decode_case(lens, Hq, Hk, D, page, layout, dtype, seed=0, scale=None, extra=3, junk=True,
                q_scale=1.0):
    """Inputs with pages in random order; rows that no request holds are NaN."""
    g = gen(seed)
    N = len(lens)
    width = -(-max(max(lens), 1) // page) + extra
    held = [-(-max(n, 0) // page) for n in lens]
    pages = sum(held) + 2
    kc, vc = make_cache(pages, page, Hk, D, layout, dtype, g, math.nan if junk else None)
    ids = torch.randperm(pages, generator=g).int()
    table = torch.full((N, width), -1, dtype=torch.int32)
    at = 0
    for n, L in enumerate(lens):
        table[n, :held[n]] = ids[at:at + held[n]]
        at += held[n]
        for t0 in range(held[n]):
            m = min(page, L - t0 * page)
            for c in (kc, vc):
                rows = torch.randn(Hk, m, D, generator=g).to(dtype)
                if layout == "NHD":
                    c[int(table[n, t0]), :m] = rows.transpose(0, 1)
                else:
                    c[int(table[n, t0]), :, :m] = rows
    q = (q_scale * torch.randn(N, Hq, D, generator=g)).to(dtype)
    return q, kc, vc, table, torch.tensor(lens, dtype=torch.int32)


def run_decode(q, kc, vc, table, lens, layout, **kw):
    out = paged_decode_attention(*(t.to(DEV) for t in (q, kc, vc, table, lens)), kv_layout=layout,
                                 **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lens,Hq,Hk,D,page,layout", [
    ([1], 28, 4, 128, 16, "NHD"), ([2081], 28, 4, 128, 16, "NHD"),
    ([0, 1, 15, 16, 17, 31, 32, 33], 8, 2, 64, 16, "NHD"),
    ([127, 128, 129, 0, 257, 1000], 12, 12, 128, 64, "HND"),
    ([700, 3, 1, 64, 63, 65], 40, 2, 128, 24, "NHD"),
    ([300, 90], 16, 1, 64, 1, "HND"), ([45, 800, 7], 4, 4, 128, 12, "NHD"),
    ([100, 0, 33], 6, 2, 96, 16, "NHD"), ([77, 200], 4, 1, 256, 32, "HND"),
    ([50, 5], 3, 3, 33, 16, "NHD"), ([0], 4, 4, 64, 16, "NHD"),
    ([5000, 11], 17, 1, 64, 128, "NHD"), ([400], 32, 1, 128, 48, "HND")])
def test_decode_matches_the_plain_form(lens, Hq, Hk, D, page, layout, dtype):
    note("paged decode", lens, Hq, Hk, D, page, layout, dtype)
    case = decode_case(lens, Hq, Hk, D, page, layout, dtype, seed=sum(lens) + D)
    out = run_decode(*case, layout)
    within(out, *ref.decode(*case, layout), dtype)
    for n, L in enumerate(lens):
        if L == 0:
            assert bool((out[n] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_decode_many_requests(dtype):
    """More requests than work-groups' threads, lengths of every size, repeated bit for bit."""
    note("paged decode, 300 requests", dtype)
    g = gen(9)
    lens = torch.exp(6.5 * torch.rand(300, generator=g)).int().tolist()
    lens[0], lens[17], lens[299] = 0, 0, 900
    case = decode_case(lens, 4, 2, 64, 16, "NHD", dtype, seed=5)
    out = run_decode(*case, "NHD")
    within(out, *ref.decode(*case, "NHD"), dtype)
    assert torch.equal(out, run_decode(*case, "NHD"))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,page,extra", [(64, 16, 0), (128, 24, 0), (128, 16, 6), (64, 5, 20)])
def test_decode_many_short_requests(D, page, extra, dtype):
    """More segments than the GPU has CUs, tables of few pages: one wave or eight to a segment."""
    note("paged decode, short requests", D, page, extra, dtype)
    g = gen(D + page)
    lens = torch.randint(0, 90, (140,), generator=g).tolist()
    case = decode_case(lens, 6, 2, D, page, "NHD", dtype, seed=page, extra=extra)
    bad = case[3].clone()
    out = run_decode(*case, "NHD")
    want, slack = ref.decode(*case, "NHD")
    within(out, want, slack, dtype)
    n = int(torch.tensor(lens).argmax())
    bad[n, 0] = -1
    out = run_decode(*case[:3], bad, case[4], "NHD").cpu()
    assert bool(torch.isnan(out[n]).all())
    keep = torch.arange(140) != n
    within(out[keep], want[keep], slack[keep], dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_forms_by_table_width(dtype):
    """The same requests under tables of other widths take other forms of the kernel: one wave a
    segment, eight, or the keys dealt out and merged, which also reads values past the caches."""
    note("paged decode, forms", dtype)
    q, kc, vc, table, lens = decode_case([40, 0, 17, 64] * 70, 4, 2, 64, 16, "NHD", dtype, seed=8)
    want, slack = ref.decode(q, kc, vc, table, lens, "NHD")
    for width in (4, 40, 64, 400, 9000):
        wide = torch.full((280, width), -1, dtype=torch.int32)
        wide[:, :4] = table[:, :4]
        within(run_decode(q, kc, vc, wide, lens, "NHD"), want, slack, dtype)


@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F32), (80, BF16)])
def test_decode_split_sequence(D, dtype):
    """One long sequence over many work-groups, keys of great weight at their borders."""
    note("paged decode, split", D, dtype)
    L, Hq, Hk, page = 20011, 7, 1, 16
    q, kc, vc, table, lens = decode_case([L], Hq, Hk, D, page, "NHD", dtype, seed=3)
    for pos in (0, 127, 128, 4097, L - 1):
        kc[int(table[0, pos // page]), pos % page, 0] = 2.0 * q[0].mean(0)
    out = run_decode(q, kc, vc, table, lens, "NHD", sm_scale=0.3)
    within(out, *ref.decode(q, kc, vc, table, lens, "NHD", 0.3), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [6, 32, 40, 96, 160, 256])
def test_decode_split_of_any_head_dim(D, dtype):
    """Partial rows of several work-groups, merged in pieces of a row or whole rows."""
    note("paged decode, split", D, dtype)
    case = decode_case([4003, 1], 5, 1, D, 12, "HND", dtype, seed=D)
    out = run_decode(*case, "HND")
    within(out, *ref.decode(*case, "HND"), dtype)
    assert torch.equal(out, run_decode(*case, "HND"))


def test_decode_agrees_with_the_contiguous_cache():
    """One request on consecutive pages is what single_decode_with_kv_cache computes."""
    note("paged decode vs single")
    g = gen(6)
    Hq, Hk, L, D, page = 28, 4, 3000, 128, 16
    q = torch.randn(Hq, D, generator=g).bfloat16().to(DEV)
    pages = -(-L // page)
    kc, vc = (torch.randn(pages, page, Hk, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    a = paged_decode_attention(q[None], kc, vc, table,
                               torch.tensor([L], dtype=torch.int32, device=DEV))[0]
    b = single_decode_with_kv_cache(q, kc.flatten(0, 1)[:L], vc.flatten(0, 1)[:L])
    d = (a.float() - b.float()).abs()
    assert float(d.max()) <= 1e-2 and float(d.mean()) <= 1e-3


@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16), (128, F32), (48, BF16)])
def test_decode_pages_that_cannot_be_read(D, dtype):
    """A page outside the cache, or a length past the table, makes that request's rows NaN and
    leaves the others as they are; a page that its keys do not need is not looked at."""
    note("paged decode, bad pages", D, dtype)
    lens = [300, 40, 2000, 33, 0, 16]
    q, kc, vc, table, l = decode_case(lens, 4, 2, D, 16, "NHD", dtype, seed=D, extra=1)
    want, slack = ref.decode(q, kc, vc, table, l, "NHD")
    table, l = table.clone(), l.clone()
    table[0, 18] = -1                      # its last page
    table[2, 5] = kc.shape[0]              # the first id behind the cache
    table[4, :] = 2 ** 31 - 1              # no key: not looked at
    table[1, 3:] = -(2 ** 31)              # behind its keys
    l[3] = table.shape[1] * 16 + 1         # longer than its table
    out = run_decode(q, kc, vc, table, l, "NHD").cpu()
    for n in (0, 2, 3):
        assert bool(torch.isnan(out[n]).all()), n
    good = [1, 4, 5]
    within(out[good], want[good], slack[good], dtype)
    l[5] = -7                              # counts as 0
    assert bool((run_decode(q, kc, vc, table, l, "NHD")[5] == 0).all())


@pytest.mark.parametrize("D,dtype", [(128, F32), (72, F32), (128, BF16), (64, F16)])
def test_decode_values_that_are_not_finite(D, dtype):
    """Infinite scores and values: as the formula has it, row by row."""
    note("paged decode, not finite", D, dtype)
    lens = [40, 300, 64, 20, 70]
    q, kc, vc, table, l = decode_case(lens, 2, 2, D, 16, "NHD", dtype, seed=2)
    def row(c, n, t): return c[int(table[n, t // 16]), t % 16]  # noqa: E704
    row(vc, 0, 7)[0, 3] = math.inf         # one value of head 0
    row(kc, 1, 150)[1] = math.nan          # a score of head 1
    row(kc, 2, 5)[0, 0] = math.inf         # +inf or -inf score of head 0, by the query's sign
    q[2, 0, 0] = -1.0                      # -inf: the key weighs nothing
    q[4] = 0
    q[4, :, 0] = 1.0
    for t in range(70):
        row(kc, 4, t)[0, 0] = -math.inf    # every score of head 0 is -inf: 0/0
    out = run_decode(q, kc, vc, table, l, "NHD").cpu()
    want, size = torch.zeros(5, 2, D).double(), torch.zeros(5, 2, D).double()
    for n, L in enumerate(lens):
        t = torch.arange(L)
        at = table[n].long()[t // 16] * 16 + t % 16
        k, v = (ref.cache_rows(c, "NHD")[at].double() for c in (kc, vc))
        s = (k * q[n].double()).sum(-1) / math.sqrt(D)
        p = torch.softmax(s, 0)
        want[n] = (p[..., None] * v).sum(0)
        size[n] = (p[..., None] * v.abs()).sum(0)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.isinf(out), torch.isinf(want))
    # Where a value is infinite, 16-bit types hold the weights to one rounding; fp32's own
    # roundings (scores of size below 8, 300 terms) stay under 2^-13 of the values' size.
    ok = torch.isfinite(want)
    u = 0.0 if dtype == F32 else ref.HALF_STEP[dtype]
    room = ref.rounded(want, (u + 2.0 ** -13) * size, dtype)
    assert bool(((out.double() - want).abs() <= room)[ok].all())


@pytest.mark.parametrize("D,dtype", [(128, F32), (72, F32), (128, BF16), (64, F16), (64, F32)])
@pytest.mark.parametrize("lens", [[1, 17, 33, 45, 130], [20, 700], [5000], [3] * 300])
def test_decode_infinite_values_by_masked_and_tiny_weights(lens, D, dtype):
    """An infinite value of the last key is not met by the zero weights of the places behind it,
    and one whose weight is too small for fp32 is infinite all the same."""
    note("paged decode, infinite values", lens[:5], D, dtype)
    q, kc, vc, table, l = decode_case(lens, 2, 2, D, 16, "NHD", dtype, seed=3, extra=0)
    def row(c, n, t): return c[int(table[n, t // 16]), t % 16]  # noqa: E704
    q[:] = 0
    q[:, :, 0] = 1.0
    high = []  # keys far above the others: 800 in their score's exponent of two
    for n, L in enumerate(lens):
        row(vc, n, L - 1)[0, 3] = math.inf
        row(vc, n, 0)[1, 5] = -math.inf
        high.append(L // 2)
        row(kc, n, L // 2)[1, 0] = 560 * math.sqrt(D)
    out = run_decode(q, kc, vc, table, l, "NHD").cpu()
    for n, L in enumerate(lens):
        v = ref.cache_rows(vc, "NHD")[table[n].long()[torch.arange(L) // 16] * 16 +
                                      torch.arange(L) % 16].double()
        k = ref.cache_rows(kc, "NHD")[table[n].long()[torch.arange(L) // 16] * 16 +
                                      torch.arange(L) % 16].double()
        p = torch.softmax((k * q[n].double()).sum(-1) / math.sqrt(D), 0)
        want = (p[..., None] * v).sum(0)
        assert want[0, 3] == math.inf and want[1, 5] == -math.inf
        assert torch.equal(torch.isnan(out[n]), torch.isnan(want))
        assert torch.equal(torch.isinf(out[n]), torch.isinf(want))
        # Scores of size below 8 have weights as in the test above; head 1's are one key's value
        # and others of at most 2^-24 (fp16's smallest weight) each.
        size = (p[..., None] * v.abs()).sum(0)
        u = 0.0 if dtype == F32 else ref.HALF_STEP[dtype]
        tiny = L * 2.0 ** -24 * v[torch.isfinite(v)].abs().max() if dtype == F16 else 0.0
        ok = torch.isfinite(want)
        room = ref.rounded(want, (u + (300 + 2 * L) * 2.0 ** -22) * size + tiny, dtype)
        assert bool(((out[n].double() - want).abs() <= room)[ok].all())


def row_of(c, table, n, t, page):
    return c[int(table[n, t // page]), t % page]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lens,Hk,D,page", [([4101], 1, 128, 16), ([4101, 77], 2, 64, 24),
                                            ([500], 2, 128, 16), ([250] * 150, 2, 64, 16),
                                            ([900], 1, 72, 16)])
def test_decode_small_weights_beside_a_great_one(lens, Hk, D, page, dtype):
    """One key far above the others (an attention sink) whose value is 0: what the others' small
    weights add up to is all of the output, in every form of the kernel."""
    note("paged decode, sink", lens[:3], Hk, D, page, dtype)
    N, g = len(lens), gen(D + page)
    _, kc, vc, table, l = decode_case(lens, 2 * Hk, Hk, D, page, "NHD", dtype, seed=D, extra=0)
    q = torch.zeros(N, 2 * Hk, D, dtype=dtype)
    q[:, :, 0] = 1.0                       # a score is feature 0 of its key, exactly
    for n, L in enumerate(lens):
        for t in range(L):
            row_of(kc, table, n, t, page)[:, 0] = (0.3 * torch.randn(Hk, generator=g)).to(dtype)
    for gap, size in ((12.0, 1.0), (16.0, 1.0), (17.0, 1.0), (18.0, 1.0), (24.0, 500.0)):
        k, v = kc.clone(), (size * (vc.abs() + 0.125)).to(dtype)
        for n, L in enumerate(lens):
            row_of(k, table, n, L // 3, page)[:, 0] = gap
            row_of(v, table, n, L // 3, page)[:] = 0
        out = run_decode(q, k, v, table, l, "NHD", sm_scale=1.0)
        want, slack = torch.zeros(N, 2 * Hk, D).double(), torch.zeros(N, 2 * Hk, D).double()
        for n, L in enumerate(lens):
            t = torch.arange(L)
            at = table[n].long()[t // page] * page + t % page
            K, V = (ref.cache_rows(c, "NHD")[at].double().repeat_interleave(2, 1) for c in (k, v))
            p = torch.softmax(K[..., 0], 0)
            want[n] = (p[..., None] * V).sum(0)
            # Roundings of 2^-24 each: scores of size below 25 in units of log2(e) (three for the
            # scaled score, one for the difference, one step of exp2: below 200 in a weight and in
            # the weights' sum together) and sums of at most 300 after one another (32 products of
            # an instruction times 8 steps, the waves' and the work-groups' merges), of weights
            # and of values: below 1000, 2^-14.  16-bit types' parts add at most 2^-18 of a weight
            # and, in fp16, 2^-44 of the greatest one.
            slack[n] = 2.0 ** -14 * want[n]
            if dtype == F16:
                slack[n] += L * 2.0 ** -44 * V.max()
        within(out, want, slack, dtype)


def test_decode_scores_whose_steps_are_large():
    """Scores of 2^27, whose neighbours lie 16 apart in powers of two: any weights of equal
    values give that value."""
    note("paged decode, large scores")
    L, N = 300, 6                          # eight waves of 32 keys: the first has two steps
    for dtype in (F16, BF16, F32):
        q, kc, vc, table, l = decode_case([L] * N, 1, 1, 64, 16, "NHD", dtype, seed=1, extra=0)
        q[:], kc[:], vc[:] = 0, 0, 1.0
        q[:, 0, 0], q[:, 0, 1] = 2048.0, 1.0
        for n in range(N):
            for t in range(L):
                row_of(kc, table, n, t, 16)[0, 0] = 4096.0
                row_of(kc, table, n, t, 16)[0, 1] = float(n + t // 256)
        out = run_decode(q, kc, vc, table, l, "NHD", sm_scale=16 / 1.4426950408889634)
        # Both sums add the same 300 weights, each off by 2^-16 at most: below half a step of bf16.
        assert bool(((out.float() - 1).abs() <= 2.0 ** -9).all()), (dtype, out[:, 0, 0])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lens,Hq,D,page", [([3000], 8, 128, 16), ([700, 33, 2100], 4, 64, 24),
                                            ([300, 64], 8, 128, 16), ([60] * 150, 4, 64, 16),
                                            ([90, 500], 6, 40, 16)])
def test_decode_finite_outputs_beside_others(lens, Hq, D, page, dtype):
    """An infinite value, a NaN in a value or in a query reaches the outputs that the formula has
    it in; all others stay as they are, bit for bit."""
    note("paged decode, beside others", lens[:3], Hq, D, page, dtype)
    q, kc, vc, table, l = decode_case(lens, Hq, 2, D, page, "NHD", dtype, seed=D, extra=0)
    clean = run_decode(q, kc, vc, table, l, "NHD")
    v, G = vc.clone(), Hq // 2
    for n, L in enumerate(lens):
        row_of(v, table, n, L // 2, page)[0, 3] = math.inf
        row_of(v, table, n, L - 1, page)[0, 9] = -math.inf
        row_of(v, table, n, L // 3, page)[1, 5] = math.nan
    want = clean.clone()
    want[:, :G, 3], want[:, :G, 9] = math.inf, -math.inf
    out = run_decode(q, kc, v, table, l, "NHD")
    assert bool(torch.isnan(out[:, G:, 5]).all())
    out[:, G:, 5] = want[:, G:, 5]
    assert torch.equal(out, want)
    q[:, 1, 7] = math.nan
    out = run_decode(q, kc, vc, table, l, "NHD")
    assert bool(torch.isnan(out[:, 1]).all())
    out[:, 1] = clean[:, 1]
    assert torch.equal(out, clean)


def test_decode_strided_views():
    """Caches in one allocation, queries and tables cut from wider ones."""
    note("paged decode, strided")
    q, kc, vc, table, lens = decode_case([100, 37, 260], 4, 2, 128, 16, "NHD", BF16, seed=4)
    both = torch.stack([kc, vc], 1).to(DEV)
    wide_q = torch.randn(3, 9, 128).bfloat16().to(DEV)
    wide_q[:, 2:6] = q.to(DEV)
    wide_t = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide_t[:, :table.shape[1]] = table.to(DEV)
    a = paged_decode_attention(wide_q[:, 2:6], both[:, 0], both[:, 1],
                               wide_t[:, :table.shape[1]], lens.to(DEV))
    assert torch.equal(a, run_decode(q, kc, vc, table, lens, "NHD"))
    # unaligned rows take another kernel
    odd = torch.zeros(*kc.shape[:3], 129, dtype=BF16, device=DEV)
    ko, vo = odd[..., 1:], torch.zeros_like(odd)[..., 1:]
    ko.copy_(kc)
    vo.copy_(vc)
    b = paged_decode_attention(q.to(DEV), ko, vo, table.to(DEV), lens.to(DEV))
    within(b, *ref.decode(q, kc, vc, table, lens, "NHD"), BF16)


@pytest.mark.parametrize("D", [128, 40])
def test_decode_offsets_past_32_bits(D):
    """Pages 2^21 elements apart: the last ones start beyond 2^32 elements."""
    note("paged decode, far pages", D)
    q, kc, vc, table, lens = decode_case([150, 40], 4, 2, D, 16, "NHD", BF16, seed=7)
    far, stride = 2100, 1 << 21
    storage = torch.empty(far * stride, dtype=BF16, device=DEV)
    ids = torch.arange(far - kc.shape[0], far)
    views = []
    for i, c in enumerate((kc, vc)):
        view = storage[i * 65536:].as_strided((far, *c.shape[1:]), (stride, *c.stride()[1:]))
        view[ids.to(DEV)] = c.to(DEV)
        views.append(view)
    moved = torch.where(table >= 0, table + (far - kc.shape[0]), table)
    out = paged_decode_attention(q.to(DEV), *views, moved.int().to(DEV), lens.to(DEV))
    assert torch.equal(out, run_decode(q, kc, vc, table, lens, "NHD"))
    rows = torch.randn(3, 2, D).bfloat16().to(DEV)
    slots = torch.tensor([(far - 1) * 16 + 3, 5, -1], device=DEV)
    write_paged_kv(rows, rows, *views, slots)
    assert torch.equal(views[0][far - 1, 3], rows[0]) and torch.equal(views[1][0, 5], rows[1])


def test_decode_streams_and_two_graphs():
    """On a side stream, and captured twice (each graph with a workspace of its own), replayed
    in turn with eager calls between."""
    note("paged decode, graphs")
    cases = [[t.to(DEV) for t in decode_case(lens, 28, 4, 128, 16, "NHD", BF16, seed=s)]
             for s, lens in ((1, [700, 30, 0, 1500]), (2, [90, 2500]))]
    want = [paged_decode_attention(*c) for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [paged_decode_attention(*c) for c in cases]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_decode_attention(*c))
        graphs.append(graph)
    for trial in range(3):
        for c in cases:
            c[4].sub_(trial).clamp_(min=0)   # other lengths in the same tensors
        for graph in graphs:
            graph.replay()
        eager = [paged_decode_attention(*c) for c in cases]
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    """What only shows with tensors on the GPU: other devices, and gradients."""
    note("refusals")
    g = gen(3)
    q, k, v = (torch.randn(5, 2, 64, generator=g, device="cpu").to(DEV) for _ in range(3))
    kc, vc = (torch.zeros(2, 16, 2, 64, device=DEV) for _ in range(2))
    slots, pos, inv = torch.arange(5, device=DEV), torch.arange(5, device=DEV), freqs(64).to(DEV)
    ok = (q, k, v, kc, vc, slots, pos, inv)
    for i in range(1, 8):
        bad = list(ok)
        bad[i] = bad[i].cpu()
        with pytest.raises(ValueError, match="tensors on"):
            qk_norm_rope_to_cache(*bad)
    w = torch.ones(64, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no backward"):
        qk_norm_rope_to_cache(*ok, w, w)
    with torch.no_grad():
        qk_norm_rope_to_cache(*ok, w, w)
    sparse = torch.zeros(5, 2, 128, device=DEV, requires_grad=True)[..., ::2]  # copied
    with pytest.raises(NotImplementedError, match="no backward"):
        write_paged_kv(k, sparse, kc, vc, slots)
    with pytest.raises(NotImplementedError, match="no backward"):
        qk_norm_rope_to_cache(q, sparse, v, kc, vc, slots, pos, inv)
    table, lens = torch.zeros(5, 1, dtype=torch.int32, device=DEV), torch.full(
        (5,), 3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="tensors on"):
        paged_decode_attention(q, kc, vc, table.cpu(), lens)
    with pytest.raises(NotImplementedError, match="no backward"):
        paged_decode_attention(q.requires_grad_(), kc, vc, table, lens)
    with pytest.raises(NotImplementedError, match="head_dim 320"):
        paged_decode_attention(torch.zeros(1, 2, 320, device=DEV),
                               *(torch.zeros(1, 16, 2, 320, device=DEV) for _ in range(2)),
                               table[:1], lens[:1])
    # nothing to do
    empty = qk_norm_rope(torch.zeros(1, 2, 0, 64, device=DEV), torch.zeros(1, 2, 0, 64, device=DEV),
                         torch.zeros(1, 0, dtype=torch.int64, device=DEV), inv)
    assert empty[0].shape == (1, 2, 0, 64)
    write_paged_kv(k[:0], v[:0], kc, vc, slots[:0])
    assert paged_decode_attention(q.detach()[:0], kc, vc, table[:0], lens[:0]).shape == (0, 2, 64)


def test_rotation_has_no_backward():
    """Each tensor of the rotation that wants a gradient is refused; without grad mode it runs."""
    note("rotation, gradients")
    g = gen(4)
    q, k = (torch.randn(1, 2, 5, 64, generator=g).to(DEV) for _ in range(2))
    w = torch.ones(64, device=DEV)
    args = [q, k, torch.arange(5, device=DEV), freqs(64).to(DEV), w, w]
    want = qk_norm_rope(*args)
    for i in (0, 1, 3, 4, 5):
        some = [a.clone().requires_grad_() if i == j else a for j, a in enumerate(args)]
        with pytest.raises(NotImplementedError, match="no backward"):
            qk_norm_rope(*some)
        with torch.no_grad():
            got = qk_norm_rope(*some)
        assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))


def test_writes_are_seen_by_autograd():
    """A cache that a graph saved for its backward pass and that a call wrote is not used by it."""
    note("versions")
    k = torch.ones(5, 2, 64, device=DEV)
    kc, vc = (torch.zeros(2, 16, 2, 64, device=DEV) for _ in range(2))
    slots, table = torch.arange(5, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    for call in (lambda: write_paged_kv(k, k, kc, vc, slots),
                 lambda: qk_norm_rope_to_cache(k, k, k, kc, vc, slots, slots, freqs(64).to(DEV))):
        loss = (vc * w).sum()
        with torch.no_grad():
            call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    lens = torch.ones(1, dtype=torch.int32, device=DEV)
    before = table._version
    paged_kv_plan(lens, lens, table, lens, 16, 1)
    assert table._version > before
    with torch.inference_mode():
        kc = torch.zeros(2, 16, 2, 64, device=DEV)
        write_paged_kv(k, k, kc, kc.clone(), slots)
        step = paged_kv_plan(lens, lens, table, lens, 16, 3)
        assert all(t.is_inference() and t.is_contiguous() for t in step)
        assert bool((kc[0, :5] == 1).all())


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype,layout", [(BF16, "NHD"), (F32, "HND")])
def test_prompts_then_generated_tokens(dtype, layout):
    """Two prompts of different lengths, then five generated tokens with a third request joining:
    plan, rotation, writes and attention as a program runs them, against one sequence at a
    time in 64 bits."""
    note("steps", dtype, layout)
    g = gen(20)
    Hq, Hk, D, page, N, width = 8, 2, 64, 16, 3, 8
    pages = 20
    shape = (pages, page, Hk, D) if layout == "NHD" else (pages, Hk, page, D)
    kc, vc = (torch.full(shape, math.nan, dtype=dtype, device=DEV) for _ in range(2))
    table = torch.full((N, width), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pages, generator=g).int().to(DEV)
    lens = torch.zeros(N, dtype=torch.int32, device=DEV)
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g) for _ in range(2))
    qw, kw = qw.to(dtype), kw.to(dtype)
    inv = freqs(D)
    seen = [([], []) for _ in range(N)]      # keys and values of each request, in 64 bits
    head = torch.zeros(1, dtype=torch.int32, device=DEV)
    for step, new in enumerate([[37, 16, 0], [1, 1, 0], [1, 1, 50], [1, 1, 1], [1, 0, 1],
                                [1, 1, 1]]):
        T = sum(new)
        q, k, v = (torch.randn(T, H, D, generator=g).to(dtype) for H in (Hq, Hk, Hk))
        p = paged_kv_plan(lens, torch.tensor(new, dtype=torch.int32, device=DEV), table, free,
                          page, T + 3, head)
        head, lens = (head + p.pages_taken).int(), p.kv_lens
        slots, pos = p.slot_mapping[:T], p.positions[:T]
        dq, dk, dv = q.to(DEV), k.to(DEV), v.to(DEV)
        if step == 0:                        # prompts: rotated as (1, H, T, D), then written
            rq, rk = qk_norm_rope(*(x.transpose(0, 1)[None] for x in (dq, dk)), pos, inv.to(DEV),
                                  qw.to(DEV), kw.to(DEV))
            rq = rq[0].transpose(0, 1)
            write_paged_kv(rk[0].transpose(0, 1), dv, kc, vc, slots, kv_layout=layout)
        else:
            rq = qk_norm_rope_to_cache(dq, dk, dv, kc, vc, slots, pos, inv.to(DEV), qw.to(DEV),
                                       kw.to(DEV), kv_layout=layout)
        last = torch.tensor([max(sum(new[:i + 1]) - 1, 0) for i in range(N)], device=DEV)
        out = paged_decode_attention(rq[last], kc, vc, table, lens, kv_layout=layout).cpu()
        at = 0
        for n in range(N):
            L0 = len(seen[n][0])
            for t in range(new[n]):
                key, _ = ref.rotate(k[at], torch.tensor(L0 + t), inv, kw)
                seen[n][0].append(key)
                seen[n][1].append(v[at].double())
                at += 1
            assert int(lens[n]) == len(seen[n][0])
            if not new[n]:
                continue
            query, _ = ref.rotate(q[at - 1], torch.tensor(L0 + new[n] - 1), inv, qw)
            K, V = (torch.stack(x).repeat_interleave(Hq // Hk, 1) for x in seen[n])
            s = (K * query).sum(-1) / math.sqrt(D)
            w = torch.softmax(s, 0)
            want = (w[..., None] * V).sum(0)
            # The queries and the cached keys are rounded to the type: a score moves by at most
            # 2u (1 + u) of the sum of its products' sizes, a weight by that factor, as does the
            # weights' sum; then the output's rounding.  fp32's own roundings: as in ref.decode.
            u = ref.HALF_STEP[dtype]
            move = ((K * query).abs().sum(-1) / math.sqrt(D)).max() * (2 * u + (D + 40) * 2.0 ** -24)
            rel = 2 * math.expm1(float(move)) + 2.0 ** -14
            within(out[n], want, rel * (w[..., None] * V.abs()).sum(0), dtype)


def test_image_prompt_then_generated_tokens():
    """A prompt with an image, rotated over three axes, beside one of text; then generated tokens
    at the positions behind each prompt's last, which for the first are not their indices."""
    note("image prompt")
    g = gen(23)
    dtype, Hq, Hk, D, page, N = F32, 4, 2, 64, 16, 2
    inv, sections = freqs(D), [8, 12, 12]
    at = [torch.cat([torch.arange(5).expand(3, 5),
                     5 + torch.stack([torch.zeros(24).long(), torch.arange(24) // 6,
                                      torch.arange(24) % 6]),
                     11 + torch.arange(7).expand(3, 7)], 1),     # 36 tokens, positions up to 17
          torch.arange(21).expand(3, 21)]
    lens = torch.zeros(N, dtype=torch.int32, device=DEV)
    table = torch.full((N, 4), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(8, generator=g).int().to(DEV)
    head = torch.zeros(1, dtype=torch.int32, device=DEV)
    deltas = torch.zeros(N, dtype=torch.int64, device=DEV)
    kc, vc = (torch.full((8, page, Hk, D), math.nan, dtype=dtype, device=DEV) for _ in range(2))
    K, V = [], []
    for n in range(N):
        S = at[n].shape[1]
        new = torch.zeros(N, dtype=torch.int32, device=DEV)
        new[n] = S
        p = paged_kv_plan(lens, new, table, free, page, S, head)
        head, lens = (head + p.pages_taken).int(), p.kv_lens
        q, k, v = (torch.randn(1, H, S, D, generator=g, dtype=dtype) for H in (Hq, Hk, Hk))
        ids = at[n][:, None].to(DEV)
        _, rk = qk_norm_rope(q.to(DEV), k.to(DEV), ids, inv.to(DEV), mrope_section=sections)
        write_paged_kv(rk[0].transpose(0, 1), v[0].transpose(0, 1).to(DEV), kc, vc, p.slot_mapping)
        deltas[n] = ids.max() + 1 - S
        K.append(ref.rotate(k[0], at[n][:, None], inv, sections=sections)[0].transpose(0, 1))
        V.append(v[0].transpose(0, 1).double())
    assert deltas.tolist() == [18 - 36, 0]
    ones = torch.ones(N, dtype=torch.int32, device=DEV)
    for step in range(3):
        p = paged_kv_plan(lens, ones, table, free, page, N + 2, head)
        head, lens = (head + p.pages_taken).int(), p.kv_lens
        positions = p.positions + deltas[p.request_ids]
        q, k, v = (torch.randn(N + 2, H, D, generator=g, dtype=dtype) for H in (Hq, Hk, Hk))
        rq = qk_norm_rope_to_cache(*(x.to(DEV) for x in (q, k, v)), kc, vc, p.slot_mapping,
                                   positions, inv.to(DEV))
        out = paged_decode_attention(rq[:N], kc, vc, table, lens).cpu()
        for n in range(N):
            pos = int(at[n].max()) + 1 + step

            def turned(x, pos):
                return ref.rotate(x, torch.tensor([pos] * 3)[:, None], inv, sections=sections)[0]

            def attend(pos):
                keys = torch.cat([K[n], turned(k[n], pos)[None]]).repeat_interleave(Hq // Hk, 1)
                s = (keys * turned(q[n], pos)).sum(-1) / math.sqrt(D)
                return keys, torch.softmax(s, 0)

            keys, w = attend(pos)
            K[n] = torch.cat([K[n], turned(k[n], pos)[None]])
            V[n] = torch.cat([V[n], v[n].double()[None]])
            values = V[n].repeat_interleave(Hq // Hk, 1)
            want = (w[..., None] * values).sum(0)
            # The rotation is off by 32 roundings of the pairs' sizes, at most sqrt(2) of the rows'
            # lengths: a score by twice that of their product and ref.decode's 2^-24 (D + 8).
            size = (keys.norm(dim=-1) * q[n].double().norm(dim=-1)).max() / math.sqrt(D)
            move = 2.0 ** -24 * (2 * 32 * math.sqrt(2) + D + 8) * float(size)
            rel = 2 * math.expm1(move) + 2.0 ** -16
            slack = rel * (w[..., None] * values.abs()).sum(0)
            within(out[n], want, slack, dtype)
            if n == 0:                           # and the bare index is another position
                K[n], last = K[n][:-1], K[n][-1:]
                bare = (attend(int(lens[0]) - 1)[1][..., None] * values).sum(0)
                K[n] = torch.cat([K[n], last])
                assert bool(((bare - want).abs() > 100 * slack).any())


@pytest.mark.parametrize("page", [16, 5])
def test_a_whole_step_in_a_graph(page):
    """Plan, rotation, writes and attention of a step in one graph that carries its state on the
    GPU, replayed on a side stream with eager work between, against the same steps run eagerly."""
    note("a step in a graph", page)
    g = gen(31)
    Hq, Hk, D, N, width, pages = 8, 2, 128, 5, 12, 64
    inv = freqs(D).to(DEV)
    qkv = [torch.randn(N, H, D, generator=g).bfloat16().to(DEV) for H in (Hq, Hk, Hk)]
    free = torch.randperm(pages, generator=g).int().to(DEV)
    ones = torch.ones(N, dtype=torch.int32, device=DEV)

    def state():
        return (torch.zeros(N, dtype=torch.int32, device=DEV),
                torch.full((N, width), -1, dtype=torch.int32, device=DEV),
                torch.zeros(1, dtype=torch.int32, device=DEV),
                *(torch.zeros(pages, page, Hk, D, dtype=torch.bfloat16, device=DEV)
                  for _ in range(4)))

    def step(lens, table, head, kc, vc, kc2, vc2):
        q, k, v = qkv
        p = paged_kv_plan(lens, ones, table, free, page, N, head)
        rq = qk_norm_rope_to_cache(q, k, v, kc, vc, p.slot_mapping, p.positions, inv)
        pq, pk = qk_norm_rope(*(x.transpose(0, 1)[None] for x in (q, k)), p.positions, inv)
        write_paged_kv(pk[0].transpose(0, 1), v, kc2, vc2, p.slot_mapping)
        a = paged_decode_attention(rq, kc, vc, table, p.kv_lens)
        b = paged_decode_attention(pq[0].transpose(0, 1), kc2, vc2, table, p.kv_lens)
        lens.copy_(p.kv_lens)
        head.add_(p.pages_taken)
        return a, b

    mine, theirs = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*state())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = step(*mine)
    for i in range(page + 3):
        fresh = [torch.randn(x.shape, generator=g).bfloat16().to(DEV) for x in qkv]
        for x, y in zip(qkv, fresh):
            x.copy_(y)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = step(*theirs)
        torch.cuda.synchronize()
        assert int(theirs[0][0]) == i + 1
        for x, y in zip((a, b, *mine), (*want, *theirs)):
            assert torch.equal(x, y), i
        assert torch.equal(a, b)

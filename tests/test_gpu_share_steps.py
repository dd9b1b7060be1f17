"""Requests that fork, grow, are compacted and attend over the prefixes that they share, step after
step as a beam search takes them, against rows that each keep their own history, on an MI355X."""
import random

import pytest
import torch

import paged_reference as ref
from vecattention_amd import (copy_paged_kv, paged_kv_compact, paged_kv_fork, paged_kv_plan,
                              paged_kv_prefix, paged_prefix_decode_attention, write_paged_kv)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
PAGE, HQ, HK, D, LAYERS, PAGES, ROWS = 16, 8, 2, 64, 2, 160, 6
# Wide enough that the prefix is computed once, and one that is not.
WIDE, NARROW = 11200, 64
PROMPTS = [300, 123]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Batch:
    """The state of a serving program: rows, pages and caches."""

    def __init__(self, width, dtype):
        self.lens = torch.zeros(ROWS, dtype=torch.int32, device=DEV)
        self.table = torch.full((ROWS, width), -1, dtype=torch.int32, device=DEV)
        self.shares = torch.zeros(PAGES, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(PAGES, generator=torch.Generator().manual_seed(1)).int().to(DEV)
        self.head = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.k = [torch.full((PAGES, PAGE, HK, D), float("nan"), dtype=dtype, device=DEV)
                  for _ in range(LAYERS)]
        self.v = [torch.full_like(k, float("nan")) for k in self.k]

    def state(self):
        return [self.lens, self.table, self.shares, self.free, self.head]

    def take(self, *new):
        for t, x in zip(self.state(), new):
            t.copy_(x)

    def grow(self, new_lens, k, v):
        """k, v: (layers, tokens, heads, D)."""
        plan = paged_kv_plan(self.lens, new_lens, self.table, self.free, PAGE, k.shape[1],
                             self.head)
        for i in range(LAYERS):
            write_paged_kv(k[i], v[i], self.k[i], self.v[i], plan.slot_mapping)
        self.lens.copy_(plan.kv_lens)
        self.head.add_(plan.pages_taken.int())

    def attend(self, q):
        prefix = paged_kv_prefix(self.lens, self.table, PAGE)
        return torch.stack([paged_prefix_decode_attention(q[i], self.k[i], self.v[i], self.table,
                                                          self.lens, prefix)
                            for i in range(LAYERS)])

    def fork(self, parents, keep=None):
        f = paged_kv_fork(self.lens, parents, self.table, self.shares, self.free, PAGE, self.head,
                          keep)
        copy_paged_kv(self.k, self.v, f.copy_src, f.copy_dst, f.copy_rows)
        self.take(f.kv_lens, f.block_tables, f.page_shares, f.free_pages, f.free_head)

    def compact(self):
        c = paged_kv_compact(self.lens, self.table, self.shares, self.free, PAGE, self.head)
        copy_paged_kv(self.k, self.v, c.copy_src, c.copy_dst)
        self.take(self.lens, c.block_tables, c.page_shares, c.free_pages, c.free_head)

    def step(self, one, k, v, q, parents):
        self.grow(one, k, v)
        out = self.attend(q)
        self.fork(parents)
        return out


def plain(history, keys, values, q, dtype):
    """(want, room) of one layer from each row's tokens alone."""
    longest = -(-max(len(h) for h in history) // PAGE)
    k = torch.zeros(len(history) * longest, PAGE, HK, D, dtype=dtype)
    v = torch.zeros_like(k)
    table = torch.arange(len(history) * longest).view(len(history), longest)
    for n, h in enumerate(history):
        k[n * longest:(n + 1) * longest].view(-1, HK, D)[:len(h)] = keys[h]
        v[n * longest:(n + 1) * longest].view(-1, HK, D)[:len(h)] = values[h]
    lens = torch.tensor([len(h) for h in history], dtype=torch.int32)
    want, slack = ref.decode(q, k, v, table, lens, "NHD")
    size, _ = ref.decode(q, k, v.abs(), table, lens, "NHD")
    # The shared keys' weights are rounded by half a step each, in both sums; fp16 holds them
    # to 2^-25 of 2^-7 of the greatest.
    slack = slack + 2 * ref.HALF_STEP[dtype] * size
    if dtype == torch.float16:
        slack = slack + 2.0 ** -31 * int(lens.max()) * float(v.abs().max())
    return want, ref.rounded(want, slack, dtype)


def whole(batch, history):
    """Every page is held as often as it is counted, or free, once."""
    lens, table = batch.lens.tolist(), batch.table.cpu().tolist()
    shares, free, head = batch.shares.tolist(), batch.free.tolist(), int(batch.head)
    assert lens == [len(h) for h in history]
    held = [p for n, row in enumerate(table) for p in row[:-(-lens[n] // PAGE)]]
    assert all(0 <= p < PAGES for p in held)
    assert sorted(set(held) | set(free[head:])) == list(range(PAGES))
    assert len(set(held)) + len(free) - head == PAGES
    assert shares == [max(held.count(p) - 1, 0) for p in range(PAGES)]
    for n, row in enumerate(table):  # the page that a row writes next is its own
        if lens[n] % PAGE:
            assert held.count(row[lens[n] // PAGE]) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [WIDE, NARROW])
def test_beams_fork_grow_and_attend(width, dtype):
    print("[case] steps", width, dtype, flush=True)
    r = random.Random(width)
    steps, g = 40, torch.Generator().manual_seed(3)
    total = sum(PROMPTS) + ROWS * (steps + 1)
    keys, values = (torch.randn(LAYERS, total, HK, D, generator=g).to(dtype) for _ in range(2))
    d_keys, d_values = keys.to(DEV), values.to(DEV)
    queries = torch.randn(steps + 1, LAYERS, ROWS, HQ, D, generator=g).to(dtype)
    one = ints([1] * ROWS)
    eager, graphed = Batch(width, dtype), Batch(width, dtype)
    # Two prompts, each forked to three rows.
    history = [list(range(PROMPTS[0])), list(range(PROMPTS[0], sum(PROMPTS)))] + [[]] * 4
    for b in (eager, graphed):
        b.grow(ints(PROMPTS + [0] * 4), d_keys[:, :sum(PROMPTS)], d_values[:, :sum(PROMPTS)])
        b.fork(ints([0, 0, 0, 1, 1, 1]))
    history = [list(history[0]) for _ in range(3)] + [list(history[1]) for _ in range(3)]
    whole(eager, history)
    # One step, to load what is loaded at a first call, then the same step as a graph.
    k, v = (torch.empty(LAYERS, ROWS, HK, D, dtype=dtype, device=DEV) for _ in range(2))
    q, parents = queries[0].to(DEV), ints(range(ROWS))
    at = sum(PROMPTS)
    k.copy_(d_keys[:, at:at + ROWS]), v.copy_(d_values[:, at:at + ROWS])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step(one, k, v, q, parents)
    torch.cuda.current_stream().wait_stream(side)
    eager.step(one, k, v, q, parents)
    for n in range(ROWS):
        history[n].append(at + n)
    graph, tidy = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.step(one, k, v, q, parents)
    with torch.cuda.graph(tidy):
        graphed.compact()
    for s in range(1, steps + 1):
        at = sum(PROMPTS) + ROWS * s
        mine = [r.randrange(3) for _ in range(3)] + [3 + r.randrange(3) for _ in range(3)]
        if s % 9 == 0:
            mine = list(range(ROWS))
        k.copy_(d_keys[:, at:at + ROWS]), v.copy_(d_values[:, at:at + ROWS])
        q.copy_(queries[s]), parents.copy_(ints(mine))
        graph.replay()
        got = out.clone()
        want = eager.step(one, k, v, q, parents)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        grown = [h + [at + n] for n, h in enumerate(history)]
        if s % 5 == 1:
            for i in range(LAYERS):
                exact, room = plain(grown, keys[i], values[i], queries[s, i], dtype)
                assert bool(((want[i].double().cpu() - exact).abs() <= room).all())
        history = [list(grown[p]) for p in mine]
        if s % 7 == 0:
            tidy.replay()
            eager.compact()
        assert all(torch.equal(a, b) for a, b in zip(eager.state(), graphed.state()))
        whole(eager, history)


def test_speculative_tokens_are_taken_back():
    """Rows that drop their last tokens (keep_lens) and rows that end give their pages back."""
    print("[case] taken back", flush=True)
    dtype, g = torch.bfloat16, torch.Generator().manual_seed(4)
    r = random.Random(2)
    keys, values = (torch.randn(LAYERS, 2000, HK, D, generator=g).to(dtype) for _ in range(2))
    b = Batch(WIDE, dtype)
    b.grow(ints([200] + [0] * 5), keys[:, :200].to(DEV), values[:, :200].to(DEV))
    b.fork(ints([0] * 6))
    history, at = [list(range(200)) for _ in range(ROWS)], 200
    for s in range(8):
        new = [r.randint(1, 20) if h else 0 for h in history]
        n = sum(new)
        b.grow(ints(new), keys[:, at:at + n].to(DEV), values[:, at:at + n].to(DEV))
        for i, c in enumerate(new):
            history[i] = history[i] + list(range(at, at + c))
            at += c
        mine = list(range(ROWS))
        if s == 3:
            mine = [0, 1, 1, -1, 4, 4]
        keep = [max(len(h) - r.randint(0, 25), 1) for h in history]
        b.fork(ints(mine), ints(keep))
        history = [history[p][:keep[i]] if p >= 0 else [] for i, p in enumerate(mine)]
        whole(b, history)
        q = torch.randn(LAYERS, ROWS, HQ, D, generator=g).to(dtype)
        out = b.attend(q.to(DEV))
        for i in range(LAYERS):
            exact, room = plain(history, keys[i], values[i], q[i], dtype)
            assert bool(((out[i].double().cpu() - exact).abs() <= room).all())

"""Attention of rows that share the beginnings of their pages where its arithmetic is at its ends,
on an MI355X."""
import pytest
import torch

import paged_reference as ref
from test_gpu_prefix_attention import make, note, run

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

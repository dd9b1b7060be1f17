"""Attention of rows that share the beginnings of their pages where its arithmetic is at its ends,
on an MI355X."""
import pytest
import torch

import paged_reference as ref
from test_gpu_prefix_attention import make, run

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


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

"""fused_sample where its weights' bound and its sums' range are used up.

Weights are integers, 2^43 w of the largest: rounded, off by 2^-44.  Those under
2^-18 come from the fp32 exponential and are off by 2^-22 of themselves besides
(sampling.cu), so the sum of n weights, m of it the small ones, is off by at most

    E = n 2^-44 + 2^-22 m        (the largest weight being 1)

and a log-probability by E / sum and one fp32 rounding, 2^-24 of itself (and fp64
arithmetic, 1e-12).  A token is drawn for certain where u * sum lies further than
E from the running sums beside it.
"""

import math
from fractions import Fraction

import pytest
import torch

from metal_liger_b200.ops.fused_sampling import fused_sample

pytestmark = pytest.mark.gpu
DEV = "cuda"
MOST = 1 << 20                                                   # tokens of a row


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B", [1, 5, 20, 40])
def test_the_most_tokens_there_can_be_all_alike(dtype, B):
    """2^20 weights of 2^43: their sum is 2^63, the most there is.  u is a
    multiple of 2^-24, so u n is exact and the token is the integer part of it."""
    x = torch.full((B, MOST), 1.5, dtype=dtype, device=DEV)
    u = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24, 2.0 ** -24, 0.25 - 2.0 ** -25, 1 / 3])
    u = u.repeat(-(-B // 6))[:B]
    if B == 1:
        u[0] = 1 - 2.0 ** -24
    for kw, n in ((dict(), MOST), (dict(top_p=0.5), MOST // 2), (dict(top_k=1000), 1000),
                  (dict(min_p=1.0), MOST), (dict(top_k=MOST - 1, top_p=0.75), None),
                  (dict(top_p=1 - 2.0 ** -24), MOST)):
        if n is None:                                            # 0.75 of 2^20 - 1, rounded up
            n = math.ceil(Fraction(3, 4) * (MOST - 1))
        ids, logp = fused_sample(x, u.to(DEV), **kw)
        want = [int(Fraction(float(v)) * n) for v in u]
        assert ids.tolist() == want, kw
        lp = -math.log(n)
        assert all(abs(v - lp) <= 2.0 ** -24 * abs(lp) + 1e-12 for v in logp.tolist()), kw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [MOST, 151936])
@pytest.mark.parametrize("log2w", [-18.5, -19.0, -19.9])
def test_small_weights_that_make_up_the_sum(dtype, V, log2w):
    """One token of weight 1, all others equal and small: whatever the fp32
    exponential is off by, they are off by together."""
    x = torch.full((V,), log2w * math.log(2.0), dtype=dtype)
    x[5] = 0.0
    w = math.exp(float(x[0]))
    assert 2.0 ** -20.1 < w < 2.0 ** -18
    total = 1.0 + (V - 1) * w
    E = V * 2.0 ** -44 + 2.0 ** -22 * (V - 1) * w
    picks = [0, 4, 5, 6, V // 3, V // 2, V - 1]
    u = []
    for j in picks:                                              # the middle of token j's stretch
        before = j * w if j <= 5 else (j - 1) * w + 1.0
        u.append((before + (0.5 if j == 5 else 0.5 * w)) / total)
    u = torch.tensor(u, dtype=torch.float64).float()
    # u's own rounding and E leave the target inside the stretch
    assert E + 2.0 ** -25 * total < 0.5 * w
    ids, logp = fused_sample(x.to(DEV).expand(len(picks), V), u.to(DEV))
    assert ids.tolist() == picks
    for j, got in zip(picks, logp.tolist()):
        lp = (0.0 if j == 5 else float(x[0])) - math.log(total)
        assert abs(got - lp) <= E / total + 2.0 ** -24 * abs(lp) + 1e-12, (j, got, lp)

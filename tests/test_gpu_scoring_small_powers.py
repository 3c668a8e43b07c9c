"""Where a probability counts as 0: below 2^-122 of the row's largest it may,
and above that it does not.

The kernels' power 2^y, y = k + i/32 + f with |f| <= 1/64, is cut where its
table entry times 2^k is no normal number: 0.24110 2^(k + i/32) < 2^-126 is
k + i/32 < -123.948, at most -123.96875 as a multiple of 1/32, which is the
nearest one for y < -123.953.  The argument is off by 3 u |y| = 2.2e-5.
"""
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("n", [1, 2000])  # one short row in one kernel; sums, then rows
def test_probabilities_near_the_cut(n):
    import torch

    from detllm_b200 import scoring as sc

    t = torch.arange(118.0, 128.0, 1 / 64, dtype=torch.float64)  # p = 2^-t of the largest
    x = torch.cat([torch.zeros(1, dtype=torch.float64), -t * math.log(2)]).float().cuda()
    xs = x.repeat(n, 1)
    tokens = torch.zeros(n, dtype=torch.int64, device="cuda")
    one = torch.full((n,), 1.0, device="cuda")
    f = sc.token_scores(xs, tokens)
    y = x[1:].double().cpu() / math.log(2)
    d = x[1:].double().cpu().abs()
    want = torch.exp2(y)  # S = 1 + 2^-117 and less
    # as the power of an entry, its argument and three products; the gradient is
    # -p, to 0 below 2^-149
    tol = want * (7.1 + 3 * d + 4) * U
    for grad in (sc.token_scores_grad(xs, tokens, f.stats, one), sc.token_scores_step(xs, tokens, one)[1]):
        p = -grad[n - 1, 1:].double().cpu()
        kept = p > 0
        assert kept[y >= -122].all()
        assert kept[y >= -123.92].all() and not kept[y < -123.98].any()
        assert ((p - want).abs() <= tol)[kept].all()

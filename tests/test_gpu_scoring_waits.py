"""The step calls' bounded waits: a wait that runs out is reported, leaves
nothing but NaN, and leaves the device usable."""
import time

import pytest

pytestmark = pytest.mark.gpu


def test_step_wait_times_out_and_device_recovers():
    """The step's kernels with one wait that nothing ends (20 ms): the library
    checks that each result, statistic and gradient of each row is NaN, those of
    rows that were finished or never drawn among them, and that the flag is set;
    calls before and after it agree."""
    import torch

    import detllm_b200 as D
    from detllm_b200 import scoring as sc

    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(9, 40001, generator=g, device="cuda")
    tokens = torch.randint(0, 40001, (9,), generator=g, device="cuda")
    one = torch.ones(9, device="cuda")
    before = sc.token_scores_step(x, tokens, one, one)
    torch.cuda.synchronize()
    t = time.time()
    code = D.lib().det_step_timeout_selftest(0)
    assert code == 67, D.lib().det_status_string(code)  # DET_ERR_TIMEOUT
    assert time.time() - t < 20
    after = sc.token_scores_step(x, tokens, one, one)
    assert all(torch.equal(a, b) for a, b in zip((*before[0][:3], before[1]), (*after[0][:3], after[1])))
    assert torch.isfinite(after[1]).all()

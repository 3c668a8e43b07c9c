"""The steps' wait self-test without a GPU."""
import pytest


def test_it_needs_a_device():
    import detllm_b200 as D

    lib = D.lib()
    if D.device_count() > 0:
        assert lib.det_step_timeout_selftest(-1) == 63  # DET_ERR_INVALID_ARGUMENT
        assert lib.det_step_timeout_selftest(D.device_count()) == 63
        pytest.skip("a GPU is visible")
    assert lib.det_step_timeout_selftest(0) == 65  # DET_ERR_NO_DEVICE

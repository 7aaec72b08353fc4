"""GPU test of the cache kernels' part of the device status word: a wait that runs out is reported."""
import ctypes
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_waits_of_the_cache_kernels_run_out_and_report(cuda_device):
    """The diagnostic's third kernel waits with the cache kernels' wait; the call fails unless its code comes back."""
    from w4a16_opt import capi, device_status
    lib = capi.load()
    codes = (ctypes.c_int32 * 2)()
    t0 = time.monotonic()
    capi.check(lib.w4a16_check_wait_limits(codes), lib)
    assert 6.0 < time.monotonic() - t0 < 60.0
    assert list(codes) == [4, 1] and device_status() == 0
    x = torch.ones(4, device="cuda")
    assert float((x * 2).sum()) == 8.0

"""The kernels' waits are bounded in time: one that nothing ends gives up and says so."""
import time

import pytest
import torch

from vdit import _lib

pytestmark = pytest.mark.gpu


def test_a_wait_that_nothing_ends_gives_up_within_its_limit():
    """The launch lasts the limit and no longer (the slack is the launch and the host's own), the error
    word names the wait, and the device goes on working."""
    lib = _lib.load()
    limit = lib.vdit_wait_limit_ms()
    assert 0 < limit <= 5000
    assert _lib.device_error(clear=True) == 0
    torch.cuda.synchronize()
    t = time.perf_counter()
    assert lib.vdit_wait_check(torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t) * 1e3
    assert limit * 0.99 <= ms <= limit + 500, ms
    assert _lib.device_error(clear=True) == 0x5754
    assert _lib.device_error(clear=True) == 0
    assert int(torch.arange(1000, device="cuda").sum()) == 499500

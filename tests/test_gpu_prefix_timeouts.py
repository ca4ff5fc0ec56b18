"""What a wait that runs out inside shared-prefix attention does.  The launches are healthy; the bound on their waits
is set so low that the warps of the prefix pass, which wait for one another all the time, give up."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_paged import BF, C_, F16, attend, make_attn  # noqa: F401

pytestmark = pytest.mark.gpu

TIMEOUT = 5

SHAPES = [
    # R, nq, nkv, hd, prefix, own, page, type
    (24, 16, 4, 128, 1333, 50, 16, BF),     # tiles of 128 rows of heads
    (90, 16, 4, 64, 3333, 50, 16, F16),     # of 256
    (8, 96, 96, 128, 2000, 300, 16, BF),    # spans across kv heads
    (130, 96, 96, 64, 1999, 20, 16, F16),
    (256, 32, 8, 128, 16400, 300, 32, BF),  # four row tiles side by side
]


@pytest.fixture
def limit(C_):  # noqa: F811
    from tritiercache_b200 import _lib
    L = _lib.lib()

    def error():
        e = ctypes.c_int(-1)
        assert L.tt_device_error(1, ctypes.byref(e)) == 0
        return e.value
    assert error() == 0
    try:
        yield L.tt_shared_prefix_wait_limit, error
    finally:
        L.tt_shared_prefix_wait_limit(-1)
        torch.cuda.synchronize()
        error()


@pytest.mark.parametrize("R,nq,nkv,hd,prefix,own,P,dt", SHAPES)
def test_waits_that_run_out(C_, limit, R, nq, nkv, hd, prefix, own, P, dt):  # noqa: F811
    set_limit, error = limit
    s = make_attn(70, R, nq, nkv, hd, prefix, np.full(R, own), P, dt)
    good = attend(C_, s)
    assert bool(torch.isfinite(good).all()) and error() == 0
    for clocks in (0, 300, 1000, 3000, 10000, 30000, 0):
        assert set_limit(clocks) == 0
        for _ in range(3):
            out = attend(C_, s)
            torch.cuda.synchronize()
            lost = torch.isnan(out)
            # a row of a head is lost as a whole or right, and what is lost is reported, once
            assert torch.equal(lost.any(-1), lost.all(-1)) and torch.equal(out[~lost], good[~lost])
            if clocks == 0:
                assert bool(lost.any())
            assert not bool(lost.any()) or error() == TIMEOUT
            error()
            assert error() == 0
        # the next call is sound
        set_limit(-1)
        assert torch.equal(attend(C_, s), good) and error() == 0


@pytest.mark.parametrize("R,nq,nkv,hd,prefix,own,P,dt", [(8, 96, 96, 128, 2000, 300, 16, BF), (256, 32, 8, 128, 16400, 300, 32, BF),
                                                          (256, 16, 4, 64, 16400, 700, 32, F16)])
def test_giving_up_takes_no_time(C_, limit, R, nq, nkv, hd, prefix, own, P, dt):  # noqa: F811
    """What is in flight when a warp gives up arrives within microseconds; nothing waits for what has been before."""
    set_limit, error = limit
    s = make_attn(71, R, nq, nkv, hd, prefix, np.full(R, own), P, dt)
    attend(C_, s)
    slowest = 0.0
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for clocks in (0, 1, 100, 300, 1000):
        set_limit(clocks)
        for _ in range(8):
            a.record()
            attend(C_, s)
            b.record()
            torch.cuda.synchronize()
            slowest = max(slowest, a.elapsed_time(b))
        assert error() == TIMEOUT
    assert slowest < 500, slowest  # milliseconds; a wait in vain takes 2000

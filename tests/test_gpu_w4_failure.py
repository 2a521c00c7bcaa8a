"""GPU: what the 4-bit products do when a wait gives up: an error word, no copy left under way, and a
context that works on.  The waits run out because a copy is not issued, after a few ms."""

from __future__ import annotations

import sys
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

SLOTS = 4


@pytest.fixture(autouse=True)
def no_error_left(cuda_dev, pkg):
    read = sys.modules["fib_b200.kernel"].read_device_error
    read(cuda_dev)
    yield
    torch.cuda.synchronize()
    read(cuda_dev)


@pytest.mark.parametrize("issues", [0, 1, 3, 4, 5, 40, 41])
@pytest.mark.parametrize("missing", [0, 2, 3, 4, 17, 39, 40, 100])
def test_ring_stops_and_drains(issues, missing, pkg, cuda_dev):
    ops = sys.modules["fib_b200._ops"]
    src = torch.randint(-2 ** 31, 2 ** 31 - 1, (max(issues, 1), 256), device=cuda_dev, dtype=torch.int32)
    report = torch.full((6,), -1, dtype=torch.int32, device=cuda_dev)
    ops.call("moe_w4_selftest_ring", cuda_dev, src.data_ptr(), issues, missing, report.data_ptr())
    issued, taken, wrong, ran_out, left_behind, landed = report.tolist()
    assert wrong == 0
    if missing >= issues:                            # nothing is missing: all stages pass
        assert (issued, taken, ran_out, left_behind, landed) == (issues, issues, 0, 0, min(issues, SLOTS))
        return
    assert taken == missing                          # no warp takes a stage that has not come
    # its slot is never filled again, so at most the three other slots are after it
    assert missing < issued <= min(issues, missing + SLOTS)
    assert ran_out == (issued < issues)
    assert left_behind == 1 and landed == min(issued, SLOTS) - 1   # all that was copied is there, the missing one is not


def test_products_work_after_a_wait_that_gave_up(pkg, cuda_dev):
    ops = sys.modules["fib_b200._ops"]
    w = pkg.W4Weights(*pkg.quantize_w4(torch.randn(64, 512, device=cuda_dev), 32), group_size=32)
    x = torch.randn(9, 512, device=cuda_dev).bfloat16()
    want = pkg.w4_matvec(x, w)
    src, report = torch.zeros(12, 256, device=cuda_dev, dtype=torch.int32), torch.zeros(6, dtype=torch.int32, device=cuda_dev)
    ops.call("moe_w4_selftest_ring", cuda_dev, src.data_ptr(), 12, 5, report.data_ptr())
    assert torch.equal(pkg.w4_matvec(x, w), want) and report[1] == 5
    read, L = sys.modules["fib_b200.kernel"].read_device_error, sys.modules["fib_b200._lib"]
    assert read(cuda_dev) == 2                       # reported once, then cleared
    assert read(cuda_dev) == 0
    assert L.load().moe_w4_read_device_error(None, None) == L.MOE_ERR_INVALID_ARGUMENT


def test_no_error_is_lost_to_a_read(pkg, cuda_dev):
    """An error that is raised on one stream while another reads is seen by that read or by the next."""
    ops, read = sys.modules["fib_b200._ops"], sys.modules["fib_b200.kernel"].read_device_error
    src, report = torch.zeros(1, 256, device=cuda_dev, dtype=torch.int32), torch.zeros(6, dtype=torch.int32, device=cuda_dev)
    raising, reading = torch.cuda.Stream(), torch.cuda.Stream()

    def raise_one():                                 # when its waits run out
        ops.call("moe_w4_selftest_ring", cuda_dev, src.data_ptr(), 1, 0, report.data_ptr())

    for _ in range(2):
        start = time.perf_counter()
        raise_one()
        torch.cuda.synchronize()
        delay = time.perf_counter() - start
    read(cuda_dev)
    lost = []
    for step in range(400):                          # the read comes close to the raise: a little later after a miss
        torch.cuda.synchronize()
        start = time.perf_counter()
        with torch.cuda.stream(raising):
            raise_one()
        while time.perf_counter() - start < delay:
            pass
        with torch.cuda.stream(reading):
            first = read(cuda_dev)
        torch.cuda.synchronize()
        if (first, read(cuda_dev)) not in ((2, 0), (0, 2)):
            lost.append((step, delay))
        delay += -2e-6 if first else 2e-6
    assert not lost

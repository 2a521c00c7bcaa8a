"""GPU: what the 4-bit products do when a wait gives up: an error word, no copy left under way, and a
context that works on.  The waits run out because a copy is not issued, with a limit of 2 ms."""

from __future__ import annotations

import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

SLOTS = 4


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
    assert sys.modules["fib_b200.kernel"].read_device_error(cuda_dev) == 0

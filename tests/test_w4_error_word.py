"""Reading the device errors of a process that has made no 4-bit product costs and needs what it did before
there were any: no synchronisation, and no device of the right kind."""

from __future__ import annotations

import subprocess
import sys

import pytest

from conftest import ROOT


def run(code):
    done = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, '.')\n" + code], cwd=ROOT, timeout=300,
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_no_product_no_device_needed():
    run("""
import ctypes, os
os.environ["CUDA_VISIBLE_DEVICES"] = ""
from __graft_entry__ import load_package
load_package()
L = sys.modules["fib_b200._lib"]
code = ctypes.c_int32(7)
assert L.load().moe_w4_read_device_error(None, ctypes.byref(code)) == L.MOE_OK and code.value == 0
""")


@pytest.mark.gpu
def test_no_product_no_synchronisation(cuda_dev):
    """In the middle of a capture, which a synchronisation would end with an error."""
    run("""
import torch
from __graft_entry__ import load_package
load_package()
read = sys.modules["fib_b200.kernel"].read_device_error
x = torch.zeros(8, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    x += 1
    assert read() == 0 and read(torch.device("cuda", 0)) == 0
graph.replay()
assert x.tolist() == [1.0] * 8
""")

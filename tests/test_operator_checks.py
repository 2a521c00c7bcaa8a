"""CPU: the operators around the expert products refuse what they cannot do
before anything is launched."""

from __future__ import annotations

import sys

import pytest
import torch


def test_cpu_tensors_are_refused(pkg):
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.sort_tokens(ids, 3)
    order = pkg.TokenOrder(torch.zeros(4, dtype=torch.int32), ids, torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        pkg.dispatch(torch.zeros(4, 8), order)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.combine(torch.zeros(8, 8), torch.zeros(4, 2), order)
    with pytest.raises(TypeError):
        pkg.dispatch([1.0], order)


def test_token_entries_check_their_arguments(pkg):
    L = sys.modules["fib_b200._lib"]
    lib, bad, big, odd = L.load(), L.MOE_ERR_INVALID_ARGUMENT, L.MOE_ERR_TOO_LARGE, L.MOE_ERR_MISALIGNED
    p = 64                                    # an address that is never read: every call below ends before a launch
    sort, disp = lib.moe_tokens_sort, lib.moe_tokens_dispatch
    assert sort(p, -1, 8, 4, 0, p, p, p, None) == bad
    assert sort(p, 4, 0, 4, 0, p, p, p, None) == bad
    assert sort(p, 4, 8, 0, 0, p, p, p, None) == bad
    assert sort(p, 4, 8, 4, -1, p, p, p, None) == bad
    assert sort(p, 4, 8, 1025, 0, p, p, p, None) == big
    assert sort(p, 1 << 27, 8, 4, 0, p, p, p, None) == big
    assert sort(None, 4, 8, 4, 0, p, p, p, None) == bad
    assert sort(p, 4, 8, 4, 0, None, p, p, None) == bad
    assert sort(p, 4, 8, 4, 0, p, p + 2, p, None) == odd
    assert disp(p, p, 4, 8, 16, 7, p, None) == bad
    assert disp(p, p, 4, 8, 0, L.MOE_F32, p, None) == bad
    assert disp(p, p, 4, 8, 16, L.MOE_F32, None, None) == bad
    assert disp(p + 1, p, 4, 8, 16, L.MOE_BF16, p, None) == odd
    assert disp(None, None, 0, 8, 16, L.MOE_BF16, None, None) == L.MOE_OK
    comb, back = lib.moe_tokens_combine, lib.moe_tokens_combine_backward
    assert comb(p, p, p, 4, 8, 16, L.MOE_BF16, L.MOE_F32, p, None) == bad
    assert comb(p, p, p, 4, 8, 16, L.MOE_F16, L.MOE_BF16, p, None) == bad
    assert comb(p, p, p, 1 << 28, 8, 16, L.MOE_F32, L.MOE_F32, p, None) == big
    assert comb(p, p, p + 1, 4, 8, 16, L.MOE_F32, L.MOE_F32, p, None) == odd
    assert comb(None, None, None, 0, 8, 16, L.MOE_F32, L.MOE_F32, None, None) == L.MOE_OK
    assert back(p, None, p, p, 4, 8, 16, L.MOE_F32, L.MOE_F32, p, p, None) == bad
    assert back(p, p, p, None, 4, 8, 16, L.MOE_F32, L.MOE_F32, p, p, None) == bad
    assert back(p, p, p, p, 4, 8, 16, L.MOE_F32, L.MOE_F32, None, None, None) == L.MOE_OK
    assert back(p, p, p, p, 4, 8, 16, L.MOE_F32, L.MOE_F32, p + 2, p, None) == odd

"""CPU: the operators around the expert products refuse what they cannot do
before anything is launched."""

from __future__ import annotations

import ctypes
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
    assert sort(p, 4, 8, 4, 2 ** 31 - 4, p, p, p, None) == big     # ids would wrap into the shard
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


def test_swiglu_and_w4_entries_check_their_arguments(pkg):
    L = sys.modules["fib_b200._lib"]
    lib, bad, big, odd = L.load(), L.MOE_ERR_INVALID_ARGUMENT, L.MOE_ERR_TOO_LARGE, L.MOE_ERR_MISALIGNED
    p = 64
    fwd, bwd = lib.moe_swiglu_forward, lib.moe_swiglu_backward
    assert fwd(p, -1, 8, L.MOE_BF16, p, None, None, None) == bad
    assert fwd(p, 4, 0, L.MOE_BF16, p, None, None, None) == bad
    assert fwd(p, 4, 8, 9, p, None, None, None) == bad
    assert fwd(p, 4, 8, L.MOE_BF16, p, p, None, None) == bad
    assert fwd(p, 4, 8, L.MOE_BF16, p, None, p, None) == bad
    assert fwd(p + 1, 4, 8, L.MOE_BF16, p, None, None, None) == odd
    assert fwd(p, 4, 1 << 30, L.MOE_BF16, p, None, None, None) == big
    assert fwd(None, 0, 8, L.MOE_BF16, None, None, None, None) == L.MOE_OK
    assert bwd(p, None, p, 4, 8, L.MOE_BF16, p, None) == bad
    assert bwd(p, p, p + 2, 4, 8, L.MOE_BF16, p, None) == odd
    assert bwd(None, None, None, 0, 8, L.MOE_BF16, None, None) == L.MOE_OK
    n8 = ctypes.c_uint64()
    ref = ctypes.byref(n8)
    size = lib.moe_w4_layout_size
    assert size(0, 16, 64, 32, 0, ref) == size(1, 0, 64, 32, 0, ref) == size(1, 16, 64, 16, 0, ref) == bad
    assert size(1, 16, 96, 64, 0, ref) == size(1, 16, 64, 32, 0, None) == bad
    assert size(1025, 16, 64, 32, 0, ref) == size(1, 16, (1 << 24) + 128, 32, 0, ref) == big
    assert size(3, 17, 160, 32, 1, ref) == L.MOE_OK and n8.value == 3 * 2 * 2 * (1024 + 4 * 48)
    assert size(1, 16, 128, 128, 0, ref) == L.MOE_OK and n8.value == 1024 + 32
    lay = lib.moe_w4_lay_out
    assert lay(None, p, None, 1, 16, 64, 32, p, None) == lay(p, None, None, 1, 16, 64, 32, p, None) == bad
    assert lay(p, p, None, 1, 16, 64, 32, None, None) == bad
    assert lay(p + 2, p, None, 1, 16, 64, 32, p, None) == lay(p, p, None, 1, 16, 64, 32, p + 8, None) == odd
    size = lib.moe_w4_workspace_size
    assert size(-1, 128, ref) == size(4, 0, ref) == size(4, 128, None) == bad
    assert size(4, 640, ref) == L.MOE_OK and n8.value == 4 * 2 * 1088 + 16
    mv = lib.moe_w4_matvec

    def call(x=p, layout=p, offsets=p, R=4, E=2, n=16, d=128, group=64, dt=L.MOE_BF16, out=L.MOE_BF16, y=p, ws=256,
             nbytes=1 << 20):
        return mv(x, layout, offsets, R, E, n, d, group, 0, dt, out, 0, y, ws, nbytes, None)
    assert call(R=-1) == call(E=0) == call(n=0) == call(d=0) == bad
    assert call(group=16) == call(group=256) == call(d=96) == bad
    assert call(offsets=None) == bad
    assert call(dt=L.MOE_F32) == call(out=L.MOE_F16) == bad
    assert call(layout=None) == call(x=None) == call(y=None) == bad
    assert call(E=1025) == big
    # 1024 * 131072 chunks of rows times 16
    assert call(R=1 << 22, E=1024, n=1, nbytes=1 << 40) == big
    assert call(x=p + 2) == call(layout=p + 8) == call(offsets=p + 2) == call(y=p + 1) == call(ws=264) == odd
    assert call(ws=None) == call(nbytes=4 * 1088) == L.MOE_ERR_WORKSPACE_TOO_SMALL
    assert call(R=0, x=None, y=None) == L.MOE_OK


def test_swiglu_and_w4_refuse_cpu_tensors_and_shapes(pkg):
    with pytest.raises(ValueError, match="CUDA"):
        pkg.swiglu(torch.zeros(2, 8))
    codes, scales, zeros = pkg.quantize_w4(torch.randn(3, 20, 64), 32)
    assert zeros is None
    W = pkg.W4Weights
    with pytest.raises(ValueError, match="CUDA"):
        W(codes, scales, group_size=32)
    with pytest.raises(TypeError):
        pkg.w4_matvec(torch.zeros(2, 64), (codes, scales))
    with pytest.raises(ValueError):
        pkg.quantize_w4(torch.randn(4, 100), 32)
    with pytest.raises(ValueError):
        W(codes, scales, group_size=16)
    with pytest.raises(ValueError):
        W(codes, scales[0], group_size=32)
    with pytest.raises(TypeError):
        W(codes, scales.float(), group_size=32)
    with pytest.raises(TypeError):
        W(codes.to(torch.int8), scales, group_size=32)


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantize_w4_takes_the_nearest_value(zero_points, pkg):
    g = torch.Generator().manual_seed(5)
    w = torch.randn(2, 10, 96, generator=g)
    w[0, 0] = 0
    codes, scales, zeros = pkg.quantize_w4(w, 32, zero_points)
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (3, 32)).float()
    z = zeros.unsqueeze(-1).float() if zero_points else 8.0
    back = ((q - z) * scales.unsqueeze(-1).float()).flatten(-2)
    step = scales.float().repeat_interleave(32, -1)
    # half a step, and at an end of the range what the rounding of the scale (bf16, 2^-8) over 15 codes and
    # of the zero point (half a step) clips
    assert bool(((w - back).abs() <= step * (0.5 + 15 * 2.0 ** -8 + (0.5 if zero_points else 0.0))).all())


def test_sizes_beyond_32_bits_are_refused(pkg):
    """Not cut to 32 bits on their way into the library; meta tensors stand for the memory."""
    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")
    much = 2 ** 31
    for make in (lambda: pkg.sort_tokens(meta(much, 1, dtype=torch.int32), 4), lambda: pkg.swiglu(meta(much, 2)),
                 lambda: pkg.swiglu(meta(1, 2 * much)),
                 lambda: pkg.dispatch(meta(1, much), pkg.TokenOrder(*[meta(1, 1, dtype=torch.int32)] * 3))):
        with pytest.raises(ValueError, match="2147483647"):
            make()
    with pytest.raises(ValueError, match="split"):
        pkg.W4Weights(meta(1, much, 16, dtype=torch.uint8), meta(1, much, 1), group_size=32)
    with pytest.raises(ValueError):
        pkg.quantize_w4(torch.zeros(2, 4), 0)

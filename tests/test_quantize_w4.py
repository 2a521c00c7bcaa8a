"""4-bit quantisation at the ends of the scales' types."""

from __future__ import annotations

import pytest
import torch

FP16, BF16 = torch.float16, torch.bfloat16


def values(codes, scales, zeros, group):
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, group)).double()
    z = zeros.unsqueeze(-1).double() if zeros is not None else 8.0
    return ((q - z) * scales.unsqueeze(-1).double()).flatten(-2)


ENDS = [*[(FP16, m * 2.0 ** -24) for m in (0.01, 0.3, 1.0, 3.4, 3.6, 7.0, 10.4, 100.0, 7000.0, 7200.0, 20000.0)],
        (FP16, 4e5), *[(BF16, m * 2.0 ** -133) for m in (0.3, 3.4, 10.4, 100.0)], (BF16, 2.0 ** -120), (BF16, 3e38)]


def quantise_an_end(dtype, largest, zero_points, pkg, dev):
    """Every weight comes within half a step of itself; at an end of the range the scale's rounding over 15
    codes (half a step of the type, none below its normal numbers, where scales are rounded up) and the zero
    point's (half a step) clip in addition.  A step is the scale."""
    g = torch.Generator().manual_seed(7)
    w = (torch.rand(6, 64, generator=g) * 2 - 1) * largest
    w[:, 0] = w[:, 32] = largest
    w[1] = w[1].abs()
    w[2] = -w[2].abs()
    w = w.to(dev)
    codes, scales, zeros = pkg.quantize_w4(w, 32, zero_points, dtype)
    assert scales.dtype == dtype and bool((scales > 0).all()) and bool(torch.isfinite(scales).all())
    info, step = torch.finfo(dtype), scales.double().repeat_interleave(32, -1)
    clip = (0.5 if zero_points else 0.0) + 15 * info.eps / 2
    assert bool(((w.double() - values(codes, scales, zeros, 32)).abs() <= step * (0.5 + clip)).all())
    # and a step is no longer than what 15 (or 7) of them have to cover, rounded once
    v = w.double().unflatten(-1, (-1, 32))
    wanted = (v.amax(-1).clamp_min(0) - v.amin(-1).clamp_max(0)) / 15 if zero_points else v.abs().amax(-1) / 7
    assert bool((scales.double() <= wanted * (1 + info.eps) + info.smallest_normal * info.eps).all())


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype,largest", ENDS)
def test_scales_at_the_ends_of_their_type(dtype, largest, zero_points, pkg):
    quantise_an_end(dtype, largest, zero_points, pkg, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype,largest", ENDS)
def test_scales_at_the_ends_of_their_type_on_the_gpu(dtype, largest, zero_points, pkg, cuda_dev):
    quantise_an_end(dtype, largest, zero_points, pkg, cuda_dev)


@pytest.mark.parametrize("zero_points", [False, True])
def test_ordinary_weights_keep_their_codes(zero_points, pkg):
    """The scales of normal size are the rounded quotients they always were."""
    w = torch.randn(5, 7, 128, generator=torch.Generator().manual_seed(3))
    v = w.unflatten(-1, (-1, 32))
    wanted = (v.amax(-1).clamp_min(0) - v.amin(-1).clamp_max(0)) / 15 if zero_points else v.abs().amax(-1) / 7
    for dtype in (FP16, BF16):
        assert torch.equal(pkg.quantize_w4(w, 32, zero_points, dtype)[1], wanted.to(dtype))


@pytest.mark.parametrize("zero_points", [False, True])
def test_scales_that_are_not_finite_are_refused(zero_points, pkg):
    w = torch.ones(2, 64)
    for dtype, bad in ((FP16, 7.0 * 65536), (FP16, 3e38), (BF16, float("inf")), (FP16, float("nan")), (BF16, -float("inf"))):
        v = w.clone()
        v[1, 40] = bad
        if zero_points and abs(bad) < 1e6:
            v[1, 40] = 15.0 * 65536
        with pytest.raises(ValueError, match="not finite"):
            pkg.quantize_w4(v, 32, zero_points, dtype)


@pytest.mark.parametrize("zero_points", [False, True])
def test_parameters_leave_no_graph_behind(zero_points, pkg):
    """Quantised weights have no gradient, and must not hold a graph with fp32 copies of the parameter."""
    w = torch.nn.Parameter(torch.randn(4, 64, generator=torch.Generator().manual_seed(1)))
    got, want = pkg.quantize_w4(w, 32, zero_points), pkg.quantize_w4(w.detach(), 32, zero_points)
    for a, b in zip(got, want):
        assert (a is None and b is None) or (torch.equal(a, b) and not a.requires_grad)

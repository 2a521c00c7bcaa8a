"""Bounds on rounding errors that the operator tests compare with.

A value that is rounded once to a type is off by at most half a step of it:
``eps / 2`` relative, and half the least subnormal number near zero.  A sum
of fp32 products made in fp32 is off by at most (number of roundings on the
longest path) * 2^-24 * (sum of the terms' magnitudes).
"""

from __future__ import annotations

import torch

U32 = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def half_step(ref, dtype):
    """Bound on the rounding of ``ref`` (fp64) to ``dtype``."""
    return ref.abs() * (torch.finfo(dtype).eps / 2) + LEAST[dtype] / 2


def assert_close(got, ref, dtype, inner, what=""):
    """``got`` is ``ref`` with an fp32 error of at most ``inner`` and one rounding to ``dtype``."""
    assert got.dtype == dtype, f"{what}: {got.dtype}"
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} is not {tuple(ref.shape)}"
    bound = inner + half_step(ref.abs() + inner, dtype)
    off = (got.double() - ref).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst by "
                                 f"{float((off / bound.clamp_min(1e-300))[bad].max()):.3g} bounds")

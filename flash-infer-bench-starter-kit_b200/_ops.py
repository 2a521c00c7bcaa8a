"""What the operators around the expert products share on the Python side:
argument checks in the manner of ``kernel(...)`` and the call into the library
on the tensors' device and its current stream."""

from __future__ import annotations

import types

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib

INT32_MAX = 2 ** 31 - 1       # the library's sizes are 32-bit integers
DTYPES = {torch.float32: _lib.MOE_F32, torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16}

_entries: dict = {}

# The handle of a device's current stream: torch's own accessor without a Stream object around it
# where there is one (1.3 us of a 10 us call less).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


# The level of forward-mode differentiation that is open, -1 for none: torch's own variable where there is
# one (unpack_dual, which would tell as well, takes 0.7 us a tensor), else asked for each tensor.
_dual_level = forward_ad if hasattr(forward_ad, "_current_level") else types.SimpleNamespace(_current_level=0)


def refuse_tangent(name, t):
    """Refuse a dual tensor of forward-mode differentiation.  It need not require a gradient, so no
    ``autograd.Function`` would see it, and its tangent would be lost without a word."""
    if _dual_level._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent: there is no forward-mode derivative")


def check_tensor(name, t, dtypes, shape, device):
    """``shape``: the expected sizes, -1 for any; ``dtypes``: the accepted types; ``device``: None
    for any CUDA device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    got = t.shape
    if len(got) != len(shape) or any((n != -1 and n != m) or m > INT32_MAX for n, m in zip(shape, got)):
        want = ", ".join(f"at most {INT32_MAX}" if n == -1 else str(n) for n in shape)
        raise ValueError(f"{name} has shape {tuple(got)}, expected ({want})")
    if _dual_level._current_level >= 0:
        refuse_tangent(name, t)
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (no CPU path)")
    if device is not None and t.get_device() != device.index:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def check_output(name, t):
    """A tensor that a call overwrites: autograd is told, so that a backward pass which saved its values
    raises, as after any operation in place."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient that writing into it would not give: detach it")
    if not t.is_inference():
        increment_version(t)


def differentiable_once(backward):
    """``once_differentiable`` at no cost to ordinary backward passes, which run without gradients."""
    marked = once_differentiable(backward)

    def run(ctx, grad):
        return (marked if torch.is_grad_enabled() else backward)(ctx, grad)
    return run


def call(name, device, *args):
    """Run entry point ``name`` with ``args`` (pointers, None for NULL, and numbers) on ``device``'s
    current stream."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    index = device.index
    stream = _raw_stream(index)
    if torch.cuda.current_device() == index:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream)
    if status != _lib.MOE_OK:
        _lib.check(status, name)

"""GPU: SwiGLU at the ends of its inputs' range."""

from __future__ import annotations

import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def kept_codes(x):
    """(codes as bytes, scales) that the forward pass keeps of x."""
    ops = sys.modules["fib_b200._ops"]
    R, I = x.shape[0], x.shape[1] // 2
    y = torch.empty(R, I, dtype=x.dtype, device=x.device)
    codes = torch.empty(R, 2 * I, dtype=torch.uint8, device=x.device)
    scales = torch.empty(2 * -(-I // BLOCK), R, device=x.device)
    ops.call("moe_swiglu_forward", x.device, x.data_ptr(), R, I, ops.DTYPES[x.dtype], y.data_ptr(), codes.data_ptr(),
             scales.data_ptr())
    return codes, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("I", [384, 128])
@pytest.mark.parametrize("shift", [False, True])
def test_codes_keep_the_sign_of_zeros(dtype, I, shift, pkg, cuda_dev):
    """Codes equal the layer's activation format bit for bit, for zeros of both signs, values that round to
    zero, and blocks of zeros alone."""
    torch.manual_seed(I)
    x = torch.randn(40, 2 * I, device=cuda_dev)
    x[:, ::3] = -0.0
    x[:, 1::5] = 0.0
    x[:, 7::16] *= -1e-6
    x[4] = -0.0
    x[5, :BLOCK] = 0.0
    x = x.to(dtype)
    if shift:                                              # single columns
        x = torch.cat([x.new_zeros(1), x.view(-1)])[1:].view(40, 2 * I)
    codes, scales = kept_codes(x)
    q, s = pkg.inputs.quant_rows_1x128(x.cpu().float())
    assert bool((q.view(torch.uint8) == 0x80).any())
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu(), q.view(torch.uint8))

"""GPU: SwiGLU at the ends of its inputs' range."""

from __future__ import annotations

import sys

import pytest
import torch

from rounding import U32, assert_close
from test_gpu_swiglu import sigmoid_error

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("up", [1.0, 2.0 ** 20, 2.0 ** 100])
def test_gates_far_below_zero(dtype, up, pkg, cuda_dev):
    """silu(gate) * up where exp(-gate) leaves fp32, and its gradient.  e = exp(gate), the sigmoid and
    gate * sigmoid may lie below fp32's normal numbers, with a step of 2^-149 each."""
    torch.manual_seed(1)
    R, I = 64, 256
    gate = (-(80 + 24 * torch.rand(R, I, device=cuda_dev))).to(dtype)
    gate[:, 0] = -448.0 * 0.25                              # the block's scale is then 1/4: its codes are exact
    gate[:, 128] = -448.0 * 0.25
    x = torch.cat([torch.full((R, I), up, device=cuda_dev).to(dtype), gate], 1).requires_grad_(True)
    y = pkg.swiglu(x)
    least = 2.0 ** -149

    def reference(g):
        sig = torch.exp(g) / (1 + torch.exp(g))             # fp64: no range to leave
        return sig, sig * sigmoid_error(g) + 2 * least      # and e's step and the quotient's
    g = gate.double()
    sig, err = reference(g)
    assert_close(y.detach(), up * g * sig, dtype, up * (g.abs() * err + least + 2 * U32 * (g * sig).abs()), "y")
    # the gradient is that of the kept values: up exactly, gates by their codes
    grad_y = torch.full((R, I), 2.0 ** 20, device=cuda_dev).to(dtype)
    got, = torch.autograd.grad(y, x, grad_y)
    codes, scales = kept_codes(x.detach())
    s = scales.t().double()[:, 2:].repeat_interleave(BLOCK, 1)
    g = codes[:, I:].view(torch.float8_e4m3fn).double() * s
    sig, err = reference(g)
    c = 2.0 ** 20
    inner = 1 + g * (1 - sig)
    d_up, d_gate = c * g * sig, c * up * sig * inner
    assert_close(got[:, :I], d_up, dtype, c * g.abs() * err + 4 * U32 * d_up.abs() + least, "grad of up")
    assert_close(got[:, I:], d_gate, dtype, c * up * inner.abs() * err + 8 * U32 * d_gate.abs() + least, "grad of gate")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_at_the_ends(dtype, pkg, cuda_dev):
    """Zeros, the type's ends, infinities and NaN: the formula's values, in torch's elementary operations."""
    inf, nan, most = float("inf"), float("nan"), torch.finfo(dtype).max
    gate = torch.tensor([0.0, -0.0, most, -most, inf, nan, 1e-7, -1e-7, 30.0, -30.0], device=cuda_dev).to(dtype)
    up = torch.full_like(gate, 0.5)
    y = pkg.swiglu(torch.stack([up, gate], 1))[:, 0]
    g = gate.double()
    want = 0.5 * g * torch.sigmoid(g)
    want[3] = 0.0                                           # exp of it is 0 in any type
    assert_close(y[[i for i in range(10) if i not in (4, 5)]].double().to(dtype), want[[i for i in range(10) if i not in (4, 5)]],
                 dtype, want[[i for i in range(10) if i not in (4, 5)]].abs() * (3 + 5 + 2 * 36) * U32, "y")
    assert y[4] == inf and bool(torch.isnan(y[5]))

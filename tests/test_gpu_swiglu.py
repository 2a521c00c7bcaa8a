"""GPU: SwiGLU and its 8-bit checkpoint against the definition in 64 bits."""

from __future__ import annotations

import sys

import pytest
import torch

from rounding import U32, assert_close

pytestmark = pytest.mark.gpu

BLOCK = 128
SIZES = [(1, 2048), (3, 1), (5, 7), (17, 128), (64, 136), (33, 129), (250, 1000), (1000, 2048), (129, 516), (4099, 1288)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def e4m3_nearest(a):
    """Nearest e4m3 value of fp64 ``a`` (|a| <= 448 after rounding), ties to even."""
    exponent = (torch.frexp(a).exponent - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(a), exponent - 3)
    return (torch.round(a / step) * step).clamp(-448.0, 448.0)


def kept(x, I):
    """What the codes and scales of x's halves stand for (fp64); scale and quotient are fp32 values."""
    out = x.double().clone()
    for half in (0, I):
        for b in range(0, I, BLOCK):
            c = out[:, half + b:half + min(b + BLOCK, I)]
            s = (c.abs().amax(1, keepdim=True) / 448.0).float().double()
            s[s == 0] = 1.0
            c.copy_(e4m3_nearest((c / s).float().double()) * s)
    return out


def sigmoid_error(g):
    """Relative error of the fp32 sigmoid: exp is documented to 2 + 1.173 |g| units of 2^-23 in its short
    form, the division to 2, one addition; twice the rounding of what follows is added by the callers."""
    return (2 + 1.173 * g.abs() + 2 + 1) * 2 * U32


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,I", SIZES)
@pytest.mark.parametrize("shift", [False, True])
def test_forward_and_gradient(R, I, dtype, shift, pkg, cuda_dev):
    torch.manual_seed(R * I)
    x = (torch.randn(R, 2 * I, device=cuda_dev) * 3).to(dtype)
    x[0] *= 20                                             # far out on both sides of the sigmoid
    grad = torch.randn(R, I, device=cuda_dev).to(dtype)
    if shift:                                              # one element past an aligned start
        x = torch.cat([x.new_zeros(1), x.view(-1)])[1:].view(R, 2 * I)
        grad = torch.cat([grad.new_zeros(1), grad.view(-1)])[1:].view(R, I)
        assert x.data_ptr() % 16 and x.is_contiguous()
    with torch.no_grad():
        y0 = pkg.swiglu(x)
    x.requires_grad_(True)
    y = pkg.swiglu(x)
    assert torch.equal(y.detach(), y0)                     # keeping the codes changes nothing
    up, gate = x.detach()[:, :I].double(), x.detach()[:, I:].double()
    ref = up * gate * torch.sigmoid(gate)
    tiny = 2.0 ** -125                                     # below this the sigmoid may be 0
    assert_close(y.detach(), ref, dtype, ref.abs() * (sigmoid_error(gate) + 2 * U32) + tiny * (up * gate).abs(), "y")

    got, = torch.autograd.grad(y, x, grad)
    k = kept(x.detach(), I)
    up, gate, g = k[:, :I], k[:, I:], grad.double()
    sig = torch.sigmoid(gate)
    rel = sigmoid_error(gate)
    d_up = g * gate * sig
    inner = 1 + gate * (1 - sig)
    d_gate = g * up * sig * inner
    err_up = d_up.abs() * (rel + 3 * U32) + tiny * (g * gate).abs()
    # inner: 1 - sig (sig's error and one rounding), times gate, plus 1
    err_inner = gate.abs() * (sig * rel + U32) + (gate * (1 - sig)).abs() * 2 * U32 + inner.abs() * U32
    err_gate = d_gate.abs() * (rel + 4 * U32) + (g * up * sig).abs() * err_inner + tiny * (g * up).abs() * (1 + gate.abs())
    # the kept values are fp32 products of a code and a scale
    err_up, err_gate = err_up + 2 * U32 * (g * (1 + gate.abs())).abs() * gate.abs(), err_gate + 4 * U32 * (
        g * up * (1 + gate.abs())).abs()
    assert_close(got, torch.cat([d_up, d_gate], 1), dtype, torch.cat([err_up, err_gate], 1), "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
def test_kept_codes_are_the_layers_activation_format(dtype, pkg, cuda_dev):
    """Codes and scales equal ``inputs.quant_rows_1x128`` bit for bit, zero blocks included."""
    ops = sys.modules["fib_b200._ops"]
    torch.manual_seed(1)
    R, I = 77, 384
    x = torch.randn(R, 2 * I, device=cuda_dev).to(dtype)
    x[3, 128:256] = 0
    x[5] *= 2.0 ** -10
    y = torch.empty(R, I, dtype=dtype, device=cuda_dev)
    codes = torch.empty(R, 2 * I, dtype=torch.float8_e4m3fn, device=cuda_dev)
    scales = torch.empty(2 * I // BLOCK, R, device=cuda_dev)
    ops.call("moe_swiglu_forward", x.device, x.data_ptr(), R, I, ops.DTYPES[dtype], y.data_ptr(), codes.data_ptr(),
             scales.data_ptr())
    q, s = pkg.inputs.quant_rows_1x128(x.cpu().float())
    assert torch.equal(scales.cpu(), s)
    assert torch.equal(codes.cpu().view(torch.uint8), q.view(torch.uint8))


def test_gradient_agrees_with_differences(pkg, cuda_dev):
    """Inputs that the codes hold exactly (e4m3 values, 448 in each block): the gradient is then that of y at
    x, and central differences of the fp64 formula come within their own error (step^2 / 6 times a third
    derivative below 1.1 * |up|)."""
    torch.manual_seed(2)
    R, I, s = 9, 130, 2.0 ** -7
    codes = torch.randn(R, 2 * I).clamp(-3, 3) * 60
    for c in (0, 128, I, I + 128):
        codes[:, c] = 448.0
    x = (e4m3_nearest(codes.double()) * s).float().to(cuda_dev).requires_grad_(True)
    grad = torch.randn(R, I, device=cuda_dev)
    got, = torch.autograd.grad(pkg.swiglu(x), x, grad)

    def f(v):
        return v[:, :I] * v[:, I:] * torch.sigmoid(v[:, I:])
    v, step = x.detach().double(), 1e-4
    for half in (0, 1):
        d = torch.zeros_like(v)
        d[:, half * I:(half + 1) * I] = step
        diff = grad.double() * (f(v + d) - f(v - d)) / (2 * step)
        off = (got[:, half * I:(half + 1) * I].double() - diff).abs()
        up, gate = v[:, :I].abs(), v[:, I:].abs()
        bound = grad.double().abs() * ((1 + up) * (1 + gate) * 32 * U32 + step ** 2 * (1 + up))
        assert bool((off <= bound).all())


def test_non_finite_blocks(pkg, cuda_dev):
    """An infinity or a NaN makes its own block's gradients NaN and no other's."""
    R, I = 20, 256
    torch.manual_seed(4)
    x = torch.randn(R, 2 * I, device=cuda_dev).bfloat16()
    x[2, 5], x[7, I + 130] = float("inf"), float("nan")
    x.requires_grad_(True)
    y = pkg.swiglu(x)
    assert bool(torch.isnan(y[7, 130])) and int((~torch.isfinite(y)).sum()) == 2
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    bad = torch.zeros(R, 2 * I, dtype=torch.bool, device=cuda_dev)
    bad[2, I:I + 128] = True            # grad of gate holds up
    bad[7, 128:256] = bad[7, I + 128:] = True
    assert torch.equal(torch.isnan(dx), bad)


def test_empty_expanded_and_captured(pkg, cuda_dev):
    x = torch.empty(0, 64, device=cuda_dev, requires_grad=True)
    pkg.swiglu(x).sum().backward()
    assert x.grad.shape == (0, 64)
    torch.manual_seed(6)
    x = torch.randn(50, 600, device=cuda_dev).half().requires_grad_(True)
    pkg.swiglu(x).sum().backward()
    y = pkg.swiglu(x)
    want, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(x.grad, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    buf = x.detach().clone().requires_grad_(True)
    with torch.cuda.graph(graph, stream=side):
        y = pkg.swiglu(buf)
        dx, = torch.autograd.grad(y, buf, torch.ones_like(y))
    for seed in (7, 8):
        new = torch.randn(50, 600, device=cuda_dev).half()
        with torch.no_grad():
            buf.copy_(new)
        graph.replay()
        new.requires_grad_(True)
        ref = pkg.swiglu(new)
        assert torch.equal(y, ref) and torch.equal(dx, torch.autograd.grad(ref, new, torch.ones_like(ref))[0])


def test_refusals(pkg, cuda_dev):
    for bad in (torch.zeros(4, 7, device=cuda_dev), torch.zeros(4, 0, device=cuda_dev), torch.zeros(8, device=cuda_dev),
                torch.zeros(4, 32, device=cuda_dev)[:, ::2]):
        with pytest.raises(ValueError):
            pkg.swiglu(bad)
    with pytest.raises(TypeError):
        pkg.swiglu(torch.zeros(4, 8, device=cuda_dev, dtype=torch.float64))

"""SwiGLU between the two expert products, with an 8-bit checkpoint for its gradient.

The fused layer computes it inside its first product
(``solution/python/main.cpp:200-213`` of the reference); around other expert
products, and for training, it is a pass of its own.
"""

from __future__ import annotations

import torch

from ._ops import DTYPES, call, check_tensor, differentiable_once

BLOCK = 128


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        R, I = x.shape[0], x.shape[1] // 2
        y = torch.empty(R, I, dtype=x.dtype, device=x.device)
        codes = torch.empty(R, 2 * I, dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty(2 * -(-I // BLOCK), R, dtype=torch.float32, device=x.device)
        call("moe_swiglu_forward", x.device, x.data_ptr(), R, I, DTYPES[x.dtype], y.data_ptr(), codes.data_ptr(),
             scales.data_ptr())
        ctx.save_for_backward(codes, scales)
        return y

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_y):
        codes, scales = ctx.saved_tensors
        grad_y = grad_y.contiguous()
        R, I = grad_y.shape
        grad_x = torch.empty(R, 2 * I, dtype=grad_y.dtype, device=grad_y.device)
        call("moe_swiglu_backward", grad_y.device, grad_y.data_ptr(), codes.data_ptr(), scales.data_ptr(), R, I,
             DTYPES[grad_y.dtype], grad_x.data_ptr())
        return grad_x


def swiglu(x: torch.Tensor) -> torch.Tensor:
    """``up * gate * sigmoid(gate)`` for rows ``x = [up | gate]`` (fp32, fp16 or bf16 [R, 2 * I], the
    order of the layer's W13): [R, I].

    When ``x`` needs a gradient, what is kept for it is not ``x`` but its 8-bit form in the layer's
    activation format: e4m3 codes with one fp32 scale (amax / 448) per 1x128 block of up and of gate,
    about 2 bytes a column pair instead of 4 (16-bit ``x``).  The gradient is that of the kept values,
    so it differs from the gradient at ``x`` by the codes' rounding (2^-4 of a value at most, or
    2^-10 of its block's scale); a block that holds an infinity or a NaN has NaN gradients."""
    check_tensor("x", x, DTYPES, (-1, -1), None)
    if x.shape[1] < 2 or x.shape[1] % 2:
        raise ValueError(f"x has {x.shape[1]} columns, expected up and gate side by side")
    if x.requires_grad and torch.is_grad_enabled():
        return _Swiglu.apply(x)
    R, I = x.shape[0], x.shape[1] // 2
    y = torch.empty(R, I, dtype=x.dtype, device=x.device)
    call("moe_swiglu_forward", x.device, x.data_ptr(), R, I, DTYPES[x.dtype], y.data_ptr(), None, None)
    return y

"""GPU: results that are written into a given tensor, as autograd sees them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def calls(pkg, dev):
    """{name: (call of an output tensor, its shape)}"""
    torch.manual_seed(0)
    w13, w2 = (pkg.W4Weights(*pkg.quantize_w4(torch.randn(3, n, d, device=dev), 32), group_size=32)
               for n, d in ((64, 64), (64, 32)))
    x = torch.randn(5, 64, device=dev).bfloat16()
    off = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=dev)
    ids = torch.randint(0, 3, (5, 2), device=dev, dtype=torch.int32)
    weights = torch.rand(5, 2, device=dev)
    return {"w4_matvec": lambda out: pkg.w4_matvec(x, w13, off, out=out),
            "moe_w4": lambda out: pkg.moe_w4(x, ids, weights, w13, w2, output=out)}


@pytest.mark.parametrize("name", ["w4_matvec", "moe_w4"])
def test_overwriting_a_saved_tensor_is_noticed(name, pkg, cuda_dev):
    call = calls(pkg, cuda_dev)[name]
    out = torch.randn(5, 64, device=cuda_dev).bfloat16()
    a = torch.randn(5, 64, device=cuda_dev, dtype=torch.bfloat16, requires_grad=True)
    loss = (a * out).sum()                               # saves out for a's gradient
    with torch.no_grad():
        call(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("name", ["w4_matvec", "moe_w4"])
def test_outputs_that_require_a_gradient(name, pkg, cuda_dev):
    call = calls(pkg, cuda_dev)[name]
    want = call(torch.empty(5, 64, device=cuda_dev, dtype=torch.bfloat16))
    leaf = torch.zeros(5, 64, device=cuda_dev, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        call(leaf)
    assert not bool(leaf.any())                          # left as it was
    with torch.no_grad():
        assert torch.equal(call(leaf), want)
    with torch.inference_mode():
        assert torch.equal(call(torch.empty(5, 64, device=cuda_dev, dtype=torch.bfloat16)), want)

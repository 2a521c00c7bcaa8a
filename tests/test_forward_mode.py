"""Forward-mode derivatives: no operator has one, and each says so instead of dropping the tangent of a
dual tensor, which need not require a gradient."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad


def test_dual_tensors_are_refused_on_the_host(pkg):
    def dual(*shape, dtype=torch.float32):
        return forward_ad.make_dual(torch.zeros(shape, dtype=dtype), torch.ones(shape, dtype=dtype))
    ids = torch.zeros(4, 2, dtype=torch.int32)
    order = pkg.TokenOrder(torch.zeros(4, dtype=torch.int32), ids, torch.zeros(8, dtype=torch.int32))
    codes = torch.zeros(8, 16, dtype=torch.uint8)
    with forward_ad.dual_level():
        for call in (lambda: pkg.swiglu(dual(2, 8)), lambda: pkg.dispatch(dual(4, 8), order),
                     lambda: pkg.combine(dual(8, 8), torch.zeros(4, 2), order),
                     lambda: pkg.W4Weights(codes, dual(8, 1, dtype=torch.bfloat16), group_size=32)):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):   # tangents pass through no_grad
                call()
        with pytest.raises(ValueError, match="CUDA"):          # an ordinary tensor is judged as ever
            pkg.swiglu(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(pkg.swiglu, (torch.zeros(2, 8),), (torch.ones(2, 8),))


@pytest.mark.gpu
def test_dual_tensors_are_refused(pkg, cuda_dev):
    torch.manual_seed(0)
    T, K, H, I, E = 6, 2, 64, 32, 4
    ids = torch.randint(0, E, (T, K), device=cuda_dev, dtype=torch.int32)
    order = pkg.sort_tokens(ids, E)
    bf = dict(device=cuda_dev, dtype=torch.bfloat16)
    hidden, rows, x = torch.randn(T, H, **bf), torch.randn(T * K, H, **bf), torch.randn(T, 2 * I, **bf)
    weights = torch.rand(T, K, device=cuda_dev)
    w13, w2 = (pkg.W4Weights(*pkg.quantize_w4(torch.randn(E, n, d, device=cuda_dev), 32), group_size=32)
               for n, d in ((2 * I, H), (H, I)))
    calls = {
        "swiglu": (pkg.swiglu, (x,), (0,)),
        "dispatch": (lambda h: pkg.dispatch(h, order), (hidden,), (0,)),
        "combine": (lambda r, w: pkg.combine(r, w, order), (rows, weights), (0, 1)),
        "w4_matvec": (lambda r: pkg.w4_matvec(r, w13, order.offsets), (rows,), (0,)),
        "moe_w4": (lambda h, w: pkg.moe_w4(h, ids, w, w13, w2), (hidden, weights), (0, 1)),
    }
    for name, (fn, args, places) in calls.items():
        want = fn(*args)
        with forward_ad.dual_level():
            assert torch.equal(fn(*args), want), name          # an open level alone changes nothing
            for i in places:
                dual = list(args)
                dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                assert not dual[i].requires_grad
                with pytest.raises(ValueError, match="tangent"):
                    fn(*dual)
                with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                    fn(*dual)

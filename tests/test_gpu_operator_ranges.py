"""GPU: the operators around the expert products beyond the sizes of the other tests: both sides of the
thresholds between kernels in 16 bits, rows of more than 8192 columns, and more than 2^31 elements."""

from __future__ import annotations

import pytest
import torch

import test_gpu_tokens as tokens
import test_gpu_w4 as w4
from rounding import U32, assert_close

pytestmark = pytest.mark.gpu

FP32, FP16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("row_dtype,out_dtype", [(BF16, BF16), (FP16, FP16), (FP32, BF16)])
@pytest.mark.parametrize("T,K,H", [(1100, 8, 2056), (1100, 8, 7168), (300, 5, 1032), (257, 8, 4104), (300, 5, 520),
                                   (1025, 3, 2048), (1024, 8, 2056), (256, 8, 1032), (256, 2, 1024), (2100, 8, 4096)])
def test_combine_at_the_kernels_thresholds(T, K, H, row_dtype, out_dtype, pkg, cuda_dev):
    tokens.test_combine_and_its_gradients(T, K, 24, 16, 4, H, row_dtype, out_dtype, False, pkg, cuda_dev)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("E,N,D,group,rows", [(1, 40, 8224, 32, [5]), (2, 33, 14336, 64, [3, 17]), (1, 64, 20608, 128, [9]),
                                              (2, 16, 8192, 128, [1, 2])])
def test_w4_rows_of_many_columns(E, N, D, group, rows, zeros, dtype, pkg, cuda_dev):
    """A row's largest magnitude may lie anywhere, so also beyond what a CTA keeps in registers."""
    codes, scales, z = w4.make(E, N, D, group, zeros, dtype, cuda_dev, D)
    weights = pkg.W4Weights(codes, scales, z, group_size=group)
    ends = torch.tensor([0] + rows).cumsum(0)
    R = int(ends[-1])
    x = torch.randn(R, D, generator=torch.Generator(device=cuda_dev).manual_seed(D), device=cuda_dev)
    x[0, D - 3] = 3e4                                # with bf16 the row's scale goes by this one
    if R > 1:
        x[1, 8190], x[1, D - 1] = -2e4, 2e3
    x = x.to(dtype)
    dense = w4.dense(codes, scales, z, group)
    y = pkg.w4_matvec(x, weights, ends.to(torch.int32).to(cuda_dev), out_dtype=FP32)
    w4.check(y, x, dense, ends.tolist(), FP32, D)


@pytest.mark.parametrize("H", [7168, 7167])
def test_more_than_2_31_elements_of_rows(H, pkg, cuda_dev):
    T, K, E = 40000, 8, 64
    assert T * K * H > 2 ** 31
    g = torch.Generator(device=cuda_dev).manual_seed(H)
    ids = torch.randint(0, E + 4, (T, K), generator=g, device=cuda_dev, dtype=torch.int32)
    order = pkg.sort_tokens(ids, E)
    hidden = torch.randn(T, H, generator=g, device=cuda_dev, dtype=BF16).requires_grad_(True)
    rows = pkg.dispatch(hidden, order)
    n = int(order.offsets[-1])
    for a in (0, 2 ** 31 // H - 500, n - 600, T * K - 300):   # the first rows, around 2^31 elements, the last ones
        part, tok = rows[a:a + 1000], order.row_token[a:a + 1000].long()
        assert torch.equal(part, torch.where((tok >= 0).unsqueeze(1), hidden[tok.clamp_min(0)], 0.0))
    # the gradient for the rows themselves: a token's row as often as it was picked, exact in fp32
    got, = torch.autograd.grad(rows, hidden, rows.detach())
    times = (order.inv_row >= 0).sum(1, keepdim=True)
    assert torch.equal(got, (hidden.detach().float() * times).to(BF16))
    del got

    rows = rows.detach().requires_grad_(True)
    weights = torch.rand(T, K, generator=g, device=cuda_dev).requires_grad_(True)
    out = pkg.combine(rows, weights, order)
    here = order.inv_row >= 0
    total = (weights.detach().double() * here).sum(1, keepdim=True)
    h = hidden.detach()
    for a in (0, T - 500):
        ref = h[a:a + 500].double() * total[a:a + 500]
        assert_close(out.detach()[a:a + 500], ref, BF16, K * U32 * ref.abs(), "out")
    grad_rows, grad_w = torch.autograd.grad(out, (rows, weights), h)
    for a in (0, T - 500):
        mine, gr = order.inv_row[a:a + 500], h[a:a + 500].double()
        want = weights.detach()[a:a + 500].double().unsqueeze(2) * gr.unsqueeze(1)
        row = torch.where(mine >= 0, mine, -1 - mine).long()
        want = torch.where((mine >= 0).unsqueeze(2), want, 0.0)
        assert_close(grad_rows[row], want, BF16, U32 * want.abs(), "grad_rows")
        square = (gr * gr).sum(1, keepdim=True) * (mine >= 0)
        assert_close(grad_w[a:a + 500], square, FP32, ((H + 31) // 32 + 16) * U32 * square, "grad_weights")


def test_more_than_2_31_elements_of_swiglu(pkg, cuda_dev):
    """A row's values do not depend on the others, so the rows around 2^31 elements and the last ones have
    what they have alone."""
    R, I = 300000, 4096
    assert R * 2 * I > 2 ** 31
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    x = torch.randn(R, 2 * I, generator=g, device=cuda_dev, dtype=BF16)
    grad = torch.randn(R, I, generator=g, device=cuda_dev, dtype=BF16)
    x.requires_grad_(True)
    y = pkg.swiglu(x)
    dx, = torch.autograd.grad(y, x, grad)
    for a in (0, 2 ** 31 // (2 * I) - 20, 2 ** 30 // I, R - 37):
        few = x.detach()[a:a + 37].clone().requires_grad_(True)
        alone = pkg.swiglu(few)
        assert torch.equal(y.detach()[a:a + 37], alone.detach())
        assert torch.equal(dx[a:a + 37], torch.autograd.grad(alone, few, grad[a:a + 37])[0])
    with torch.no_grad():
        assert torch.equal(pkg.swiglu(x), y)


def test_more_than_2_32_bytes_of_4_bit_weights(pkg, cuda_dev):
    E, N, D, group = 65, 8192, 16384, 128
    codes, scales, z = w4.make(E, N, D, group, True, BF16, cuda_dev, 2)
    assert codes.numel() > 2 ** 32
    weights = pkg.W4Weights(codes, scales, z, group_size=group)
    x = torch.randn(E, D, generator=torch.Generator(device=cuda_dev).manual_seed(3), device=cuda_dev, dtype=BF16)
    y = pkg.w4_matvec(x, weights, torch.arange(E + 1, dtype=torch.int32, device=cuda_dev))
    for e in (0, E - 2, E - 1):
        dense = w4.dense(codes[e:e + 1], scales[e:e + 1], z[e:e + 1], group)
        w4.check(y[e:e + 1], x[e:e + 1], dense, [0, 1], BF16, D)


def test_more_than_2_31_elements_of_4_bit_products(pkg, cuda_dev):
    R, N, D, group = 300000, 8192, 128, 128
    codes, scales, _ = w4.make(1, N, D, group, False, BF16, cuda_dev, 4)
    weights = pkg.W4Weights(codes, scales, group_size=group)
    x = torch.randn(R, D, generator=torch.Generator(device=cuda_dev).manual_seed(5), device=cuda_dev, dtype=BF16)
    y = pkg.w4_matvec(x, weights, torch.tensor([0, R - 5], dtype=torch.int32, device=cuda_dev))
    dense = w4.dense(codes, scales, None, group)
    for a in (0, 2 ** 31 // N - 50, R - 105):
        w4.check(y[a:a + 100], x[a:a + 100], dense, [0, 100], BF16, D)
    assert not bool(y[R - 5:].any())

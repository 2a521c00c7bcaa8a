"""GPU: tokens sorted by expert and back, against a walk over the pairs on the
host and sums in 64 bits."""

from __future__ import annotations

import pytest
import torch

from rounding import U32, assert_close

pytestmark = pytest.mark.gpu

INT_MIN = -2 ** 31


def order_on_host(ids, E, first):
    T, K = ids.shape
    places = [[] for _ in range(E + 1)]
    for p, i in enumerate(ids.reshape(-1).tolist()):
        places[i - first if first <= i < first + E else E].append(p)
    offsets, inv, token, row = [0], [0] * (T * K), [], 0
    for e, mine in enumerate(places):
        for p in mine:
            inv[p] = row if e < E else -1 - row
            token.append(p // K if e < E else -1)
            row += 1
        if e < E:
            offsets.append(row)
    i32 = torch.int32
    return (torch.tensor(offsets, dtype=i32), torch.tensor(inv, dtype=i32).view(T, K),
            torch.tensor(token, dtype=i32))


def make_ids(T, K, total, seed, dev):
    """Random picks with repeats inside a token, popular experts, and ids that are no expert's."""
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(T, K, generator=g) ** 2 * total).long().clamp_max(total - 1)
    odd = torch.rand(T, K, generator=g)
    ids[odd < 0.03] = -1
    ids[(odd >= 0.03) & (odd < 0.05)] = INT_MIN
    ids[(odd >= 0.05) & (odd < 0.07)] = 2 ** 31 - 1
    return ids.to(torch.int32).to(dev)


@pytest.mark.parametrize("T,K,total,E,first", [
    (0, 8, 256, 256, 0), (1, 1, 1, 1, 0), (1, 8, 256, 256, 0), (3, 8, 256, 32, 64), (31, 1, 5, 5, 0),
    (33, 8, 256, 256, 0), (129, 7, 60, 30, 17), (512, 8, 256, 256, 0), (513, 8, 256, 256, 0),
    (1000, 20, 1024, 1024, 0), (4099, 8, 256, 64, 192), (70001, 2, 40, 39, 0), (64, 64, 16, 4, 16),
])
def test_sort_tokens(T, K, total, E, first, pkg, cuda_dev):
    ids = make_ids(T, K, total, T + K, cuda_dev)
    order = pkg.sort_tokens(ids, E, first)
    for got, want, name in zip(order, order_on_host(ids, E, first), order._fields):
        assert torch.equal(got.cpu(), want), name
    again = pkg.sort_tokens(ids, E, first)
    assert all(torch.equal(a, b) for a, b in zip(order, again))


def misaligned(t):
    """The same contiguous values, one element past an allocation's start."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    return out


SHAPES = [  # T, K, total, E, first, H
    (1, 8, 256, 256, 0, 7168), (5, 3, 8, 8, 0, 1), (37, 8, 64, 64, 0, 1030), (64, 1, 16, 16, 0, 2048),
    (130, 12, 60, 30, 17, 257), (300, 5, 60, 60, 0, 96), (9, 4, 16, 4, 100, 512), (513, 2, 4, 2, 1, 1001),
    (40, 8, 32, 16, 8, 4100), (4099, 8, 64, 32, 16, 1040), (8200, 3, 12, 12, 0, 520), (1100, 8, 8, 6, 1, 2048),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K,total,E,first,H", SHAPES)
@pytest.mark.parametrize("shift", [False, True])
def test_dispatch_and_its_gradient(T, K, total, E, first, H, dtype, shift, pkg, cuda_dev):
    torch.manual_seed(T * H)
    ids = make_ids(T, K, total, H, cuda_dev)
    order = pkg.sort_tokens(ids, E, first)
    hidden = torch.randn(T, H, device=cuda_dev).to(dtype)
    grad = torch.randn(T * K, H, device=cuda_dev).to(dtype)
    if shift:
        hidden, grad = misaligned(hidden), misaligned(grad)
    hidden.requires_grad_(True)
    rows = pkg.dispatch(hidden, order)
    n, tok = int(order.offsets[-1]), order.row_token.long()
    want = torch.zeros(T * K, H, dtype=dtype, device=cuda_dev)
    want[:n] = hidden.detach()[tok[:n]]
    assert torch.equal(rows, want)
    got, = torch.autograd.grad(rows, hidden, grad)
    ref = torch.zeros(T, H, dtype=torch.float64, device=cuda_dev).index_add_(0, tok[:n], grad[:n].double())
    mag = torch.zeros(T, H, dtype=torch.float64, device=cuda_dev).index_add_(0, tok[:n], grad[:n].double().abs())
    assert_close(got, ref, dtype, K * U32 * mag, "gradient")


@pytest.mark.parametrize("row_dtype,out_dtype", [
    (torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
    (torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("T,K,total,E,first,H", SHAPES)
@pytest.mark.parametrize("shift", [False, True])
def test_combine_and_its_gradients(T, K, total, E, first, H, row_dtype, out_dtype, shift, pkg, cuda_dev):
    torch.manual_seed(T + H)
    ids = make_ids(T, K, total, H + 1, cuda_dev)
    order = pkg.sort_tokens(ids, E, first)
    rows = torch.randn(T * K, H, device=cuda_dev).to(row_dtype)
    n = int(order.offsets[-1])
    rows[n:] = float("nan")                          # rows of no expert are not read
    w = torch.randn(T, K, device=cuda_dev)
    grad = torch.randn(T, H, device=cuda_dev).to(out_dtype)
    if shift:
        rows, grad, w = misaligned(rows), misaligned(grad), misaligned(w)
    rows.requires_grad_(True)
    w.requires_grad_(True)
    out = pkg.combine(rows, w, order, out_dtype=out_dtype)
    here = order.inv_row >= 0
    picked = torch.where(here.unsqueeze(2), rows.detach()[order.inv_row.clamp_min(0).long()].double(), 0.0)
    wd = (w.detach().double() * here).unsqueeze(2)
    assert_close(out.detach(), (picked * wd).sum(1), out_dtype, K * U32 * (picked * wd).abs().sum(1), "out")
    grad_rows, grad_w = torch.autograd.grad(out, (rows, w), grad)
    g = grad.double().unsqueeze(1)
    ref = torch.zeros(T * K, H, dtype=torch.float64, device=cuda_dev)
    ref[order.inv_row[here].long()] = (g * wd)[here]
    # one fp32 product, then the type
    assert_close(grad_rows, ref, row_dtype, U32 * ref.abs(), "grad_rows")
    assert not bool(grad_rows[n:].any())
    # a thread's chain is at most ceil(H / 32) products, then at most 5 + 4 sums over the threads
    chain = (H + 31) // 32 + 16
    assert_close(grad_w, (picked * g).sum(2), torch.float32, chain * U32 * (picked * g).abs().sum(2), "grad_weights")


def test_gradients_agree_with_differences(pkg, cuda_dev):
    """The gradient of a weighted sum of the outputs, against central differences (the outputs are linear
    in rows and in weights, so the difference has rounding errors only)."""
    torch.manual_seed(3)
    T, K, H = 6, 3, 40
    order = pkg.sort_tokens(make_ids(T, K, 6, 1, cuda_dev), 4, 1)
    rows = torch.randn(T * K, H, device=cuda_dev, requires_grad=True)
    w = torch.randn(T, K, device=cuda_dev, requires_grad=True)
    c = torch.randn(T, H, device=cuda_dev)

    def loss(r, v):
        return (pkg.combine(r, v, order).double() * c.double()).sum()

    grads = torch.autograd.grad(loss(rows, w), (rows, w))
    for leaf, grad in zip((rows, w), grads):
        step = torch.randn_like(leaf).sign() * 0.5
        with torch.no_grad():
            up = loss(leaf + step, w) if leaf is rows else loss(rows, leaf + step)
            down = loss(leaf - step, w) if leaf is rows else loss(rows, leaf - step)
        # each loss sums T * H outputs with |out| below 60 here, each off by at most K * 2^-24 of its terms
        assert abs(float(up - down) - 2 * float((grad.double() * step.double()).sum())) < T * H * 60 * 8 * U32


def test_broadcast_gradient_and_skipped_gradients(pkg, cuda_dev):
    """sum().backward() hands an expanded gradient; a leaf that needs none gets none."""
    T, K, H = 12, 2, 64
    order = pkg.sort_tokens(make_ids(T, K, 4, 2, cuda_dev), 4)
    w = torch.rand(T, K, device=cuda_dev)
    rows = torch.randn(T * K, H, device=cuda_dev, requires_grad=True)
    pkg.combine(rows, w, order).sum().backward()
    here = (order.inv_row >= 0)
    want = torch.zeros(T * K, device=cuda_dev)
    want[order.inv_row[here].long()] = w[here]
    assert torch.equal(rows.grad, want.unsqueeze(1).expand(-1, H))
    w.requires_grad_(True)
    pkg.combine(rows.detach(), w, order).sum().backward()
    assert torch.equal(w.grad != 0, here)
    hidden = torch.randn(T, H, device=cuda_dev, requires_grad=True)
    pkg.dispatch(hidden, order).sum().backward()
    assert torch.equal(hidden.grad, here.sum(1, keepdim=True).float().expand(-1, H))


def test_no_tokens(pkg, cuda_dev):
    order = pkg.sort_tokens(torch.empty(0, 4, dtype=torch.int32, device=cuda_dev), 6)
    assert order.offsets.tolist() == [0] * 7
    hidden = torch.empty(0, 32, device=cuda_dev, requires_grad=True)
    rows = pkg.dispatch(hidden, order)
    w = torch.empty(0, 4, device=cuda_dev, requires_grad=True)
    out = pkg.combine(rows, w, order)
    assert rows.shape == (0, 32) and out.shape == (0, 32)
    out.sum().backward()
    assert hidden.grad.shape == (0, 32) and w.grad.shape == (0, 4)


def test_streams_and_graph_replay(pkg, cuda_dev):
    """Captured on a side stream and replayed with new inputs; eager calls on another stream in between."""
    T, K, H, E = 77, 4, 520, 16
    g = torch.Generator(device=cuda_dev).manual_seed(0)

    def fresh():
        return (torch.randint(0, 20, (T, K), generator=g, device=cuda_dev, dtype=torch.int32),
                torch.randn(T, H, generator=g, device=cuda_dev).bfloat16(),
                torch.rand(T, K, generator=g, device=cuda_dev),
                torch.randn(T, H, generator=g, device=cuda_dev).bfloat16())

    def step(ids, hidden, w, grad):
        order = pkg.sort_tokens(ids, E)
        rows = pkg.dispatch(hidden, order)
        out = pkg.combine(rows, w, order)
        return (out.detach(), *torch.autograd.grad(out, (hidden, w), grad))

    bufs = fresh()
    bufs[1].requires_grad_(True)
    bufs[2].requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*bufs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(*bufs)
    torch.cuda.current_stream().wait_stream(side)
    other = torch.cuda.Stream()
    for _ in range(3):
        new = fresh()
        with torch.no_grad():
            for b, v in zip(bufs, new):
                b.copy_(v)
        other.wait_stream(torch.cuda.current_stream())
        new[1].requires_grad_(True)
        new[2].requires_grad_(True)
        graph.replay()
        with torch.cuda.stream(other):
            want = step(*new)
        torch.cuda.current_stream().wait_stream(other)
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
    torch.cuda.synchronize()


def test_ids_at_the_ends_of_their_range(pkg, cuda_dev):
    E = 5
    first = 2 ** 31 - 1 - E
    ids = torch.tensor([[first, INT_MIN], [INT_MIN + 1, 2 ** 31 - 2], [-1, 2 ** 31 - 1]], dtype=torch.int32, device=cuda_dev)
    order = pkg.sort_tokens(ids, E, first)
    for got, want in zip(order, order_on_host(ids.cpu(), E, first)):
        assert torch.equal(got.cpu(), want)


def test_no_second_derivative(pkg, cuda_dev):
    """A gradient may be asked for with a graph of its own, but that graph has no gradient and says so."""
    order = pkg.sort_tokens(torch.zeros(4, 1, dtype=torch.int32, device=cuda_dev), 2)
    x = torch.randn(4, 16, device=cuda_dev, requires_grad=True)
    w = torch.rand(4, 1, device=cuda_dev, requires_grad=True)
    for y in (pkg.dispatch(x, order), pkg.combine(x, w, order), pkg.swiglu(x)):
        first, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()


def test_refusals(pkg, cuda_dev):
    L = __import__("sys").modules["fib_b200._lib"]
    ids = torch.zeros(4, 2, dtype=torch.int32, device=cuda_dev)
    order = pkg.sort_tokens(ids, 3)
    with pytest.raises(TypeError):
        pkg.sort_tokens(ids.long(), 3)
    with pytest.raises(ValueError):
        pkg.sort_tokens(ids.view(-1), 3)
    with pytest.raises(ValueError):
        pkg.sort_tokens(ids.t(), 3)
    with pytest.raises(ValueError):
        pkg.sort_tokens(torch.zeros(4, 0, dtype=torch.int32, device=cuda_dev), 3)
    for E, first in ((3, 2 ** 32), (2 ** 32 + 3, 0)):
        with pytest.raises(ValueError):
            pkg.sort_tokens(ids, E, first)
    for E, first in ((0, 0), (-1, 0), (1025, 0), (3, -1), (3, 2 ** 31 - 3)):
        with pytest.raises(L.MoeError):
            pkg.sort_tokens(ids, E, first)
    x = torch.zeros(4, 16, device=cuda_dev)
    with pytest.raises(ValueError):
        pkg.dispatch(x[:3], order)
    with pytest.raises(ValueError):
        pkg.dispatch(x[:, ::2], order)
    with pytest.raises(TypeError):
        pkg.dispatch(x.double(), order)
    with pytest.raises(TypeError):
        pkg.dispatch(x, tuple(order))
    with pytest.raises(L.MoeError):
        pkg.dispatch(x[:, :0].contiguous(), order)
    rows = torch.zeros(8, 16, device=cuda_dev, dtype=torch.bfloat16)
    w = torch.zeros(4, 2, device=cuda_dev)
    with pytest.raises(ValueError):
        pkg.combine(rows[:7], w, order)
    with pytest.raises(ValueError):
        pkg.combine(rows, w[:3], order)
    with pytest.raises(TypeError):
        pkg.combine(rows, w.bfloat16(), order)
    with pytest.raises(TypeError):
        pkg.combine(rows, w, order, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        pkg.combine(rows, w.cpu(), order)

"""GPU: the layer's steps as a training step uses them, sort, dispatch, expert products, SwiGLU, expert
products and combine, against the whole's formula in 64 bits, outputs and all gradients."""

from __future__ import annotations

import pytest
import torch

from rounding import U32, assert_close
from test_gpu_swiglu import kept, sigmoid_error

pytestmark = pytest.mark.gpu


def eighths(shape, most, g, dev):
    """Random multiples of 1/8: products and short sums of them are exact in fp32."""
    return (torch.randint(-most, most + 1, shape, generator=g) / 8).to(dev)


def experts(x, w, offsets):
    """Rows of expert e times its matrix, zeros behind the last expert's rows."""
    o = offsets.tolist()
    parts = [x[a:b] @ m.T for a, b, m in zip(o, o[1:], w)]
    return torch.cat(parts + [x.new_zeros(x.shape[0] - o[-1], w.shape[1])])


@pytest.mark.parametrize("T,K,total,E,first,H,I", [(1, 1, 1, 1, 0, 16, 128), (29, 3, 6, 4, 1, 64, 130), (70, 4, 8, 8, 0, 40, 257)])
def test_training_step(T, K, total, E, first, H, I, pkg, cuda_dev):
    g = torch.Generator().manual_seed(T)
    ids = torch.rand(T, total, generator=g).topk(K).indices.to(torch.int32).to(cuda_dev)
    hidden = eighths((T, H), 8, g, cuda_dev).requires_grad_(True)
    w13 = eighths((E, 2 * I, H), 4, g, cuda_dev).requires_grad_(True)
    w2 = eighths((E, H, I), 4, g, cuda_dev).requires_grad_(True)
    weights = torch.rand(T, K, generator=g).to(cuda_dev).requires_grad_(True)
    grad = eighths((T, H), 8, g, cuda_dev)

    order = pkg.sort_tokens(ids, E, first)
    rows = pkg.dispatch(hidden, order)
    ug = experts(rows, w13, order.offsets)                    # exact: at most 64 multiples of 1/64 below 1
    out = pkg.combine(experts(pkg.swiglu(ug), w2, order.offsets), weights, order)
    got = torch.autograd.grad(out, (hidden, w13, w2, weights), grad)

    pairs = [(t, k, int(ids[t, k]) - first) for t in range(T) for k in range(K) if first <= int(ids[t, k]) < first + E]
    t, k, e = (torch.tensor(v, dtype=torch.long, device=cuda_dev) for v in (zip(*pairs) if pairs else ((), (), ())))
    h, a, b, w, gr = (v.detach().double() for v in (hidden, w13, w2, weights, grad))
    times = lambda x, m: torch.einsum("pj,pij->pi", x, m)     # a row for each pair, its expert's matrix
    back = lambda x, m: torch.einsum("pi,pij->pj", x, m)
    ug64 = times(h[t], a[e])
    up, gate = ug64[:, :I], ug64[:, I:]
    act = up * gate * torch.sigmoid(gate)
    act_err = act.abs() * (sigmoid_error(gate) + 3 * U32)     # sigmoid, two products
    down = times(act, b[e])
    down_err = times(act_err, b[e].abs()) + (I + 1) * U32 * times(act.abs(), b[e].abs())   # a sum of I
    wp = w[t, k].unsqueeze(1)

    def add(shape, at, v):
        return torch.zeros(shape, dtype=torch.float64, device=cuda_dev).index_put_(at, v, accumulate=True)

    assert_close(out.detach(), add((T, H), (t,), wp * down), torch.float32,
                 add((T, H), (t,), wp * (down_err + (K + 1) * U32 * down.abs())), "out")
    # gradients; the kept values are those of ug, which is exact
    d_down = wp * gr[t]                                       # one product
    d_act = back(d_down, b[e])
    d_act_err = (H + 3) * U32 * back(d_down.abs(), b[e].abs())
    v = kept(ug64.float(), I)
    u, q = v[:, :I], v[:, I:]
    sig, rel = torch.sigmoid(q), sigmoid_error(q)
    inner = 1 + q * (1 - sig)
    d_up, d_gate = d_act * q * sig, d_act * u * sig * inner
    err_inner = q.abs() * (sig * rel + U32) + 3 * U32 * (1 + q.abs())
    # d_act's error, the sigmoid's, the products', and the kept values' (one product of code and scale)
    up_err = (q * sig).abs() * (d_act_err + d_act.abs() * (rel + 4 * U32)) + 2 * U32 * (d_act * q * (1 + q.abs())).abs()
    gate_err = (u * sig * inner).abs() * (d_act_err + d_act.abs() * (rel + 5 * U32)) + (d_act * u * sig).abs() * err_inner + (
        4 * U32 * (d_act * u).abs() * (1 + q.abs()))
    d_ug, d_ug_err = torch.cat([d_up, d_gate], 1), torch.cat([up_err, gate_err], 1)
    n = 2 * I + K + T * K                                     # terms of the longest sum that follows
    want = (
        (add((T, H), (t,), back(d_ug, a[e])), add((T, H), (t,), back(d_ug_err + n * U32 * d_ug.abs(), a[e].abs()))),
        (add((E, 2 * I, H), (e,), torch.einsum("pi,pj->pij", d_ug, h[t])),
         add((E, 2 * I, H), (e,), torch.einsum("pi,pj->pij", d_ug_err + n * U32 * d_ug.abs(), h[t].abs()))),
        (add((E, H, I), (e,), torch.einsum("pi,pj->pij", d_down, act)),
         add((E, H, I), (e,), torch.einsum("pi,pj->pij", d_down.abs(), act_err + n * U32 * act.abs()))),
        (add((T, K), (t, k), (gr[t] * down).sum(1)),
         add((T, K), (t, k), (gr[t].abs() * (down_err + (H + 1) * U32 * down.abs())).sum(1))))
    for x, (ref, err), name in zip(got, want, ("hidden", "w13", "w2", "weights")):
        assert_close(x, ref, torch.float32, err, name)

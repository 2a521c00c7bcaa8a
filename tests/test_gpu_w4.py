"""GPU: products with 4-bit weights, and the layer made of them, in 64 bits."""

from __future__ import annotations

import sys

import pytest
import torch

from rounding import U32, assert_close, half_step

pytestmark = pytest.mark.gpu


def make(E, N, D, group, zeros, dtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    codes = torch.randint(0, 256, (E, N, D // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(E, N, D // group, generator=g, device=dev)) / D ** 0.5).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, device=dev, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def dense(codes, scales, zeros, group):
    """fp64 weights [E, N, D], and (code + zero) * |scale|: a product is made as sum of code * x minus zero *
    (sum of x), so these are the magnitudes of the terms that are added."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    z = zeros.double().repeat_interleave(group, -1) if zeros is not None else 8.0
    s = scales.double().repeat_interleave(group, -1)
    return (q - z) * s, (q + z) * s.abs()


def sum_error(D):
    """Roundings on the way of a product to the output, in units of 2^-24 of the terms' sum: the sum of x over a
    group (8 values, then a tree over 16 threads) and its product with the zero point; a tensor core step adds
    16 exact products and the sum so far with at least 24 bits each (17 units), at most 8 steps a group; then
    one for the scale and its sum for each group of a quarter of the columns, and 4 quarters or 8 eighths."""
    return 7 + 4 + 1 + 8 * 17 + (D // 32 + 3) // 4 + 4 + 8


def check(y, x, W, offsets, dtype, D):
    R = x.shape[0]
    W, M = W
    ref = torch.zeros(R, W.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(ref)
    for e in range(W.shape[0]):
        a, b = offsets[e], offsets[e + 1]
        ref[a:b] = x[a:b].double() @ W[e].t()
        mag[a:b] = x[a:b].double().abs() @ M[e].t()
    assert_close(y, ref, dtype, sum_error(D) * U32 * mag, "y")


CASES = [  # E, N, D, group, rows of each expert
    (1, 64, 64, 64, [1]), (1, 1, 32, 32, [3]), (1, 4096, 7168, 128, [1]), (1, 17, 96, 32, [8]),
    (3, 100, 128, 128, [0, 9, 0]), (5, 130, 192, 64, [16, 0, 17, 1, 33]), (4, 2048, 416, 32, [2, 31, 32, 70]),
    (40, 48, 256, 128, [1] * 40), (2, 7168, 2048, 128, [5, 24]), (3, 96, 640, 128, [25, 49, 23]), (2, 80, 384, 128, [32, 65]), (3, 16, 1024, 64, [0, 0, 0]),
    (300, 33, 64, 32, [i % 3 for i in range(300)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("E,N,D,group,rows", CASES)
def test_w4_matvec(E, N, D, group, rows, zeros, dtype, pkg, cuda_dev):
    codes, scales, z = make(E, N, D, group, zeros, dtype, cuda_dev, N + D)
    w = pkg.W4Weights(codes, scales, z, group_size=group)
    ends = torch.tensor([0] + rows).cumsum(0)
    R = int(ends[-1])
    x = torch.randn(R, D, device=cuda_dev).to(dtype)
    off = ends.to(torch.int32).to(cuda_dev)
    W = dense(codes, scales, z, group)
    y = pkg.w4_matvec(x, w, off)
    check(y, x, W, ends.tolist(), dtype, D)
    y32 = pkg.w4_matvec(x, w, off, out_dtype=torch.float32)
    check(y32, x, W, ends.tolist(), torch.float32, D)
    assert torch.equal(y32.to(dtype), y)                       # one rounding
    assert torch.equal(pkg.w4_matvec(x, w, off), y)            # the same every time
    if E == 1:
        single = pkg.W4Weights(codes[0], scales[0], z[0] if z is not None else None, group_size=group)
        assert torch.equal(pkg.w4_matvec(x, single), y)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,D,group", [(16, 128, 64), (20, 96, 32), (33, 256, 128), (1, 32, 32), (48, 192, 64), (150, 1184, 32)])
def test_layout_is_the_documented_one(N, D, group, zeros, pkg, cuda_dev):
    """Every code, scale and zero point is where the header says, padding is zero."""
    E = 2
    codes, scales, z = make(E, N, D, group, zeros, torch.float16, cuda_dev, N + D)
    w = pkg.W4Weights(codes, scales, z, group_size=group)
    n16, steps, groups = -(-N // 16), -(-D // 128), 128 // group
    size = 1024 + groups * (48 if zeros else 32)
    flat = w.layout.cpu().view(E, n16 * steps, size)
    rec = torch.empty(E, n16, steps, size, dtype=torch.uint8)
    at = 0
    for tile in range(0, n16, 8):
        for step in range(0, steps, 4):
            part = rec[:, tile:tile + 8, step:step + 4]
            part.copy_(flat[:, at:at + part.shape[1] * part.shape[2]].view(part.shape))
            at += part.shape[1] * part.shape[2]
    assert at == n16 * steps
    words = rec[..., :1024].contiguous().view(E, n16, steps, 2, 32, 16)
    got = torch.zeros(E, n16 * 16, steps * 128, dtype=torch.uint8)
    for lane in range(32):
        row, t = lane // 4, lane % 4
        for j in range(4):
            for i, k in enumerate((0, 2, 1, 3)):
                byte = words[:, :, :, :, lane, 4 * j + i]                      # [E, n16, steps, 2]
                c = 32 * (j // 2) + 8 * t + 4 * (j % 2) + k
                got[:, row::16, c::64] = (byte & 15).flatten(2)
                got[:, row + 8::16, c::64] = (byte >> 4).flatten(2)
    want = torch.zeros_like(got)
    want[:, :N, 0:D:2], want[:, :N, 1:D:2] = (codes & 15).cpu(), (codes >> 4).cpu()
    assert torch.equal(got, want)
    tail = rec[..., 1024:1024 + 32 * groups].contiguous().view(torch.float16)
    for part, plain in ((tail, scales), (rec[..., 1024 + 32 * groups:], z)):
        if plain is None:
            assert part.numel() == 0
            continue
        full = torch.zeros(E, n16 * 16, steps * groups, dtype=plain.dtype)
        full[:, :N, :D // group] = plain.cpu()
        part = part.reshape(E, n16, steps, 8, groups, 2).permute(0, 1, 5, 3, 2, 4)
        assert torch.equal(part.reshape(E, n16 * 16, -1), full)


def test_pruned_weights_and_outliers(pkg, cuda_dev):
    """Codes equal to their zero points, and a value far above its row's others that has no weight: within the
    roundings of code * x and zero * x, which do not cancel exactly."""
    torch.manual_seed(0)
    N, D = 40, 256
    z = torch.randint(0, 16, (1, N, D // 32), device=cuda_dev, dtype=torch.uint8)
    q = z.repeat_interleave(32, -1)
    s = torch.rand(1, N, D // 32, device=cuda_dev).bfloat16() + 1
    x = torch.randn(3, D, device=cuda_dev).bfloat16() * 1000
    off = torch.tensor([0, 3], dtype=torch.int32, device=cuda_dev)
    for codes, zeros in ((q[..., 0::2] | q[..., 1::2] << 4, z),
                         (torch.full((1, N, D // 2), 0x88, dtype=torch.uint8, device=cuda_dev), None)):
        w = pkg.W4Weights(codes, s, zeros, group_size=32)
        W = dense(codes, s, zeros, 32)
        assert not bool(W[0].any())
        check(pkg.w4_matvec(x, w, off), x, W, [0, 3], torch.bfloat16, D)
    codes = torch.full((1, N, D // 2), 0x88, dtype=torch.uint8, device=cuda_dev)
    codes[0, :, 5] = 0x89                                       # column 10 counts once, column 11 not at all
    w = pkg.W4Weights(codes, s, group_size=32)
    for small in (2.0 ** -20, 2.0 ** -6, 1.0):
        x = torch.zeros(1, D, device=cuda_dev).bfloat16()
        x[0, 10], x[0, 11] = 1.5 * small, 2.0 ** 8
        check(pkg.w4_matvec(x, w, out_dtype=torch.float32), x, dense(codes, s, None, 32), [0, 1], torch.float32, D)


@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -60, 2.0 ** 60, 2.0 ** 120])
def test_rows_of_any_size(size, pkg, cuda_dev):
    """bf16 rows at the ends of the type's range, next to ordinary ones."""
    codes, scales, z = make(1, 33, 128, 64, True, torch.bfloat16, cuda_dev, 3)
    w = pkg.W4Weights(codes, scales, z, group_size=64)
    x = torch.randn(4, 128, device=cuda_dev).bfloat16()
    x[1] *= size
    y = pkg.w4_matvec(x, w, out_dtype=torch.float32)
    check(y, x, dense(codes, scales, z, 64), [0, 4], torch.float32, 128)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinities(value, zeros, pkg, cuda_dev):
    """No finite products in the row of an infinity or a NaN, and no other row touched."""
    codes, scales, z = make(1, 64, 128, 64, zeros, torch.bfloat16, cuda_dev, 4)
    w = pkg.W4Weights(codes, scales, z, group_size=64)
    x = torch.randn(3, 128, device=cuda_dev).bfloat16()
    clean = pkg.w4_matvec(x, w)
    x[1, 7] = value
    y = pkg.w4_matvec(x, w)
    assert not bool(torch.isfinite(y[1]).any())
    assert torch.equal(y[0], clean[0]) and torch.equal(y[2], clean[2])


def test_rows_of_no_expert(pkg, cuda_dev):
    """Zero in a new result, untouched in a given one; a NaN row spoils no other."""
    codes, scales, _ = make(3, 70, 128, 64, False, torch.bfloat16, cuda_dev, 0)
    w = pkg.W4Weights(codes, scales, group_size=64)
    x = torch.randn(20, 128, device=cuda_dev).bfloat16()
    off = torch.tensor([4, 6, 6, 15], dtype=torch.int32, device=cuda_dev)
    y = pkg.w4_matvec(x, w, off)
    assert not bool(y[:4].any()) and not bool(y[15:].any()) and bool(y[4:15].any(1).all())
    given = torch.full((20, 70), 7.0, device=cuda_dev, dtype=torch.bfloat16)
    assert pkg.w4_matvec(x, w, off, out=given) is given
    assert torch.equal(given[4:15], y[4:15])
    assert bool((given[:4] == 7).all()) and bool((given[15:] == 7).all())
    x2 = x.clone()
    x2[5], x2[:4], x2[15:] = float("nan"), float("inf"), float("nan")
    y2 = pkg.w4_matvec(x2, w, off)
    assert bool(torch.isnan(y2[5]).all())
    keep = [i for i in range(20) if i != 5]
    assert torch.equal(y2[keep], y[keep])


@pytest.mark.parametrize("bad", [[0, 900, 2, 900], [-5, 3, -9, 2 ** 31 - 1], [10, 5, 3, 0], [-2 ** 31, 0, 6, 6]])
def test_offsets_outside_the_rows_stay_inside_the_output(bad, pkg, cuda_dev):
    codes, scales, _ = make(3, 48, 64, 32, False, torch.float16, cuda_dev, 0)
    w = pkg.W4Weights(codes, scales, group_size=32)
    x = torch.randn(9, 64, device=cuda_dev).half()
    room = torch.full((29, 48), 3.0, device=cuda_dev, dtype=torch.float16)
    pkg.w4_matvec(x, w, torch.tensor(bad, dtype=torch.int32, device=cuda_dev), out=room[10:19])
    assert bool((room[:10] == 3).all()) and bool((room[19:] == 3).all())


def test_misaligned_rows_and_streams(pkg, cuda_dev):
    codes, scales, z = make(2, 40, 160, 32, True, torch.bfloat16, cuda_dev, 1)
    w = pkg.W4Weights(codes, scales, z, group_size=32)
    x = torch.randn(11, 160, device=cuda_dev).bfloat16()
    off = torch.tensor([0, 3, 11], dtype=torch.int32, device=cuda_dev)
    y = pkg.w4_matvec(x, w, off)
    moved = torch.cat([x.new_zeros(1), x.view(-1)])[1:].view(11, 160)
    assert torch.equal(pkg.w4_matvec(moved, w, off), y)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        with torch.cuda.stream(s):
            outs += [pkg.w4_matvec(x, w, off) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)
    assert sys.modules["fib_b200.kernel"].read_device_error(cuda_dev) == 0


def layer_inputs(T, K, total, E, first, H, I, dtype, dev, group=32, zeros=True):
    torch.manual_seed(T + H)
    a = make(E, 2 * I, H, group, zeros, dtype, dev, 1)
    b = make(E, H, I, group, zeros, dtype, dev, 2)
    hidden = torch.randn(T, H, device=dev).to(dtype)
    ids = torch.rand(T, total, device=dev).topk(K).indices.to(torch.int32)
    weights = torch.rand(T, K, device=dev)
    return hidden, ids, weights, a, b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,total,E,first,H,I", [(1, 8, 32, 32, 0, 256, 128), (21, 4, 16, 8, 5, 320, 160),
                                                  (64, 2, 40, 8, 32, 128, 192), (5, 1, 9, 3, 9, 64, 32)])
def test_moe_w4(T, K, total, E, first, H, I, dtype, pkg, cuda_dev):
    """The whole layer against 64 bits: the two intermediates are rounded to the type (u = half a step each),
    so silu(gate) * up is off by its own u, up's u and gate's u times |up| * |silu'| <= 1.1 |up|, and the
    second product carries that through |W2|."""
    hidden, ids, weights, a, b = layer_inputs(T, K, total, E, first, H, I, dtype, cuda_dev)
    w13, w2 = (pkg.W4Weights(*m, group_size=32) for m in (a, b))
    out = pkg.moe_w4(hidden, ids, weights, w13, w2, first)
    (W13, M13), (W2, M2) = dense(*a, 32), dense(*b, 32)
    u = torch.finfo(dtype).eps / 2
    ref = torch.zeros(T, H, dtype=torch.float64, device=cuda_dev)
    err = torch.zeros_like(ref)
    for t in range(T):
        for k in range(K):
            e = int(ids[t, k]) - first
            if not 0 <= e < E:
                continue
            h = hidden[t].double()
            z, zm = W13[e] @ h, M13[e] @ h.abs()
            dz = z.abs() * u + sum_error(H) * U32 * zm + half_step(torch.zeros(1, device=cuda_dev).double(), dtype)
            up, gate, dup, dgate = z[:I], z[I:], dz[:I], dz[I:]
            s = up * gate * torch.sigmoid(gate)
            ds = dup * (gate * torch.sigmoid(gate)).abs() + 1.1 * dgate * (up.abs() + dup) + s.abs() * (u + 64 * U32)
            ds = ds + half_step(torch.zeros(1, device=cuda_dev).double(), dtype) + dup * dgate
            ds = ds * (1 + u)
            w = float(weights[t, k])
            ref[t] += w * (W2[e] @ s)
            err[t] += w * (W2[e].abs() @ ds + sum_error(I) * U32 * (M2[e] @ (s.abs() + ds))) * (1 + K * 2 * U32)
    err = err + K * 2 * U32 * ref.abs()
    assert_close(out, ref, dtype, err, "layer")
    given = torch.full_like(out, float("nan"))
    assert pkg.moe_w4(hidden, ids, weights, w13, w2, first, output=given) is given
    assert torch.equal(given, out)


def test_moe_w4_captured_twice(pkg, cuda_dev):
    """Two graphs of different sizes captured from the same weights, replayed in turn and at once."""
    sizes = [(1, 4), (30, 4)]
    cases = [layer_inputs(T, K, 12, 12, 0, 256, 128, torch.bfloat16, cuda_dev) for T, K in sizes]
    w13, w2 = (pkg.W4Weights(*m, group_size=32) for m in cases[0][3:])
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for hidden, ids, weights, *_ in cases:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            pkg.moe_w4(hidden, ids, weights, w13, w2)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(pkg.moe_w4(hidden, ids, weights, w13, w2))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for step in range(4):
        for hidden, ids, weights, *_ in cases:
            hidden.copy_(torch.randn(hidden.shape, device=cuda_dev))
            ids.copy_(torch.rand(ids.shape[0], 12, device=cuda_dev).topk(ids.shape[1]).indices)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (hidden, ids, weights, *_), out in zip(cases, outs):
            assert torch.equal(out, pkg.moe_w4(hidden, ids, weights, w13, w2))


def test_moe_w4_without_tokens_or_experts(pkg, cuda_dev):
    hidden, ids, weights, m13, m2 = layer_inputs(5, 2, 8, 4, 0, 64, 32, torch.bfloat16, cuda_dev)
    w13, w2 = pkg.W4Weights(*m13, group_size=32), pkg.W4Weights(*m2, group_size=32)
    assert pkg.moe_w4(hidden[:0], ids[:0], weights[:0], w13, w2).shape == (0, 64)
    out = torch.full_like(hidden, 3.0)
    assert pkg.moe_w4(hidden, torch.full_like(ids, -1), weights, w13, w2, output=out) is out
    assert not bool(out.any())
    with pytest.raises(ValueError, match="gradient"):
        pkg.moe_w4(hidden, ids, weights.clone().requires_grad_(True), w13, w2)


def test_refusals(pkg, cuda_dev):
    codes, scales, _ = make(2, 32, 64, 32, False, torch.bfloat16, cuda_dev, 0)
    w = pkg.W4Weights(codes, scales, group_size=32)
    x = torch.zeros(4, 64, device=cuda_dev, dtype=torch.bfloat16)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda_dev)
    with pytest.raises(ValueError, match="gradient"):
        pkg.w4_matvec(x.clone().requires_grad_(True), w, off)
    with torch.no_grad():
        pkg.w4_matvec(x.clone().requires_grad_(True), w, off)
    for args, kw, err in [((x, w), {}, ValueError), ((x, w, off[:2]), {}, ValueError), ((x, w, off.long()), {}, TypeError),
                          ((x.half(), w, off), {}, TypeError), ((x.t().contiguous().t(), w, off), {}, ValueError),
                          ((x, w, off), {"out_dtype": torch.float16}, TypeError),
                          ((x, w, off), {"out": x}, ValueError), ((x, w, off.cpu()), {}, ValueError)]:
        with pytest.raises(err):
            pkg.w4_matvec(*args, **kw)
    for bad in ((codes, scales[0]), (codes[:, :, :8], scales), (codes, scales, torch.full(
            scales.shape, 16, dtype=torch.uint8, device=cuda_dev)), (codes, scales.cpu())):
        with pytest.raises(ValueError):
            pkg.W4Weights(*bad, group_size=32)
    with pytest.raises(ValueError):
        pkg.W4Weights(codes, scales, group_size=64)
    ids = torch.zeros(4, 1, dtype=torch.int32, device=cuda_dev)
    with pytest.raises(ValueError):
        pkg.moe_w4(x, ids, torch.zeros(4, 1, device=cuda_dev), w, w)

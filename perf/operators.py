"""What is timed of the operators around the expert products, and what they compute.

Four operators, each in its plain form (elementary torch operations in fp32)
and through the package:

* ``dispatch``  tokens sorted by expert (``sort_tokens``) and copied to their
                rows, with the gradient that adds a token's rows up again;
* ``combine``   expert rows back to token order with the routing weights
                applied, with the gradients of the rows and of the weights;
* ``swiglu``    silu(gate) * up between the two expert products, its input kept
                for the backward pass as e4m3 codes with one scale per 1x128
                block, and the input's gradient computed from those codes;
* ``w4``        products of few rows with 4-bit weights that have one scale (and
                possibly one zero point) per group, one matrix per expert.

Definitions.  ids [T, K] are global expert ids; an id outside [first, first + E)
is not on this shard.  The pairs (t, k) on the shard are ordered by expert, then
by t * K + k; the others follow in t * K + k order, so every pair has one of the
T * K rows.  ``inv_row[t, k]`` is a pair's row, or -1 - row for a pair that is not
on the shard; those rows are zero, have no weight and get zero gradients.
"""

import math

import torch

own = False

HIDDEN, INTER = 7168, 2048          # the layer's sizes
BLOCK, E4M3_MAX = 128, 448.0

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    from __graft_entry__ import load_package
    return load_package()


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoded token through a layer with all of its experts on this GPU
        dict(name="dispatch_decode_1", op="dispatch", T=1, K=8, total=256, E=256, first=0, H=HIDDEN, dtype="bf16",
             train=False),
        # a training micro-batch of 4096 tokens, all experts here
        dict(name="dispatch_train_4096", op="dispatch", T=4096, K=8, total=256, E=256, first=0, H=HIDDEN,
             dtype="bf16", train=True),
        # a shard with half of the experts, a small odd model in fp32
        dict(name="dispatch_train_odd", op="dispatch", T=777, K=5, total=60, E=30, first=17, H=1001, dtype="fp32",
             train=True),
        # a decode batch: fp32 rows of the down product, bf16 output
        dict(name="combine_decode_64", op="combine", T=64, K=8, total=256, E=256, first=0, H=HIDDEN, rows="fp32",
             dtype="bf16", train=False),
        # the same micro-batch as dispatch_train_4096, on its way back
        dict(name="combine_train_4096", op="combine", T=4096, K=8, total=256, E=256, first=0, H=HIDDEN, rows="bf16",
             dtype="bf16", train=True),
        # a shard with a quarter of the experts, an odd width in fp16
        dict(name="combine_train_odd", op="combine", T=1501, K=6, total=64, E=16, first=32, H=1030, rows="fp16",
             dtype="fp16", train=True),
        # between the two products of a decode batch of 64 tokens, 8 experts each, nothing kept
        dict(name="swiglu_decode_512", op="swiglu", R=512, I=INTER, dtype="bf16", train=False),
        # the micro-batch of 4096 tokens between its two expert products
        dict(name="swiglu_train_32768", op="swiglu", R=32768, I=INTER, dtype="bf16", train=True),
        # one token and one matrix: the first product of a dense or shared expert
        dict(name="w4_dense_1", op="w4", T=1, K=0, E=1, N=2 * INTER, D=HIDDEN, group=128, zeros=False, dtype="bf16"),
        # one token through 8 of 32 local experts, first product
        dict(name="w4_experts_1", op="w4", T=1, K=8, E=32, N=2 * INTER, D=HIDDEN, group=128, zeros=False,
             dtype="bf16"),
        # a decode batch on a shard: about two rows for each expert, second product, small groups with zero points
        dict(name="w4_experts_64", op="w4", T=64, K=1, E=32, N=HIDDEN, D=INTER, group=32, zeros=True, dtype="fp16"),
        # a decode batch with every expert of a small layer here: about 16 rows for each expert
        dict(name="w4_experts_512", op="w4", T=64, K=8, E=32, N=2 * INTER, D=HIDDEN, group=128, zeros=False,
             dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "swiglu", "w4"])
    if op in ("dispatch", "combine"):
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        total = rng.choice([8, 16, 60, 64, 128, 256])
        E = rng.choice([total, total, max(1, total // 2), max(1, total // 4)])
        K = rng.randint(1, min(8, total))
        H = rng.choice([HIDDEN, 4096, 2048, 1024, _spread(rng, 64, HIDDEN), 8 * _spread(rng, 8, HIDDEN // 8)])
        most = 4096 * 8 * HIDDEN * 2 // (K * H * 4)
        case = dict(op=op, T=_spread(rng, 1, min(8192, most)), K=K, total=total, E=E, first=rng.randint(0, total - E),
                    H=H, dtype=dtype, train=rng.random() < 0.7)
        if op == "combine":
            case["rows"] = rng.choice([dtype, "fp32"])
        return case
    if op == "swiglu":
        I = rng.choice([INTER, 1024, 512, 8 * _spread(rng, 2, INTER // 8), _spread(rng, 16, INTER)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 32768 * INTER * 2 // (I * SIZE[dtype])
        return dict(op=op, R=_spread(rng, 1, min(32768, most)), I=I, dtype=dtype, train=rng.random() < 0.7)
    group = rng.choice([32, 64, 128])
    N = rng.choice([2 * INTER, HIDDEN, 2048, _spread(rng, 64, 4096)])
    D = group * _spread(rng, 2, (INTER if N == HIDDEN else HIDDEN) // group)
    E = rng.choice([1, 8, 16, 32])
    K = 0 if E == 1 else rng.randint(1, 8)
    T = _spread(rng, 1, 16 if E == 1 else 64)
    if T * max(K, 1) > 16 * E:
        T = max(1, 16 * E // max(K, 1))
    return dict(op=op, T=T, K=K, E=E, N=N, D=D, group=group, zeros=rng.random() < 0.4,
                dtype=rng.choice(["bf16", "fp16"]))


# ------------------------------------------------------------------ inputs
def _routing(T, K, total, g):
    """Expert ids as a router picks them (ascending, some experts more popular) and their weights."""
    scores = torch.randn(T, total, generator=g, device="cuda") + torch.randn(total, generator=g, device="cuda") * 0.3
    top, ids = scores.topk(K, dim=1)
    ids, order = ids.sort(dim=1)
    w = torch.sigmoid(top).gather(1, order)
    return ids.to(torch.int32), w / w.sum(1, keepdim=True) * 2.5


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    st = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op in ("dispatch", "combine"):
        T, K, H = case["T"], case["K"], case["H"]
        ids, weights = _routing(T, K, case["total"], g)
        st["ids"] = ids
        if op == "dispatch":
            st["hidden"] = normal(T, H).to(dt)
            if case["train"]:
                st["grad_rows"] = normal(T * K, H).to(dt)
                st["hidden"].requires_grad_(own)
        else:
            st["rows"] = normal(T * K, H).to(DTYPES[case["rows"]])
            st["weights"] = weights
            if case["train"]:
                st["grad_out"] = normal(T, H).to(dt)
                st["rows"].requires_grad_(own)
                st["weights"].requires_grad_(own)
            # the order that the tokens were dispatched by is there already
            if own:
                st["order"] = _package().sort_tokens(ids, case["E"], case["first"])
            else:
                st["inv_row"] = _plain_sort(ids, case["E"], case["first"])[1]
    elif op == "swiglu":
        st["x"] = (normal(case["R"], 2 * case["I"]) * 1.5).to(dt)
        if case["train"]:
            st["grad_y"] = normal(case["R"], case["I"]).to(dt)
            st["x"].requires_grad_(own)
    else:
        T, K, E, N, D, G = (case[k] for k in ("T", "K", "E", "N", "D", "group"))
        R = T * max(K, 1)
        st["x"] = normal(R, D).to(dt)
        codes = torch.randint(0, 256, (E, N, D // 2), generator=g, device="cuda", dtype=torch.uint8)
        scales = ((0.5 + torch.rand(E, N, D // G, generator=g, device="cuda")) * (0.25 / math.sqrt(D))).to(dt)
        zeros = (torch.randint(4, 13, (E, N, D // G), generator=g, device="cuda", dtype=torch.uint8)
                 if case["zeros"] else None)
        st["offsets"] = None
        if K:
            ids = _routing(T, K, E, g)[0].reshape(-1).long()
            st["offsets"] = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
            st["offsets"][1:] = torch.zeros(E, dtype=torch.int64, device="cuda").index_add_(
                0, ids, torch.ones_like(ids)).cumsum(0).to(torch.int32)
        if own:
            st["weights"] = _package().W4Weights(codes, scales, zeros, group_size=G)
        else:
            st["codes"], st["scales"], st["zeros"] = codes, scales, zeros
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


def _own_dispatch(st, case):
    fib = _package()
    order = fib.sort_tokens(st["ids"], case["E"], case["first"])
    rows = fib.dispatch(st["hidden"], order)
    out = [order.offsets, order.inv_row, order.row_token, rows.detach()]
    if case["train"]:
        out += torch.autograd.grad(rows, st["hidden"], st["grad_rows"])
    return out


def _own_combine(st, case):
    out = _package().combine(st["rows"], st["weights"], st["order"], out_dtype=DTYPES[case["dtype"]])
    if not case["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, (st["rows"], st["weights"]), st["grad_out"])]


def _own_swiglu(st, case):
    y = _package().swiglu(st["x"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, st["x"], st["grad_y"])]


def _own_w4(st, case):
    return [_package().w4_matvec(st["x"], st["weights"], st["offsets"])]


_own = {"dispatch": _own_dispatch, "combine": _own_combine, "swiglu": _own_swiglu, "w4": _own_w4}


def _plain_sort(ids, E, first):
    T, K = ids.shape
    local = ids.reshape(-1).long() - first
    key = torch.where((local >= 0) & (local < E), local, E)
    pair = torch.sort(key, stable=True).indices
    at = torch.arange(T * K, device=ids.device)
    row = torch.empty_like(pair)
    row[pair] = at
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:E].cumsum(0)])
    inv_row = torch.where(key < E, row, -1 - row).view(T, K)
    row_token = torch.where(at < offsets[E], pair // K, -1)
    return offsets.to(torch.int32), inv_row.to(torch.int32), row_token.to(torch.int32)


def _plain_dispatch(st, case):
    offsets, inv_row, row_token = _plain_sort(st["ids"], case["E"], case["first"])
    hidden = st["hidden"]
    here = (row_token >= 0).unsqueeze(1)
    rows = torch.where(here, hidden[row_token.clamp_min(0).long()], hidden.new_zeros(()))
    out = [offsets, inv_row, row_token, rows]
    if case["train"]:
        grad = st["grad_rows"][inv_row.clamp_min(0).long()].float() * (inv_row >= 0).unsqueeze(2)
        out.append(grad.sum(1).to(hidden.dtype))
    return out


def _plain_combine(st, case):
    inv_row, w, rows = st["inv_row"], st["weights"], st["rows"]
    here = (inv_row >= 0)
    picked = rows[inv_row.clamp_min(0).long()].float() * here.unsqueeze(2)          # [T, K, H]
    out = (picked * w.unsqueeze(2)).sum(1).to(DTYPES[case["dtype"]])
    if not case["train"]:
        return [out]
    g = st["grad_out"].float()
    grad_w = (picked * g.unsqueeze(1)).sum(2)
    del picked
    grad_rows = torch.empty_like(rows)
    at = torch.where(here, inv_row, -1 - inv_row).reshape(-1).long()
    grad_rows[at] = (g.unsqueeze(1) * (w * here).unsqueeze(2)).to(rows.dtype).view(-1, rows.shape[1])
    return [out, grad_rows, grad_w]


def _plain_swiglu(st, case):
    x, I = st["x"], case["I"]
    up, gate = x[:, :I].float(), x[:, I:].float()
    y = (gate * torch.sigmoid(gate) * up).to(x.dtype)
    if not case["train"]:
        return [y]

    def kept(v):                                          # what the e4m3 codes and scales stand for
        pad = -I % BLOCK
        b = torch.cat([v, v.new_zeros(v.shape[0], pad)], dim=1).view(v.shape[0], -1, BLOCK)
        s = b.abs().amax(2, keepdim=True)
        s = s / torch.full_like(s, E4M3_MAX)              # a true division: by a plain number it is a product here
        s = torch.where(s > 0, s, torch.ones_like(s))
        return ((b / s).to(torch.float8_e4m3fn).float() * s).view(v.shape[0], -1)[:, :I]

    up, gate = kept(up), kept(gate)
    sig = torch.sigmoid(gate)
    g = st["grad_y"].float()
    grad = torch.cat([g * gate * sig, g * up * sig * (1 + gate * (1 - sig))], dim=1)
    return [y, grad.to(x.dtype)]


def _plain_w4(st, case):
    x, codes, G = st["x"].float(), st["codes"], case["group"]
    R, E, N, D = x.shape[0], case["E"], case["N"], case["D"]
    out = torch.zeros(R, N, device=x.device)
    at = torch.arange(R, device=x.device, dtype=torch.int32)
    for e in range(E):
        q = torch.stack([codes[e] & 15, codes[e] >> 4], dim=2).view(N, D // G, G).float()
        z = st["zeros"][e].float().unsqueeze(2) if st["zeros"] is not None else 8.0
        w = ((q - z) * st["scales"][e].float().unsqueeze(2)).view(N, D)
        mine = x
        if st["offsets"] is not None:
            mine = x * ((at >= st["offsets"][e]) & (at < st["offsets"][e + 1])).unsqueeze(1)
        out += mine @ w.t()
    return [out.to(st["x"].dtype)]


_plain = {"dispatch": _plain_dispatch, "combine": _plain_combine, "swiglu": _plain_swiglu, "w4": _plain_w4}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"dispatch": _exact_dispatch, "combine": _exact_combine, "swiglu": _exact_swiglu,
            "w4": _exact_w4}[case["op"]](st, case)


def _exact_order(ids, E, first):
    """(offsets, inv_row, row_token) by walking the pairs expert by expert, on the host."""
    T, K = ids.shape
    flat = ids.reshape(-1).tolist()
    places = [[] for _ in range(E + 1)]
    for p, i in enumerate(flat):
        places[i - first if first <= i < first + E else E].append(p)
    offsets, inv, token, row = [0], [0] * (T * K), [], 0
    for e in range(E + 1):
        for p in places[e]:
            inv[p] = row if e < E else -1 - row
            token.append(p // K if e < E else -1)
            row += 1
        if e < E:
            offsets.append(row)

    def tensor(v):
        return torch.tensor(v, dtype=torch.int32, device=ids.device)
    return tensor(offsets), tensor(inv).view(T, K), tensor(token)


def _exact_dispatch(st, case):
    offsets, inv_row, row_token = _exact_order(st["ids"], case["E"], case["first"])
    hidden, n = st["hidden"].double(), int(offsets[-1])
    rows = torch.zeros(case["T"] * case["K"], case["H"], dtype=torch.float64, device=hidden.device)
    rows[:n] = hidden.index_select(0, row_token[:n].long())
    out = [offsets, inv_row, row_token, rows]
    if case["train"]:
        out.append(torch.zeros_like(hidden).index_add_(0, row_token[:n].long(), st["grad_rows"][:n].double()))
    return out


def _exact_combine(st, case):
    offsets, inv_row, row_token = _exact_order(st["ids"], case["E"], case["first"])
    n, tok = int(offsets[-1]), row_token.long()
    rows = st["rows"].double()
    pair_of_row = torch.zeros(rows.shape[0], dtype=torch.int64, device=rows.device)
    flat = inv_row.reshape(-1).long()
    mine = (flat >= 0).nonzero().view(-1)
    pair_of_row[flat[mine]] = mine
    w = st["weights"].double().reshape(-1)[pair_of_row[:n]].unsqueeze(1)
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device=rows.device)
    out.index_add_(0, tok[:n], rows[:n] * w)
    if not case["train"]:
        return [out]
    g = st["grad_out"].double().index_select(0, tok[:n])
    grad_rows = torch.zeros_like(rows)
    grad_rows[:n] = g * w
    grad_w = torch.zeros(case["T"] * case["K"], dtype=torch.float64, device=rows.device)
    grad_w[pair_of_row[:n]] = torch.einsum("rh,rh->r", g, rows[:n])
    return [out, grad_rows, grad_w.view(case["T"], case["K"])]


def _exact_swiglu(st, case):
    I, parts, kept = case["I"], [], []
    for half in (0, 1):
        v = st["x"][:, half * I:(half + 1) * I].double()
        parts.append(v)
        if not case["train"]:
            continue
        val = torch.empty_like(v)
        for b in range(0, I, BLOCK):
            c = v[:, b:b + BLOCK]
            # the scale and the quotient are fp32 values by definition
            s = (c.abs().amax(1, keepdim=True) / E4M3_MAX).float().double()
            s[s == 0] = 1.0
            a = (c / s).float().double()
            exponent = (torch.frexp(a).exponent - 1).clamp_min(-6)         # e4m3: 3 bits, least exponent -6
            step = torch.ldexp(torch.ones_like(a), exponent - 3)
            val[:, b:b + BLOCK] = (torch.round(a / step) * step).clamp(-E4M3_MAX, E4M3_MAX) * s
        kept.append(val)
    up, gate = parts
    y = up * gate / (1 + torch.exp(-gate))
    if not case["train"]:
        return [y]
    up, gate = kept
    e = torch.exp(-gate)
    g = st["grad_y"].double()
    return [y, torch.cat([g * gate / (1 + e), g * up * (1 + e + gate * e) / (1 + e) ** 2], dim=1)]


def _exact_w4(st, case):
    x, E, N, D, G = st["x"].double(), case["E"], case["N"], case["D"], case["group"]
    ends = st["offsets"].tolist() if st["offsets"] is not None else [0, x.shape[0]]
    out = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        w = torch.empty(N, D, dtype=torch.float64, device=x.device)
        w[:, 0::2] = st["codes"][e].remainder(16).double()
        w[:, 1::2] = st["codes"][e].div(16, rounding_mode="floor").double()
        zero = st["zeros"][e].double() if st["zeros"] is not None else torch.full((N, D // G), 8.0, device=x.device)
        w -= zero.repeat_interleave(G, dim=1)
        w *= st["scales"][e].double().repeat_interleave(G, dim=1)
        out[a:b] = x[a:b] @ w.t()
    return [out]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op in ("dispatch", "combine"):
        T, K, H, s = case["T"], case["K"], case["H"], SIZE[case["dtype"]]
        pairs = T * K
        here = pairs * case["E"] / case["total"]           # rows on this shard, on average
        if op == "dispatch":
            nbytes = pairs * 4 + (case["E"] + 1 + 2 * pairs) * 4 + T * H * s + pairs * H * s
            flops = 0
            if case["train"]:
                nbytes += here * H * s + T * H * s
                flops = here * H
            return {"bytes": int(nbytes), "flops": int(flops)}
        r = SIZE[case["rows"]]
        nbytes = pairs * 8 + here * H * r + T * H * s
        flops = 2 * here * H
        if case["train"]:                                  # the rows are read again: the forward pass ended long before
            nbytes += pairs * 8 + T * H * s + here * H * r + pairs * H * r + pairs * 4
            flops += 3 * here * H
        return {"bytes": int(nbytes), "flops": int(flops)}
    if op == "swiglu":
        n, s = case["R"] * case["I"], SIZE[case["dtype"]]
        if not case["train"]:
            return {"bytes": n * 3 * s, "flops": 5 * n}
        kept = 2 * n + case["R"] * 2 * -(-case["I"] // BLOCK) * 4
        return {"bytes": n * 3 * s + kept + kept + n * s + 2 * n * s, "flops": 20 * n}
    T, K, E, N, D, G = (case[k] for k in ("T", "K", "E", "N", "D", "group"))
    R = T * max(K, 1)
    # experts that at least one token picks, on average
    active = E * (1 - (1 - K / E) ** T) if K else 1
    per_matrix = N * D / 2 + N * (D // G) * (3 if case["zeros"] else 2)
    return {"bytes": int(active * per_matrix + R * (D + N) * 2 + (4 * (E + 1) if K else 0)), "flops": 2 * R * N * D}

"""Expert products with 4-bit weights, for decoding.

Reading the experts' weights bounds a decode step of the layer, and 4-bit
weights with group scales are half as many bytes as its FP8 experts (what that
gives in time depends on the batch: with all of 256 experts here and 16 tokens
``moe_w4`` takes 475 us and ``kernel(...)`` 516, with 64 tokens 1040 and 925):

    w13 = W4Weights(*quantize_w4(w, group_size=128), group_size=128)   # once: [E, N, D] weights
    y   = w4_matvec(rows, w13, order.offsets)     # rows sorted by expert (sort_tokens, dispatch)
    out = moe_w4(hidden_states, topk_ids, topk_weights, w13, w2)       # the whole routed layer

For inference only: there is no gradient (``quantize_w4`` takes trained
parameters, and leaves no graph behind).  The reference has no weights below
8 bits.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._ops import DTYPES, INT32_MAX, call, check_output, check_tensor, refuse_tangent
from .activation import swiglu
from .tokens import _combine, dispatch, sort_tokens

GROUP_SIZES = (32, 64, 128)


@torch.no_grad()
def quantize_w4(w: torch.Tensor, group_size: int, zero_points: bool = False, dtype: torch.dtype = torch.bfloat16):
    """``(codes, scales, zeros)`` of weights ``w`` [..., N, D], each group of ``group_size`` columns to the
    nearest of 16 values: codes uint8 [..., N, D / 2] (column 2j in the low half of byte j), scales
    ``dtype`` [..., N, D / group_size] and, with ``zero_points``, zeros uint8 of the same shape (the code
    that stands for 0; without, it is 8 and ``zeros`` is None).  A scale that ``dtype`` cannot hold (fp16 ends
    at 65504), or one of an infinity or a NaN, is refused, which waits for the GPU."""
    if group_size < 2 or w.shape[-1] % group_size or group_size % 2:
        raise ValueError(f"{w.shape[-1]} columns do not split into groups of {group_size}")
    v = w.float().unflatten(-1, (-1, group_size))
    if zero_points:
        low, high = v.amin(-1).clamp_max(0), v.amax(-1).clamp_min(0)
        wanted = (high / 2 - low / 2) / 7.5                # high - low may leave fp32
    else:
        wanted = v.abs().amax(-1) / 7
    # Below the type's normal numbers, where its steps are no longer small, a scale is rounded up: down, the
    # group's ends would be clipped, or all of it lost with a scale of 0.
    info = torch.finfo(dtype)
    step = info.smallest_normal * info.eps
    wanted = torch.where(wanted < info.smallest_normal, (torch.ceil(wanted.double() / step) * step).float(), wanted)
    scales = torch.where(wanted == 0, torch.ones_like(wanted), wanted).to(dtype)
    if not bool(torch.isfinite(scales).all()):
        raise ValueError(f"weights whose scales are not finite in {dtype}")
    s = scales.float()
    zeros = torch.round(-low / s).clamp(0, 15) if zero_points else torch.full_like(s, 8)
    q = (torch.round(v / s.unsqueeze(-1)) + zeros.unsqueeze(-1)).clamp(0, 15).to(torch.uint8).flatten(-2)
    codes = q[..., 0::2] | (q[..., 1::2] << 4)
    return codes, scales, zeros.to(torch.uint8) if zero_points else None


class W4Weights:
    """One 4-bit matrix per expert (``codes`` uint8 [E, N, D / 2], or [N, D / 2] for a single matrix), laid
    out once for ``w4_matvec``.

    Column 2j of a row is the low half of its byte j.  A weight is ``(code - zero) * scale`` with
    ``scales`` [E, N, D / group_size] in fp16 or bf16, the type of the rows it will multiply, and
    ``zeros`` uint8 of the same shape (0 to 15) or None for 8 everywhere.  Scales of magnitude 2^-100 to 2^100
    keep all sums within fp32's normal numbers."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
                 group_size: int):
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size is {group_size}, expected one of {GROUP_SIZES}")
        for name, t, dtypes in (("codes", codes, (torch.uint8,)), ("scales", scales, (torch.float16, torch.bfloat16)),
                                ("zeros", zeros, (torch.uint8,))):
            if t is None and name == "zeros":
                continue
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype not in dtypes:
                raise TypeError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
            if t.dim() not in (2, 3) or t.dim() != codes.dim() or t.device != codes.device:
                raise ValueError(f"{name} must be [E, N, ...] or [N, ...], as and where the codes are")
            refuse_tangent(name, t)
        if codes.dim() == 2:
            codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
            zeros = zeros.unsqueeze(0) if zeros is not None else None
        E, N, D = codes.shape[0], codes.shape[1], codes.shape[2] * 2
        if E < 1 or N < 1 or D < 1 or D % group_size or max(E, N, D) > INT32_MAX:
            raise ValueError(f"codes of shape {tuple(codes.shape)} do not split into groups of {group_size} columns")
        for name, t in (("scales", scales), ("zeros", zeros)):
            if t is not None and t.shape != (E, N, D // group_size):
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(E, N, D // group_size)}")
        if not codes.is_cuda:
            raise ValueError("codes, scales and zeros must be CUDA tensors (no CPU path)")
        if zeros is not None and int(zeros.max()) > 15:
            raise ValueError("zeros must be 0 to 15")
        self.num_experts, self.n, self.d, self.group_size = E, N, D, group_size
        self.dtype, self.device, self.with_zeros = scales.dtype, codes.device, zeros is not None
        nbytes = ctypes.c_uint64(0)
        _lib.check(_lib.load().moe_w4_layout_size(E, N, D, group_size, int(self.with_zeros), ctypes.byref(nbytes)),
                   "moe_w4_layout_size")
        self.layout = torch.empty(nbytes.value, dtype=torch.uint8, device=self.device)
        codes, scales = codes.contiguous(), scales.contiguous()
        zeros = zeros.contiguous() if zeros is not None else None
        if codes.data_ptr() % 4:
            codes = codes.clone()
        call("moe_w4_lay_out", self.device, codes.data_ptr(), scales.data_ptr(),
             None if zeros is None else zeros.data_ptr(), E, N, D, group_size, self.layout.data_ptr())


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows, d):
    n = ctypes.c_uint64(0)
    _lib.check(_lib.load().moe_w4_workspace_size(rows, d, ctypes.byref(n)), "moe_w4_workspace_size")
    return int(n.value)


def w4_matvec(x: torch.Tensor, weights: W4Weights, offsets: torch.Tensor | None = None,
              out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``y[r] = W[e] x[r]`` for the rows ``offsets[e] <= r < offsets[e + 1]`` of each expert e ([R, N]), in
    fp32, rounded once to ``out_dtype`` (``x``'s type or fp32).

    ``x`` [R, D] has the weights' type; ``offsets`` int32 [E + 1] as ``sort_tokens`` gives them, None for a
    single matrix.  Rows outside ``[offsets[0], offsets[E])`` are zero in a new result and left as they
    were in a given ``out``.  The weights of each expert with rows are read once for up to 32 rows, so
    this is the product for decode batches; prefill batches want a GEMM.  A row of ``x`` with an infinity or a
    NaN has no finite products.  Equal calls give equal bits; a row's last bits may differ between calls with
    other rows beside it, since the order of its sums goes by the whole call's share for each SM."""
    if not isinstance(weights, W4Weights):
        raise TypeError("weights must be W4Weights")
    check_tensor("x", x, (weights.dtype,), (-1, weights.d), None)
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("w4_matvec has no gradient: detach x or call it under torch.no_grad()")
    dev = x.device
    if weights.device != dev:
        raise ValueError(f"weights are on {weights.device}, expected {dev}")
    if offsets is not None:
        check_tensor("offsets", offsets, (torch.int32,), (weights.num_experts + 1,), dev)
    elif weights.num_experts != 1:
        raise ValueError(f"{weights.num_experts} experts need offsets")
    R, fresh = x.shape[0], out is None
    if fresh:
        out_dtype = x.dtype if out_dtype is None else out_dtype
        if out_dtype not in (x.dtype, torch.float32):
            raise TypeError(f"out_dtype is {out_dtype}, expected {x.dtype} or torch.float32")
        out = torch.empty(R, weights.n, dtype=out_dtype, device=dev)
    else:
        check_tensor("out", out, (x.dtype, torch.float32) if out_dtype is None else (out_dtype,), (R, weights.n), dev)
        check_output("out", out)
    if x.data_ptr() % 16:
        x = x.clone()
    need = _workspace_bytes(R, weights.d)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    call("moe_w4_matvec", dev, x.data_ptr(), weights.layout.data_ptr(),
         None if offsets is None else offsets.data_ptr(), R, weights.num_experts, weights.n, weights.d,
         weights.group_size, int(weights.with_zeros), DTYPES[x.dtype], DTYPES[out.dtype], int(fresh), out.data_ptr(),
         workspace.data_ptr(), need)
    return out


def moe_w4(hidden_states: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, w13: W4Weights,
           w2: W4Weights, local_expert_offset: int = 0, output: torch.Tensor | None = None) -> torch.Tensor:
    """The routed layer with 4-bit experts: ``sum_k topk_weights[t, k] * W2[e] swiglu(W13[e] hidden[t])``
    over the experts ``e = topk_ids[t, k]`` on this shard ([T, H], the type of ``hidden_states``; written
    to ``output`` if given).  ``w13`` [E, 2 * I, H] holds up's rows, then gate's."""
    for name, w in (("w13", w13), ("w2", w2)):
        if not isinstance(w, W4Weights):
            raise TypeError(f"{name} must be W4Weights")
    if w13.num_experts != w2.num_experts or w13.n != 2 * w2.d:
        raise ValueError(f"w13 has {w13.num_experts} experts of {w13.n} rows, w2 {w2.num_experts} of {w2.d} columns")
    for name, t in (("hidden_states", hidden_states), ("topk_weights", topk_weights)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    if (hidden_states.requires_grad or topk_weights.requires_grad) and torch.is_grad_enabled():
        raise ValueError("moe_w4 has no gradient: detach its inputs or call it under torch.no_grad()")
    order = sort_tokens(topk_ids, w13.num_experts, local_expert_offset)
    T, K = topk_ids.shape
    check_tensor("topk_weights", topk_weights, (torch.float32,), (T, K), topk_ids.device)
    check_tensor("hidden_states", hidden_states, (w13.dtype,), (T, w13.d), topk_ids.device)
    if output is not None:
        check_tensor("output", output, (hidden_states.dtype,), (T, w2.n), topk_ids.device)
        check_output("output", output)
    rows = w4_matvec(dispatch(hidden_states, order), w13, order.offsets)
    # fp32 from the second product to the sum over k: one rounding, as in the fused layer
    down = w4_matvec(swiglu(rows), w2, order.offsets, out_dtype=torch.float32)
    return _combine(down, topk_weights, order.inv_row, hidden_states.dtype, output)

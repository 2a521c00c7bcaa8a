"""Tokens sorted by expert and back, for training and serving around any expert products.

    order = sort_tokens(topk_ids, num_local_experts, local_expert_offset)
    rows  = dispatch(hidden_states, order)            # [T * K, H], expert e's rows at offsets[e]:offsets[e + 1]
    ...                                               # the expert products
    out   = combine(rows, topk_weights, order)        # [T, H]

``dispatch`` and ``combine`` are differentiable (``combine`` in the rows and in
the weights).  All of it runs on the current stream without a host
synchronisation and may be captured in a CUDA graph.  The fused layer
(``kernel(...)``) keeps these steps inside its own launches
(``solution/python/kernel.cu:321-351, 809-839`` of the reference).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._ops import DTYPES, INT32_MAX, call, check_tensor, differentiable_once


class TokenOrder(NamedTuple):
    """Where each (token, pick) pair's row is.  A pair whose expert is not on the shard has a row
    behind the last expert's, and ``inv_row`` holds ``-1 - row`` for it."""
    offsets: torch.Tensor      # int32 [E + 1]: rows of local expert e are offsets[e] .. offsets[e + 1] - 1
    inv_row: torch.Tensor      # int32 [T, K]: row of a pair, or -1 - row
    row_token: torch.Tensor    # int32 [T * K]: token of a row, -1 behind the last expert


def sort_tokens(topk_ids: torch.Tensor, num_local_experts: int, local_expert_offset: int = 0) -> TokenOrder:
    """Order the T * K pairs of ``topk_ids`` (int32 [T, K], global expert ids) by local expert, then by
    token and pick.  Ids outside ``[local_expert_offset, local_expert_offset + num_local_experts)``,
    negative ones among them, are not on this shard.  At most 1024 experts."""
    check_tensor("topk_ids", topk_ids, (torch.int32,), (-1, -1), None)
    T, K = topk_ids.shape
    if K < 1:
        raise ValueError("topk_ids needs at least one pick a token")
    E, first = int(num_local_experts), int(local_expert_offset)
    if E > INT32_MAX or abs(first) > INT32_MAX:
        raise ValueError(f"experts {first} .. {first} + {E} are not numbered by int32 ids")
    dev = topk_ids.device
    offsets = torch.empty(E + 1 if E > 0 else 1, dtype=torch.int32, device=dev)
    inv_row = torch.empty_like(topk_ids)
    row_token = torch.empty(T * K, dtype=torch.int32, device=dev)
    call("moe_tokens_sort", dev, topk_ids.data_ptr(), T, K, E, first, offsets.data_ptr(),
         inv_row.data_ptr(), row_token.data_ptr())
    return TokenOrder(offsets, inv_row, row_token)


def _check_order(order, device):
    if not isinstance(order, TokenOrder):
        raise TypeError("order must be a TokenOrder (sort_tokens)")
    check_tensor("order.inv_row", order.inv_row, (torch.int32,), (-1, -1), device)
    return order.inv_row.shape


def _dispatch(hidden, inv_row):
    (T, K), H, dev = inv_row.shape, hidden.shape[1], hidden.device
    rows = torch.empty(T * K, H, dtype=hidden.dtype, device=dev)
    call("moe_tokens_dispatch", dev, hidden.data_ptr(), inv_row.data_ptr(), T, K, H, DTYPES[hidden.dtype],
         rows.data_ptr())
    return rows


def _combine(rows, weights, inv_row, out_dtype, out=None):
    (T, K), H, dev = inv_row.shape, rows.shape[1], rows.device
    if out is None:
        out = torch.empty(T, H, dtype=out_dtype, device=dev)
    call("moe_tokens_combine", dev, rows.data_ptr(), inv_row.data_ptr(),
         None if weights is None else weights.data_ptr(), T, K, H, DTYPES[rows.dtype], DTYPES[out_dtype],
         out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, inv_row):
        ctx.save_for_backward(inv_row)
        return _dispatch(hidden, inv_row)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_rows):
        inv_row, = ctx.saved_tensors
        return _combine(grad_rows.contiguous(), None, inv_row, grad_rows.dtype), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, inv_row, out_dtype):
        # the rows are needed only for the weights' gradient
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights, inv_row)
        ctx.rows_like = rows.shape, rows.dtype
        return _combine(rows, weights, inv_row, out_dtype)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_out):
        rows, weights, inv_row = ctx.saved_tensors
        shape, dtype = ctx.rows_like
        grad_out = grad_out.contiguous()
        dev = grad_out.device
        grad_rows = torch.empty(shape, dtype=dtype, device=dev) if ctx.needs_input_grad[0] else None
        grad_weights = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        call("moe_tokens_combine_backward", dev, grad_out.data_ptr(), None if rows is None else rows.data_ptr(),
             inv_row.data_ptr(), weights.data_ptr(), *inv_row.shape, shape[1], DTYPES[dtype], DTYPES[grad_out.dtype],
             None if grad_rows is None else grad_rows.data_ptr(),
             None if grad_weights is None else grad_weights.data_ptr())
        return grad_rows, grad_weights, None, None


def dispatch(hidden_states: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """Copy each token's row (``hidden_states`` [T, H], fp32, fp16 or bf16) to the rows of its K pairs:
    [T * K, H], expert by expert; rows of pairs that are not on the shard are zero.  The gradient adds
    a token's rows in fp32, in ascending pick order, and rounds once."""
    check_tensor("hidden_states", hidden_states, DTYPES, (-1, -1), None)
    T, _ = _check_order(order, hidden_states.device)
    if hidden_states.shape[0] != T:
        raise ValueError(f"hidden_states has {hidden_states.shape[0]} tokens, the order {T}")
    if hidden_states.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(hidden_states, order.inv_row)
    return _dispatch(hidden_states, order.inv_row)


def combine(rows: torch.Tensor, topk_weights: torch.Tensor, order: TokenOrder,
            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``out[t] = sum_k topk_weights[t, k] * rows[row of (t, k)]`` over the pairs on the shard, in fp32
    and ascending k, rounded once: [T, H].  ``rows`` [T * K, H] are fp32, fp16 or bf16, ``topk_weights``
    fp32 [T, K]; fp32 rows may be combined to another ``out_dtype``."""
    check_tensor("rows", rows, DTYPES, (-1, -1), None)
    T, K = _check_order(order, rows.device)
    if rows.shape[0] != T * K:
        raise ValueError(f"rows has {rows.shape[0]} rows, the order {T * K}")
    check_tensor("topk_weights", topk_weights, (torch.float32,), (T, K), rows.device)
    out_dtype = rows.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPES or (out_dtype != rows.dtype and rows.dtype != torch.float32):
        raise TypeError(f"rows of {rows.dtype} cannot be combined to {out_dtype}")
    if (rows.requires_grad or topk_weights.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(rows, topk_weights, order.inv_row, out_dtype)
    return _combine(rows, topk_weights, order.inv_row, out_dtype)

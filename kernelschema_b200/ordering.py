"""Tokens in the order of their experts, and back: what a mixture of experts does around its products, with gradients for training.

    order = route_sort(ids, num_experts)               # ids of `route_topk`
    rows = sort_tokens(x, order)                       # one expert's tokens after the other's: order.offsets are the segments
    y = unsort_tokens(experts(rows), order, weights)   # back, the routes' weights applied

`mm_8bit_grouped` takes the sorted rows and the offsets. Every computation runs in libb200moe.so."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ops import _ROW_TYPES, _here, _ptr, _row_stride, _stream, _unit_rows


class RouteOrder(NamedTuple):
    """Where the routes of T tokens with top_k experts each stand once sorted by expert (int32, on the device)."""
    offsets: torch.Tensor        # [E + 1] first row of each expert's segment; the last: rows that hold a route
    row_of: torch.Tensor         # [T, top_k] row of a route, -1 where its id is no expert
    route_of_row: torch.Tensor   # [T * top_k] t * top_k + k of a row, -1 behind the last segment


def route_sort(ids: torch.Tensor, num_experts: int) -> RouteOrder:
    """Stable counting sort of int32 expert ids [T, top_k]: within a segment rows ascend by token. Ids outside [0, num_experts) (other ranks'
    experts, -1) are no route; an expert twice in a token is two. num_experts <= 1024."""
    if ids.dim() != 2 or ids.dtype != torch.int32 or not ids.shape[1]:
        raise ValueError("ids must be int32 [T, top_k]")
    if not 0 < num_experts <= 1024:
        raise ValueError("num_experts must be in 1..1024")
    _here(ids)
    ids = _unit_rows(ids)
    t, k = ids.shape
    lib = _lib.load()
    made = torch.empty(num_experts + 1 + 2 * t * k, dtype=torch.int32, device=ids.device)      # one allocation for the three
    offsets, row_of, route_of_row = made.split((num_experts + 1, t * k, t * k))
    need = lib.b200moe_route_sort_workspace_bytes(t, k, num_experts)
    ws = torch.empty(need, dtype=torch.uint8, device=ids.device) if need > 0 else None
    _lib.check(lib.b200moe_route_sort(ids.data_ptr(), _row_stride(ids), t, k, num_experts, offsets.data_ptr(), row_of.data_ptr(), route_of_row.data_ptr(),
                                      _ptr(ws), max(need, 0), _stream()), "b200moe_route_sort")
    return RouteOrder(offsets, row_of.view(t, k), route_of_row)


def _check_order(order, tokens: int | None, rows: int | None) -> None:
    offsets, row_of = order.offsets, order.row_of
    if row_of.dim() != 2 or row_of.dtype != torch.int32 or offsets.dtype != torch.int32 or not row_of.is_contiguous() or not offsets.is_contiguous():
        raise ValueError("order must come from route_sort")
    if (tokens is not None and row_of.shape[0] != tokens) or (rows is not None and row_of.numel() != rows):
        raise ValueError(f"the order is of {row_of.shape[0]} tokens and {row_of.numel()} rows, the tensor has {tokens if rows is None else rows}")


def _launch_sort(x, offsets, row_of):
    t, k = row_of.shape
    x = _unit_rows(x)
    rows = torch.empty((t * k, x.shape[1]), dtype=x.dtype, device=x.device)
    size = x.element_size()
    _lib.check(_lib.load().b200moe_sort_rows(x.data_ptr(), _row_stride(x) * size, t, x.shape[1] * size, row_of.data_ptr(), k,
                                             offsets.data_ptr() + 4 * (offsets.numel() - 1), rows.data_ptr(), _stream()), "b200moe_sort_rows")
    return rows


def _launch_unsort(rows, row_of, weights):
    t, k = row_of.shape
    rows = _unit_rows(rows)
    y = torch.empty((t, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    _lib.check(_lib.load().b200moe_unsort_rows(rows.data_ptr(), _row_stride(rows), rows.shape[0], row_of.data_ptr(), _ptr(weights), t, k, rows.shape[1],
                                               _ROW_TYPES[rows.dtype], y.data_ptr(), y.shape[1], _stream()), "b200moe_unsort_rows")
    return y


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, row_of):
        ctx.save_for_backward(row_of)
        return _launch_sort(x, offsets, row_of)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        row_of, = ctx.saved_tensors
        return _launch_unsort(grad, row_of, None), None, None


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, offsets, row_of):
        ctx.save_for_backward(rows, weights, offsets, row_of)
        return _launch_unsort(rows, row_of, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, weights, offsets, row_of = ctx.saved_tensors
        t, k = row_of.shape
        grad, rows = _unit_rows(grad), _unit_rows(rows)
        grad_rows = torch.empty((t * k, rows.shape[1]), dtype=rows.dtype, device=rows.device) if ctx.needs_input_grad[0] else None
        grad_weights = torch.empty((t, k), dtype=torch.float32, device=rows.device) if weights is not None and ctx.needs_input_grad[1] else None
        _lib.check(_lib.load().b200moe_unsort_rows_backward(
            grad.data_ptr(), _row_stride(grad), rows.data_ptr(), _row_stride(rows), row_of.data_ptr(), _ptr(weights), t, k, rows.shape[1],
            _ROW_TYPES[rows.dtype], offsets.data_ptr() + 4 * (offsets.numel() - 1), _ptr(grad_rows), _ptr(grad_weights), _stream()),
            "b200moe_unsort_rows_backward")
        return grad_rows, grad_weights, None, None


def sort_tokens(x: torch.Tensor, order: RouteOrder) -> torch.Tensor:
    """rows[row_of[t, k]] = x[t] -> [T * top_k, H] in x's type, rows behind the last segment zero. x: [T, H] of any 1-, 2- or 4-byte type (8-bit rows,
    scales [T] as well). Differentiable where x is bf16, fp16 or fp32: the gradient of a token is the sum over its rows (fp32, rounded once)."""
    if x.dim() not in (1, 2) or x.element_size() > 4 or x.is_complex() or (x.dim() == 2 and not x.shape[1]):
        raise ValueError("sort_tokens expects [T, H] or [T] of a 1-, 2- or 4-byte type")
    _check_order(order, x.shape[0], None)
    _here(x, order.row_of, order.offsets)
    if x.dim() == 1:
        return sort_tokens(x.unsqueeze(1), order).squeeze(1)
    if torch.is_grad_enabled() and x.requires_grad:
        if x.dtype not in _ROW_TYPES:
            raise ValueError("sort_tokens has a gradient for bf16, fp16 and fp32 rows")
        return _Sort.apply(x, order.offsets, order.row_of)
    return _launch_sort(x, order.offsets, order.row_of)


def unsort_tokens(rows: torch.Tensor, order: RouteOrder, weights: torch.Tensor | None = None) -> torch.Tensor:
    """y[t] = sum_k weights[t, k] * rows[row_of[t, k]] -> [T, H] in the rows' type (bf16, fp16 or fp32), fp32 sums in ascending k, rounded once;
    a token without routes becomes 0, rows behind the last segment are not read. weights fp32 [T, top_k] or None (1). Differentiable in
    rows and weights: grad_rows = weight * grad_y (zero behind the last segment), grad_weights = <row, grad_y> in fp32 (0 without a route)."""
    if rows.dim() != 2 or rows.dtype not in _ROW_TYPES or not rows.shape[1]:
        raise ValueError("unsort_tokens expects bf16, fp16 or fp32 [T * top_k, H]")
    _check_order(order, None, rows.shape[0])
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != order.row_of.shape):
        raise ValueError(f"weights must be float32 {tuple(order.row_of.shape)}")
    _here(rows, order.row_of, order.offsets, weights)
    weights = None if weights is None else weights.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        return _Unsort.apply(rows, weights, order.offsets, order.row_of)
    return _launch_unsort(rows, order.row_of, weights)

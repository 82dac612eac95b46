"""Tokens in the order of their experts, and back: what a mixture of experts does around its products, with gradients for training.

    order = route_sort(ids, num_experts)               # ids of `route_topk`
    rows = sort_tokens(x, order)                       # one expert's tokens after the other's: order.offsets are the segments
    y = unsort_tokens(experts(rows), order, weights)   # back, the routes' weights applied

`mm_8bit_grouped` takes the sorted rows and the offsets. Every computation runs in libb200moe.so. In a CUDA graph the gradients are captured like the
rest; a call whose leaf still has a live graph that was built on the default stream is refused (capture with ``x.detach().requires_grad_()``). The derivatives
are those of reverse mode, once: an input, or an incoming gradient, with a tangent of forward mode (`torch.autograd.forward_ad`) is refused, and
`torch.func` transforms raise."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .ops import _calls


class RouteOrder(NamedTuple):
    """Where the routes of T tokens with top_k experts each stand once sorted by expert (int32, on the device)."""
    offsets: torch.Tensor        # [E + 1] first row of each expert's segment; the last: rows that hold a route
    row_of: torch.Tensor         # [T, top_k] row of a route, -1 where its id is no expert
    route_of_row: torch.Tensor   # [T * top_k] t * top_k + k of a row, -1 behind the last segment


def route_sort(ids: torch.Tensor, num_experts: int) -> RouteOrder:
    """Stable counting sort of int32 expert ids [T, top_k]: within a segment rows ascend by token. Ids outside [0, num_experts) (other ranks'
    experts, -1) are no route; an expert twice in a token is two. num_experts <= 1024."""
    return RouteOrder(*_calls().route_sort(ids, num_experts))


def sort_tokens(x: torch.Tensor, order: RouteOrder) -> torch.Tensor:
    """rows[row_of[t, k]] = x[t] -> [T * top_k, H] in x's type, rows behind the last segment zero. x: [T, H] of any 1-, 2- or 4-byte type (8-bit rows,
    scales [T] as well). Differentiable where x is bf16, fp16 or fp32: the gradient of a token is the sum over its rows (fp32, rounded once)."""
    return _calls().sort_tokens(x, order.offsets, order.row_of)


def unsort_tokens(rows: torch.Tensor, order: RouteOrder, weights: torch.Tensor | None = None) -> torch.Tensor:
    """y[t] = sum_k weights[t, k] * rows[row_of[t, k]] -> [T, H] in the rows' type (bf16, fp16 or fp32), fp32 sums in ascending k, rounded once;
    a token without routes becomes 0, rows behind the last segment are not read. weights fp32 [T, top_k] or None (1). Differentiable in
    rows and weights: grad_rows = weight * grad_y (zero behind the last segment), grad_weights = <row, grad_y> in fp32 (0 without a route)."""
    return _calls().unsort_tokens(rows, order.offsets, order.row_of, weights)

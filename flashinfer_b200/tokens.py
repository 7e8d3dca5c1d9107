"""Tokens sorted by expert and back, with the routing weights applied, and the gradients.

``sort_by_expert`` turns the routing's picks (``route``, or any top-k) into an ``ExpertOrder``;
``sort_tokens`` copies token rows into expert order, where one product per expert (for instance
``int8_expert_matmul`` with ``order.expert_base``) can run over them; ``unsort_tokens`` adds the
experts' output rows back up per token, each times its routing weight. The tables stay on the
device and nothing waits for it, so the whole run can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FmoeTokenOrder
from ._op import (DTYPE_TAG, F32, I32, INT_MAX, call, first, first_order_only, need, not_traced, ptr,
                  recording, written)


class ExpertOrder:
    """The row of every pick, and back. Made by ``sort_by_expert``; all tensors on one device.

    ``expert_base`` int32 [E+1]: first row of each local expert (a multiple of ``align``); the
    last entry is where the rows end. ``row_pick`` int32 [num_rows]: the flat pick ``t * top_k + k``
    of each row, -1 for a row without one (padding, and every row from ``expert_base[E]`` on).
    ``pick_row`` int32 [T, top_k]: the row of each pick, -1 if its expert is not local. Rows are
    ordered by expert, within an expert by pick. The attributes cannot be set: the library is given the
    tables' addresses once.
    """

    __slots__ = ("_tables", "_sizes", "_index", "_c", "_ref")

    def __init__(self, expert_base: torch.Tensor, row_pick: torch.Tensor, pick_row: torch.Tensor):
        index = first(pick_row, "pick_row", I32, 2)
        need(expert_base, "expert_base", index, None, I32)
        need(row_pick, "row_pick", index, None, I32)
        T, K = pick_row.shape
        if expert_base.dim() != 1 or not 2 <= expert_base.shape[0] <= 1025:
            raise ValueError(f"expert_base must hold 2..1025 rows, got {tuple(expert_base.shape)}")
        if K < 1 or row_pick.dim() != 1 or row_pick.shape[0] < T * K:
            raise ValueError(f"row_pick {tuple(row_pick.shape)} must hold a row for every pick of "
                             f"pick_row {(T, K)}")
        self._set(index, expert_base, row_pick, pick_row)

    def _set(self, index: int, expert_base, row_pick, pick_row) -> None:
        T, K = pick_row.shape
        rows = row_pick.shape[0]
        self._tables, self._sizes, self._index = (expert_base, row_pick, pick_row), (T, K, rows), index
        self._c = FmoeTokenOrder(T, K, expert_base.shape[0] - 1, rows, expert_base.data_ptr(),
                                 row_pick.data_ptr(), pick_row.data_ptr())
        self._ref = ctypes.byref(self._c)

    expert_base = property(lambda self: self._tables[0])
    row_pick = property(lambda self: self._tables[1])
    pick_row = property(lambda self: self._tables[2])
    num_tokens = property(lambda self: self._sizes[0])
    top_k = property(lambda self: self._sizes[1])
    num_rows = property(lambda self: self._sizes[2])
    device = property(lambda self: self._tables[2].device)


@lru_cache(maxsize=1024)
def _sizes(T: int, K: int, E: int, align: int) -> Tuple[int, int]:
    """Rows and scratch bytes of an order of these sizes."""
    rows, scratch = ctypes.c_int64(), ctypes.c_size_t()
    _lib.check(_lib.load().fmoe_sort_size(T, K, E, align, ctypes.byref(rows),
                                          ctypes.byref(scratch)), "fmoe_sort_size")
    return rows.value, scratch.value


def sort_by_expert(topk_ids: torch.Tensor, num_local_experts: int, local_expert_offset: int = 0,
                   *, align: int = 1) -> ExpertOrder:
    """The expert order of int32 picks ``topk_ids`` [T, top_k].

    Local are the experts [local_expert_offset, local_expert_offset + num_local_experts); picks of
    other ids (-1 = no pick) get no row. Every expert's rows start at a multiple of ``align``
    (1..1024). A token may pick the same expert twice: each pick has its own row. Stable: equal
    inputs give equal tables.
    """
    index = first(topk_ids, "topk_ids", I32, 2)
    T, K = topk_ids.shape
    if K < 1:
        raise ValueError("topk_ids needs at least one pick per token")
    if not 1 <= num_local_experts <= 1024:
        raise ValueError(f"num_local_experts must be 1..1024, got {num_local_experts}")
    if not 0 <= local_expert_offset <= INT_MAX:
        raise ValueError("local_expert_offset must not be negative, nor beyond int32, got "
                         f"{local_expert_offset}")
    if not 1 <= align <= 1024:
        raise ValueError(f"align must be 1..1024, got {align}")
    if T * K > INT_MAX:
        raise ValueError(f"topk_ids holds {T * K} picks: fewer than 2^31 rows are possible")
    rows, scratch_bytes = _sizes(T, K, num_local_experts, align)
    order = ExpertOrder.__new__(ExpertOrder)  # of tables that need no checks
    order._set(index, topk_ids.new_empty(num_local_experts + 1), topk_ids.new_empty(rows),
               topk_ids.new_empty((T, K)))
    scratch = topk_ids.new_empty(scratch_bytes // 4) if scratch_bytes else None
    call("fmoe_sort_by_expert", index, topk_ids.data_ptr(), local_expert_offset, align, order._ref,
         ptr(scratch), scratch_bytes)
    return order


def _rows_shape(x: torch.Tensor, n: int):
    return (n,) if x.dim() == 1 else (n, x.shape[1])


def _sort(x: torch.Tensor, order: ExpertOrder, output: Optional[torch.Tensor]) -> torch.Tensor:
    given = output is not None
    if not given:
        output = x.new_empty(_rows_shape(x, order.num_rows))
    row_bytes = x.element_size() * (1 if x.dim() == 1 else x.shape[1])
    call("fmoe_sort_rows", order._index, x.data_ptr(), row_bytes, order._ref, output.data_ptr(),
         int(not given))
    return written(output) if given else output


def _unsort(rows: torch.Tensor, order: ExpertOrder, weights: Optional[torch.Tensor],
            output: Optional[torch.Tensor]) -> torch.Tensor:
    given = output is not None
    if not given:
        output = rows.new_empty(_rows_shape(rows, order.num_tokens))
    call("fmoe_unsort_rows", order._index, rows.data_ptr(), DTYPE_TAG[rows.dtype],
         1 if rows.dim() == 1 else rows.shape[1], order._ref, ptr(weights), output.data_ptr())
    return written(output) if given else output


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order = order
        return _sort(x, order, None)

    @staticmethod
    def backward(ctx, grad_rows):
        first_order_only()
        return _unsort(grad_rows.contiguous(), ctx.order, None, None), None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        ctx.order = order
        ctx.weighted = weights is not None
        # the rows are needed again only for the weights' gradient
        keep = rows if ctx.weighted and ctx.needs_input_grad[1] else None
        ctx.save_for_backward(keep, weights)
        return _unsort(rows, order, weights, None)

    @staticmethod
    def backward(ctx, grad_y):
        first_order_only()
        rows, weights = ctx.saved_tensors
        order = ctx.order
        grad_y = grad_y.contiguous()
        grad_rows = grad_weights = None
        if ctx.needs_input_grad[0]:
            grad_rows = grad_y.new_empty(_rows_shape(grad_y, order.num_rows))
        if ctx.weighted and ctx.needs_input_grad[1]:
            grad_weights = torch.empty_like(weights)
        call("fmoe_unsort_rows_backward", order._index, grad_y.data_ptr(), ptr(rows),
             DTYPE_TAG[grad_y.dtype], 1 if grad_y.dim() == 1 else grad_y.shape[1], order._ref,
             ptr(weights), ptr(grad_rows), ptr(grad_weights))
        return grad_rows, grad_weights, None


def _check(t, name: str, order, n: int) -> None:
    not_traced()
    if not isinstance(order, ExpertOrder):
        raise TypeError("order must be an ExpertOrder (sort_by_expert)")
    need(t, name, order._index, None, None)
    if t.dim() not in (1, 2) or t.shape[0] != n or (t.dim() == 2 and t.shape[1] < 1):
        raise ValueError(f"{name} must have shape [{n}] or [{n}, H], got {tuple(t.shape)}")


def sort_tokens(x: torch.Tensor, order: ExpertOrder, *,
                output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Token rows ``x`` [T, H] (or one value per token, [T]) in expert order: [num_rows, H].

    Any element type (int8 and e4m3 rows and fp32 scales among them). Padding rows inside an
    expert's range are zero. Rows from ``order.expert_base[E]`` on are zero in a new tensor and
    left as they were in a given ``output``. Differentiable for bf16, fp16 and fp32 ``x`` (without
    ``output``): a token's gradient is the sum of its rows' gradients in fp32, rounded once.
    """
    _check(x, "x", order, order.num_tokens if isinstance(order, ExpertOrder) else 0)
    if output is not None:
        need(output, "output", order._index, _rows_shape(x, order.num_rows), (x.dtype,))
        if output.is_conj():
            raise ValueError("output must not be a conjugate view")
    if x.is_conj():  # its bytes are those before the conjugation
        x = x.resolve_conj()
    if recording(x, output):
        if output is not None:
            raise ValueError("output cannot be given where gradients are recorded")
        if x.dtype not in DTYPE_TAG:
            raise TypeError(f"no gradient for {x.dtype} rows")
        return _SortTokens.apply(x, order)
    return _sort(x, order, output)


def unsort_tokens(rows: torch.Tensor, order: ExpertOrder,
                  topk_weights: Optional[torch.Tensor] = None, *,
                  output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Expert rows back per token: ``y[t] = sum_k topk_weights[t, k] * rows[pick_row[t, k]]``.

    ``rows`` [num_rows, H] (or [num_rows]) bf16, fp16 or fp32, ``topk_weights`` fp32 [T, top_k] or
    None for ones. Sums in fp32 in pick order, rounded once; picks without a row add nothing,
    whatever their weight, and rows without a pick are not read. Differentiable in ``rows`` and
    ``topk_weights`` (without ``output``); rows without a pick get a zero gradient.
    """
    _check(rows, "rows", order, order.num_rows if isinstance(order, ExpertOrder) else 0)
    if rows.dtype not in DTYPE_TAG:
        raise TypeError(f"rows must be bfloat16, float16 or float32, got {rows.dtype}")
    if topk_weights is not None:
        need(topk_weights, "topk_weights", order._index, (order.num_tokens, order.top_k), F32)
    if output is not None:
        need(output, "output", order._index, _rows_shape(rows, order.num_tokens), (rows.dtype,))
    if recording(rows, topk_weights, output):
        if output is not None:
            raise ValueError("output cannot be given where gradients are recorded")
        return _UnsortTokens.apply(rows, topk_weights, order)
    return _unsort(rows, order, topk_weights, output)

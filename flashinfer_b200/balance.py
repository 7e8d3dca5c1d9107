"""The balance loss of a router with its gradient, and the picks per expert.

Training a router needs a term that keeps its experts evenly used: ``balance_loss`` compares how often
each expert is picked with how much of the score it gets, over a batch or per sequence. The counts that
it needs come back with it, and ``expert_counts`` gives them alone (for instance to step a routing bias).
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FmoeBalanceArgs
from ._op import (DTYPE_TAG, FLOATS, I32, INT_MAX, call, first, first_order_only, need, ptr,
                  recording)

_SCORING = {"softmax": _lib.SCORING_SOFTMAX, "sigmoid": _lib.SCORING_SIGMOID}
MAX_EXPERTS = 1024
MAX_SEQUENCES = 4096


@lru_cache(maxsize=1024)
def _workspace_bytes(T: int, E: int, S: int) -> int:
    size = ctypes.c_size_t()
    _lib.check(_lib.load().fmoe_balance_workspace_size(T, E, S, ctypes.byref(size)),
               "fmoe_balance_workspace_size")
    return size.value


def _sequences(base: Optional[torch.Tensor], index: int) -> int:
    if base is None:
        return 1
    need(base, "sequence_base", index, None, I32)
    if base.dim() != 1 or not 2 <= base.shape[0] <= MAX_SEQUENCES + 1:
        raise ValueError(f"sequence_base must hold the bases of 1..{MAX_SEQUENCES} sequences and their "
                         f"end, got shape {tuple(base.shape)}")
    return base.shape[0] - 1


def _forward(logits, topk_ids, E, S, scoring, base):
    T, K = topk_ids.shape
    if T * K > INT_MAX:
        raise ValueError(f"topk_ids holds {T * K} picks: counts are int32")
    a = FmoeBalanceArgs(T, E, K, S, 0 if logits is None else DTYPE_TAG[logits.dtype], scoring,
                        ptr(logits), topk_ids.data_ptr(), ptr(base))
    counts = topk_ids.new_empty((E,) if base is None else (S, E))
    a.counts = counts.data_ptr()
    loss = factor = None
    if logits is not None:
        loss = logits.new_empty((), dtype=torch.float32)
        factor = logits.new_empty(S, dtype=torch.float32)
        a.loss, a.factor = loss.data_ptr(), factor.data_ptr()
    size = _workspace_bytes(T, E, S)
    workspace = topk_ids.new_empty(size // 4)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    call("fmoe_balance_loss", topk_ids.get_device(), ctypes.byref(a))
    return loss, counts, factor


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk_ids, S, scoring, base):
        loss, counts, factor = _forward(logits, topk_ids, logits.shape[1], S, scoring, base)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, counts, factor, base)
        ctx.rest = (topk_ids.shape[1], S, scoring)
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _):
        first_order_only()
        if grad_loss is None:
            return None, None, None, None, None
        logits, counts, factor, base = ctx.saved_tensors
        K, S, scoring = ctx.rest
        T, E = logits.shape
        grad = torch.empty_like(logits)
        a = FmoeBalanceArgs(T, E, K, S, DTYPE_TAG[logits.dtype], scoring, logits.data_ptr(), None,
                            ptr(base), None, counts.data_ptr(), factor.data_ptr(),
                            grad_loss.data_ptr(), grad.data_ptr())
        call("fmoe_balance_loss_backward", logits.get_device(), ctypes.byref(a))
        return grad, None, None, None, None


def balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, *, scoring: str = "softmax",
                 sequence_base: Optional[torch.Tensor] = None,
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The router's balance loss (an fp32 scalar) and the int32 picks per expert.

    ``logits`` [T, E] bf16, fp16 or fp32 (E up to 1024), ``topk_ids`` int32 [T, top_k], the experts that
    each token was sent to (ids outside [0, E), -1 among them, are no picks). The scores ``p[t]`` are the
    softmax of row t, or with ``scoring="sigmoid"`` its sigmoids divided by their sum. Over the T tokens

        loss = sum_e f[e] * mean_t p[t, e],   f[e] = E / (top_k * T) * counts[e]

    which is 1 where picks or scores are even. With ``sequence_base`` (int32 [S + 1], S up to 4096, read on
    the device: sequence s has the rows sequence_base[s] .. sequence_base[s + 1], a base smaller than an
    earlier one counts as that one) the loss is that of each sequence, averaged over those that have
    tokens, and ``counts`` is [S, E] instead of [E]; rows in no sequence (padding) count for nothing. A row
    of which every logit is -infinity has no scores. Without any token the loss is 0.

    Differentiable in ``logits`` (the counts are constants): rows of no sequence get a zero gradient.
    Scores, sums and the loss are fp32 or more; sums run in a fixed order.
    """
    index = first(logits, "logits", FLOATS, 2)
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"logits must have 1..{MAX_EXPERTS} experts, got {E}")
    need(topk_ids, "topk_ids", index, None, I32)
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_ids.shape[1] < 1:
        raise ValueError(f"topk_ids must have shape [{T}, top_k], got {tuple(topk_ids.shape)}")
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    S = _sequences(sequence_base, index)
    if recording(logits):
        return _BalanceLoss.apply(logits, topk_ids, S, _SCORING[scoring], sequence_base)
    return _forward(logits, topk_ids, E, S, _SCORING[scoring], sequence_base)[:2]


def expert_counts(topk_ids: torch.Tensor, num_experts: int, *,
                  sequence_base: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The picks of every expert in int32 ``topk_ids`` [T, top_k]: int32 [num_experts] (up to 1024), or
    [S, num_experts] with ``sequence_base`` as in ``balance_loss``. Other ids (-1 = no pick) count for
    nothing."""
    index = first(topk_ids, "topk_ids", I32, 2)
    if topk_ids.shape[1] < 1:
        raise ValueError("topk_ids needs at least one pick per token")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be 1..{MAX_EXPERTS}, got {num_experts}")
    S = _sequences(sequence_base, index)
    return _forward(None, topk_ids, num_experts, S, 0, sequence_base)[1]

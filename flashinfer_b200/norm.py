"""The RMS norms before and after a block, fused with the block's gate and the residual scale.

One call sits between two blocks of a model: it normalises what the block returned, gates it, adds
it to the scaled residual stream and normalises the sum for the next block; for an FP8 expert layer
the result leaves as ``run``'s e4m3 input with its scales. Forward and backward are one pass each.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import FmoeBlockNormArgs
from ._op import DTYPE_TAG, FLOATS, call, first, first_order_only, need, ptr, recording, written

BLOCK = 128


_PARAMS = {t: (t, torch.float32) for t in FLOATS}
_ONE = {t: (t,) for t in FLOATS}


def _tag(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else DTYPE_TAG[t.dtype]


def _args(branch, residual, post_weight, gate, pre_weight, kind, residual_scale, eps):
    T, H = residual.shape
    return FmoeBlockNormArgs(T, H, DTYPE_TAG[residual.dtype], ptr(branch), residual.data_ptr(),
                             ptr(post_weight), ptr(gate), ptr(pre_weight), _tag(post_weight),
                             _tag(gate), _tag(pre_weight), kind, residual_scale, eps)


def _forward(branch, residual, post_weight, gate, pre_weight, kind, residual_scale, eps, quantize,
             hidden, want_stats):
    a = _args(branch, residual, post_weight, gate, pre_weight, kind, residual_scale, eps)
    T, H = residual.shape
    given = hidden is not None
    if given:
        a.hidden = hidden.data_ptr()
    elif branch is None and residual_scale == 1.0 and not want_stats:
        hidden = residual  # without a block output and with scale 1 it is what it was
    else:
        hidden = torch.empty_like(residual)
        a.hidden = hidden.data_ptr()
    normed = stats = None
    if quantize:
        q = residual.new_empty((T, H), dtype=torch.float8_e4m3fn)
        scale = residual.new_empty((H // BLOCK, T), dtype=torch.float32)
        a.normed_q, a.normed_scale = q.data_ptr(), scale.data_ptr()
        normed = (q, scale)
    elif pre_weight is not None:
        normed = torch.empty_like(residual)
        a.normed = normed.data_ptr()
    if want_stats:
        stats = residual.new_empty((T, 2), dtype=torch.float32)
        a.stats = stats.data_ptr()
    call("fmoe_block_norm", residual.get_device(), ctypes.byref(a))
    if given:
        written(hidden)
    return hidden, normed, stats


@lru_cache(maxsize=1024)
def _workspace_bytes(T: int, H: int) -> int:
    size = ctypes.c_size_t()
    _lib.check(_lib.load().fmoe_block_norm_workspace_size(T, H, ctypes.byref(size)),
               "fmoe_block_norm_workspace_size")
    return size.value


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, post_weight, gate, pre_weight, kind, residual_scale, eps):
        hidden, normed, stats = _forward(branch, residual, post_weight, gate, pre_weight, kind,
                                         residual_scale, eps, False, None, True)
        ctx.save_for_backward(branch, residual, post_weight, gate, pre_weight, stats)
        ctx.rest = (kind, residual_scale, eps)
        ctx.set_materialize_grads(False)
        return hidden, normed

    @staticmethod
    def backward(ctx, grad_hidden, grad_normed):
        first_order_only()
        branch, residual, post_weight, gate, pre_weight, stats = ctx.saved_tensors
        a = _args(branch, residual, post_weight, gate, pre_weight, *ctx.rest)
        if grad_hidden is not None:
            grad_hidden = grad_hidden.contiguous()
            a.grad_hidden = grad_hidden.data_ptr()
        if grad_normed is not None:
            grad_normed = grad_normed.contiguous()
            a.grad_normed = grad_normed.data_ptr()
        a.stats = stats.data_ptr()
        need_f, need_x, need_wp, need_g, need_wq = ctx.needs_input_grad[:5]
        d_f = d_x = d_wp = d_g = d_wq = workspace = None
        if need_f:
            d_f = torch.empty_like(branch)
            a.grad_branch = d_f.data_ptr()
        if need_x:
            d_x = torch.empty_like(residual)
            a.grad_residual = d_x.data_ptr()
        if need_wp:
            d_wp = torch.empty_like(post_weight)
            a.grad_post_weight = d_wp.data_ptr()
        if need_g:
            d_g = torch.empty_like(gate)
            a.grad_gate = d_g.data_ptr()
        if need_wq:
            d_wq = torch.empty_like(pre_weight)
            a.grad_pre_weight = d_wq.data_ptr()
        if need_wp or need_g or need_wq:
            size = _workspace_bytes(*residual.shape)
            workspace = stats.new_empty(size // 4)
            a.workspace, a.workspace_bytes = ptr(workspace), size
        call("fmoe_block_norm_backward", residual.get_device(), ctypes.byref(a))
        return d_f, d_x, d_wp, d_g, d_wq, None, None, None


def block_norm(branch: Optional[torch.Tensor], residual: torch.Tensor, *,
               post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
               residual_scale: float = 1.0, pre_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6, quantize: bool = False,
               output: Optional[torch.Tensor] = None,
               ) -> Tuple[torch.Tensor, Union[None, torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]]:
    """``hidden = residual_scale * residual + gate * norm(branch) * post_weight`` and
    ``normed = norm(hidden) * pre_weight``, with ``norm(v) = v / sqrt(mean(v^2) + eps)`` per token.

    branch, residual [T, H] of one type (bf16, fp16, fp32), H up to 16384; branch None where no
    block came before (``hidden`` is then the scaled residual; with scale 1 and no gradient
    recorded it is ``residual`` itself). post_weight [H]: None for no norm
    after the block. gate: one factor per token [T, 1], per channel [H] or per element [T, H], or
    None. pre_weight [H]: None for no norm before the next block (``normed`` is then None). Weights
    and gate are of the activations' type or fp32. hidden stays in fp32 between the two norms.

    Returns ``(hidden, normed)``. With ``quantize`` (H a multiple of 128, 16-byte aligned tensors)
    normed is the pair ``(e4m3 [T, H], fp32 scales [H/128, T])`` that ``run`` takes as
    ``hidden_states`` and ``hidden_states_scale``; that form has no gradient. ``output`` receives
    hidden and may be ``residual`` itself (no gradient either). Otherwise differentiable in every
    tensor; weight gradients are summed over tokens in a fixed order.
    """
    index = first(residual, "residual", FLOATS, 2)
    T, H = shape = residual.shape
    if not 1 <= H <= 16384:
        raise ValueError(f"the hidden size must be 1..16384, got {H}")
    same, params = _ONE[residual.dtype], _PARAMS[residual.dtype]
    if branch is not None:
        need(branch, "branch", index, shape, same)
    elif post_weight is not None or gate is not None:
        raise ValueError("post_weight and gate need a branch")
    if post_weight is not None:
        need(post_weight, "post_weight", index, (H,), params)
    if pre_weight is not None:
        need(pre_weight, "pre_weight", index, (H,), params)
    kind = _lib.GATE_NONE
    if gate is not None:
        need(gate, "gate", index, None, params)
        if gate.shape == (H,):
            kind = _lib.GATE_CHANNEL
        elif gate.shape == (T, 1):
            kind = _lib.GATE_TOKEN
        elif gate.shape == shape:
            kind = _lib.GATE_FULL
        else:
            raise ValueError(f"gate must have shape {(T, 1)}, {(H,)} or {(T, H)}, "
                             f"got {tuple(gate.shape)}")
    if quantize:
        if pre_weight is None:
            raise ValueError("quantize needs a pre_weight")
        if H % BLOCK:
            raise ValueError(f"quantize needs a hidden size that is a multiple of {BLOCK}, got {H}")
    if output is not None:
        need(output, "output", index, shape, same)
    residual_scale, eps = float(residual_scale), float(eps)
    if recording(branch, residual, post_weight, gate, pre_weight, output):
        if quantize:
            raise ValueError("the quantised form has no gradient: call it under torch.no_grad()")
        if output is not None:
            raise ValueError("output cannot be given where gradients are recorded")
        return _BlockNorm.apply(branch, residual, post_weight, gate, pre_weight, kind,
                                residual_scale, eps)
    hidden, normed, _ = _forward(branch, residual, post_weight, gate, pre_weight, kind,
                                 residual_scale, eps, quantize, output, False)
    return hidden, normed

"""Products of 16-bit activations with weights of 4 bits.

``quantize_int4`` puts weights (of one matrix, or of all experts) into 4-bit values with a scale, and on
request a zero point, per group along the depth; ``int4_matmul`` multiplies activations with one such
matrix and ``int4_expert_matmul`` with one matrix per expert, over rows in the expert order of
``sort_by_expert``. The activations stay in 16 bits: a decode step reads a quarter of the weights' bytes
and needs no calibration. None of them has a gradient: a call that autograd would record (a tensor that
requires a gradient, outside ``torch.no_grad()``) is refused.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FmoeInt4Args
from ._op import (DTYPE_TAG, F32, FLOATS, I32, INT_MAX, call, first, need, no_gradient, ptr, recording,
                  written)

_HALVES = (torch.bfloat16, torch.float16)
_SCALES = {t: (t, torch.float32) for t in _HALVES}
_U8 = (torch.uint8,)


def _groups(K: int, group: int) -> int:
    """The groups of a row of depth K; checks both."""
    if K < 32 or K % 32 or K > 131072:
        raise ValueError(f"the depth K must be a multiple of 32 from 32 to 131072, got {K}")
    if group not in (32, 64) and (group < 128 or group % 128 or group > INT_MAX - 131072):
        raise ValueError(f"group must be 32, 64 or a multiple of 128, got {group}")
    return -(-K // group)


def quantize_int4(w: torch.Tensor, *, group: int = 128, symmetric: bool = True,
                  ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Weights [N, K] or [E, N, K] (bf16, fp16, fp32; K a multiple of 32) in 4 bits.

    Returns ``(packed, scale, zero)``: packed uint8 [..., K / 2] with value 2i in the low half of byte i,
    scale [..., groups] of the weights' type, groups = ceil(K / group), and zero uint8 [..., groups], or
    None with ``symmetric``. A value q stands for ``scale * (q - zero)``, with zero 8 where it is None.
    ``group`` is 32, 64 or a multiple of 128 (one of K or more: a scale per row); the last may be shorter.

    symmetric: ``scale = max|w| / 7``, ``q = round(w / scale) + 8``. Else, with low = min(w, 0) and
    high = max(w, 0): ``scale = (high - low) / 15``, ``zero = round(-low / scale)``,
    ``q = round(w / scale) + zero``. The scale is rounded to its type before the division by it (and is at
    least 2^-100, fp16: 2^-24), ties round to even, q stays within 1..15 and 0..15. A group with a NaN or an
    infinity has a NaN or infinite scale.
    """
    index = first(w, "w", FLOATS, 3 if isinstance(w, torch.Tensor) and w.dim() == 3 else 2)
    K = w.shape[-1]
    n = _groups(K, group)
    if recording(w):
        no_gradient("quantize_int4")
    rows = w.shape[:-1]
    packed = w.new_empty((*rows, K // 2), dtype=torch.uint8)
    scale = w.new_empty((*rows, n))
    zero = None if symmetric else w.new_empty((*rows, n), dtype=torch.uint8)
    call("fmoe_quantize_int4", index, w.data_ptr(), DTYPE_TAG[w.dtype], w.numel() // K, K, group,
         packed.data_ptr(), scale.data_ptr(), ptr(zero))
    return packed, scale, zero


def dequantize_int4(packed: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None, *,
                    group: int = 128, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The weights that 4-bit values stand for: ``scale * (q - zero)`` in fp32, rounded to ``out_dtype``.

    packed uint8 [..., K / 2] of two or three axes, scale [..., groups] bf16, fp16 or fp32, zero uint8
    [..., groups] (the low four bits count) or None for 8.
    """
    index = first(packed, "packed", _U8, 3 if isinstance(packed, torch.Tensor) and packed.dim() == 3 else 2)
    K = packed.shape[-1] * 2
    shape = (*packed.shape[:-1], _groups(K, group))
    need(scale, "scale", index, shape, FLOATS)
    if zero is not None:
        need(zero, "zero", index, shape, _U8)
    if out_dtype not in DTYPE_TAG:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if recording(scale):
        no_gradient("dequantize_int4")
    w = packed.new_empty((*packed.shape[:-1], K), dtype=out_dtype)
    call("fmoe_dequantize_int4", index, packed.data_ptr(), scale.data_ptr(), DTYPE_TAG[scale.dtype],
         ptr(zero), w.numel() // K, K, group, w.data_ptr(), DTYPE_TAG[out_dtype])
    return w


@lru_cache(maxsize=1024)
def _workspace_bytes(M: int, N: int, K: int, E: int) -> int:
    size = ctypes.c_size_t()
    _lib.check(_lib.load().fmoe_int4_workspace_size(M, N, K, E, ctypes.byref(size)),
               "fmoe_int4_workspace_size")
    return size.value


def _product(what, x, weight, scale, zero, bias, base, group, output, index, E, N):
    M, K = x.shape
    n = _groups(K, group)
    if E * N > INT_MAX - 1024:
        raise ValueError(f"fewer than 2^31 - 1024 output channels are possible, got {E * N}")
    shape = (N, n) if base is None else (E, N, n)
    need(scale, "scale", index, shape, _SCALES[x.dtype])
    if zero is not None:
        need(zero, "zero", index, shape, _U8)
    if recording(x, scale, bias, output):
        no_gradient(what)
    given = output is not None
    if given:
        need(output, "output", index, (M, N), (x.dtype,))
    else:
        output = x.new_empty((M, N))
    a = FmoeInt4Args(M, N, K, E, group, DTYPE_TAG[x.dtype], DTYPE_TAG[scale.dtype], x.data_ptr(),
                     weight.data_ptr(), scale.data_ptr(), ptr(zero), ptr(bias), ptr(base),
                     output.data_ptr(), 0 if given else 1)
    size = _workspace_bytes(M, N, K, E)
    if size:
        workspace = x.new_empty(size, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    call("fmoe_int4_matmul", index, ctypes.byref(a))
    return written(output) if given else output


def int4_matmul(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor,
                zero: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                group: int = 128, output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[m, n] = sum_k x[m, k] * w[n, k] (+ bias[n])`` with ``w = scale * (q - zero)`` in 4 bits.

    x [M, K] bf16 or fp16 (K a multiple of 32), weight uint8 [N, K / 2] with scale [N, groups] (x's type or
    fp32) and zero uint8 [N, groups] or None, as ``quantize_int4`` returns them for this ``group``; bias
    fp32 [N]. Sums in fp32. The result is [M, N] of x's type, or is written to ``output``. x and weight
    start on 16-byte boundaries.

    Up to 16 rows multiply the exact 4-bit values and scale each group's sum in fp32. More rows go over the tensor
    cores, where each ``w`` is rounded to x's type first: off by half a step of that type, or in fp16 by 2^-29 of
    the largest scale of its row where that is more (scales of one row that are 2^18 and more apart).
    """
    index = first(x, "x", _HALVES, 2)
    need(weight, "weight", index, None, _U8)
    if weight.dim() != 2 or weight.shape[1] * 2 != x.shape[1] or weight.shape[0] < 1:
        raise ValueError(f"x [M, K] and weight [N, K / 2] do not fit: {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}")
    N = weight.shape[0]
    if bias is not None:
        need(bias, "bias", index, (N,), F32)
    return _product("int4_matmul", x, weight, scale, zero, bias, None, group, output, index, 1, N)


def int4_expert_matmul(rows: torch.Tensor, weights: torch.Tensor, scale: torch.Tensor,
                       expert_base: torch.Tensor, zero: Optional[torch.Tensor] = None, *,
                       group: int = 128, output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One 4-bit product per expert: rows expert_base[e] .. expert_base[e+1] times ``weights[e]``.

    rows [R, K] bf16 or fp16 in expert order, weights uint8 [E, N, K / 2] (E up to 256) with scale
    [E, N, groups] (the rows' type or fp32) and zero uint8 [E, N, groups] or None, expert_base int32 [E+1]
    (``ExpertOrder.expert_base``), read on the device: a base smaller than an earlier one counts as that
    one, so a row has one expert at most. Returns [R, N] of the rows' type; rows before ``expert_base[0]``
    and from ``expert_base[E]`` on are zero in a new tensor and left as they were in a given ``output``. Weights
    are exact where R is up to 8 E, however many of the rows each expert has, and rounded as in ``int4_matmul``
    from there on.
    """
    index = first(rows, "rows", _HALVES, 2)
    need(weights, "weights", index, None, _U8)
    if weights.dim() != 3 or weights.shape[2] * 2 != rows.shape[1] or weights.shape[1] < 1:
        raise ValueError(f"rows [R, K] and weights [E, N, K / 2] do not fit: {tuple(rows.shape)}, "
                         f"{tuple(weights.shape)}")
    E, N, _ = weights.shape
    if not 1 <= E <= 256:
        raise ValueError(f"weights must hold 1..256 experts, got {E}")
    need(expert_base, "expert_base", index, (E + 1,), I32)
    return _product("int4_expert_matmul", rows, weights, scale, zero, None, expert_base, group, output,
                    index, E, N)


def int4_status(device: Optional[torch.device] = None) -> int:
    """``_lib.STATUS_TIMEOUT_INT4`` if a wait inside a 4-bit product on the device ran out since the last
    call (its output is not valid), else 0. Synchronises the current stream: products on other streams are
    covered as far as they had finished, and by the next call otherwise."""
    index = None if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    status = ctypes.c_int32(0)
    call("fmoe_int4_status", index, ctypes.byref(status))
    return status.value

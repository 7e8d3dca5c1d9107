"""Products in 8-bit integers with one scale per token and one per output channel.

``quantize_int8`` turns activations (or, once, weights) into int8 rows and their scales;
``int8_matmul`` multiplies them with one weight matrix and ``int8_expert_matmul`` with one matrix
per expert, over rows in the expert order of ``sort_by_expert``. Sums are exact in int32. None of them
has a gradient: a call that autograd would record (a tensor that requires a gradient, outside
``torch.no_grad()``) is refused.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._op import (DTYPE_TAG, F32, FLOATS, I32, I8, INT_MAX, call, first, need, no_gradient, ptr,
                  recording, written)

_HALVES = (torch.bfloat16, torch.float16)


def quantize_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 or fp16 rows [R, K] -> (int8 [R, K], fp32 scales [R]), symmetric per row.

    ``amax = max(max|x|, 1e-30)``, ``scale = amax / 127`` and the values are ``127 x / amax`` rounded
    to the nearest integer (ties to even), so ``q * scale`` is off by at most half a step of
    ``amax / 127``. A row with a NaN or an infinity gets a NaN or infinite scale: its products are
    NaN. Weights [N, K] are quantised per output channel by the same call.
    """
    index = first(x, "x", _HALVES, 2)
    R, K = x.shape
    if K < 1:
        raise ValueError("x needs at least one column")
    if recording(x):
        no_gradient("quantize_int8")
    q = x.new_empty((R, K), dtype=torch.int8)
    scale = x.new_empty(R, dtype=torch.float32)
    call("fmoe_quantize_int8", index, x.data_ptr(), DTYPE_TAG[x.dtype], R, K, q.data_ptr(),
         scale.data_ptr())
    return q, scale


def _check_sizes(channels: int, K: int) -> None:
    if channels > INT_MAX:
        raise ValueError(f"at most 2^31 - 1 output channels are possible, got {channels}")
    if K < 16 or K % 16 or K > 131056:
        raise ValueError(f"the depth K must be a multiple of 16 from 16 to 131056, got {K}")


def _output(output, out_dtype, a, index, shape):
    if output is None:
        if out_dtype not in DTYPE_TAG:
            raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        return a.new_empty(shape, dtype=out_dtype)
    need(output, "output", index, shape, FLOATS)
    return output


def int8_matmul(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, out_dtype: torch.dtype = torch.bfloat16,
                output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[m, n] = a_scale[m] * b_scale[n] * sum_k a[m, k] * b[n, k] (+ bias[n])``.

    a int8 [M, K] (tokens), b int8 [N, K] (weights), scales fp32 [M] and [N], bias fp32 [N]; K a
    multiple of 16. The result is [M, N] of ``out_dtype`` (bf16, fp16 or fp32), or is written to
    ``output`` in that tensor's type.
    """
    index = first(a, "a", I8, 2)
    need(b, "b", index, None, I8)
    if b.dim() != 2 or a.shape[1] != b.shape[1] or b.shape[0] < 1:
        raise ValueError(f"a [M, K] and b [N, K] do not fit: {tuple(a.shape)}, {tuple(b.shape)}")
    M, K = a.shape
    N = b.shape[0]
    _check_sizes(N, K)
    need(a_scale, "a_scale", index, (M,), F32)
    need(b_scale, "b_scale", index, (N,), F32)
    if bias is not None:
        need(bias, "bias", index, (N,), F32)
    if recording(a_scale, b_scale, bias, output):
        no_gradient("int8_matmul")
    given = output is not None
    output = _output(output, out_dtype, a, index, (M, N))
    call("fmoe_int8_matmul", index, a.data_ptr(), b.data_ptr(), a_scale.data_ptr(),
         b_scale.data_ptr(), ptr(bias), M, N, K, output.data_ptr(), DTYPE_TAG[output.dtype])
    return written(output) if given else output


def int8_expert_matmul(rows: torch.Tensor, weights: torch.Tensor, row_scale: torch.Tensor,
                       weight_scale: torch.Tensor, expert_base: torch.Tensor, *,
                       out_dtype: torch.dtype = torch.bfloat16,
                       output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One int8 product per expert: rows expert_base[e] .. expert_base[e+1] times ``weights[e]``.

    rows int8 [R, K] in expert order, weights int8 [E, N, K] (E up to 256), row_scale fp32 [R],
    weight_scale fp32 [E, N], expert_base int32 [E+1] (``ExpertOrder.expert_base``), read on the
    device: a base smaller than an earlier one counts as that one, so a row has one expert at most.
    Returns [R, N]; rows before ``expert_base[0]`` and from ``expert_base[E]`` on are zero
    in a new tensor and left as they were in a given ``output``.
    """
    index = first(rows, "rows", I8, 2)
    need(weights, "weights", index, None, I8)
    if weights.dim() != 3 or rows.shape[1] != weights.shape[2] or weights.shape[1] < 1:
        raise ValueError(f"rows [R, K] and weights [E, N, K] do not fit: {tuple(rows.shape)}, "
                         f"{tuple(weights.shape)}")
    R, K = rows.shape
    E, N, _ = weights.shape
    if not 1 <= E <= 256:
        raise ValueError(f"weights must hold 1..256 experts, got {E}")
    _check_sizes(N, K)
    need(row_scale, "row_scale", index, (R,), F32)
    need(weight_scale, "weight_scale", index, (E, N), F32)
    need(expert_base, "expert_base", index, (E + 1,), I32)
    if recording(row_scale, weight_scale, output):
        no_gradient("int8_expert_matmul")
    given = output is not None
    output = _output(output, out_dtype, rows, index, (R, N))
    call("fmoe_int8_expert_matmul", index, rows.data_ptr(), weights.data_ptr(),
         row_scale.data_ptr(), weight_scale.data_ptr(), expert_base.data_ptr(), R, E, N, K,
         output.data_ptr(), DTYPE_TAG[output.dtype], int(not given))
    return written(output) if given else output


def int8_status(device: Optional[torch.device] = None) -> int:
    """``_lib.STATUS_TIMEOUT_INT8`` if a wait inside an int8 product on the device ran out since the
    last call (its output is not valid), else 0. Synchronises the current stream: products on other
    streams are covered as far as they had finished, and by the next call otherwise."""
    index = None if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    status = ctypes.c_int32(0)
    call("fmoe_int8_status", index, ctypes.byref(status))
    return status.value

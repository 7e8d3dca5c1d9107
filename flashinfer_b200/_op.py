"""What the operators around the experts share: tensor checks and the call into the library."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

DTYPE_TAG = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
             torch.float16: _lib.DTYPE_F16}


def need(t, name: str, device: Optional[torch.device], shape=None, dtypes=None) -> None:
    """A contiguous CUDA tensor (on ``device`` if given) of one of ``dtypes`` and of ``shape``."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def call(name: str, device: torch.device, *args) -> None:
    """One library call on ``device`` and its current stream; raises on an error code."""
    fn = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        _lib.check(rc, name)


def recording(*tensors) -> bool:
    """Whether autograd records a call on these tensors (None among them allowed)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)

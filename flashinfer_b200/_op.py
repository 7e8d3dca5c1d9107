"""What the operators around the experts share: tensor checks and the call into the library.

The calls of one decode step take a few microseconds on the device, so the checks test everything
in one expression per tensor and look for the reason only when it fails.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream
from torch._C import _is_tracing
from torch._C import _len_torch_dispatch_stack as _dispatch_modes
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.graph import increment_version as _increment_version

from . import _lib

DTYPE_TAG = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
             torch.float16: _lib.DTYPE_F16}
I8 = (torch.int8,)
I32 = (torch.int32,)
F32 = (torch.float32,)
FLOATS = tuple(DTYPE_TAG)
INT_MAX = 2 ** 31 - 1  # what is passed as a C int; ctypes drops the bits above without a word


_FUNCTIONS = {}  # the library's entry points by name


def _refuse(t, name: str, index: Optional[int], shape, dtypes) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    raise ValueError(f"{name} must be contiguous")


def first(t, name: str, dtypes, dim: int) -> int:
    """The device index of a call's first tensor: CUDA, contiguous, ``dim`` axes, of ``dtypes``."""
    if _is_tracing() or _dispatch_modes():
        not_traced()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != dim:
        raise ValueError(f"{name} must be a tensor of {dim} axes, got shape {tuple(t.shape)}")
    if not (t.is_cuda and t.dtype in dtypes and t.is_contiguous()):
        _refuse(t, name, None, None, dtypes)
    return t.get_device()


def need(t, name: str, index: int, shape, dtypes) -> None:
    """A contiguous tensor on CUDA device ``index``, of ``shape`` and one of ``dtypes`` (None: any)."""
    if not (isinstance(t, torch.Tensor) and t.get_device() == index
            and (shape is None or t.shape == shape) and (dtypes is None or t.dtype in dtypes)
            and t.is_contiguous()):
        _refuse(t, name, index, shape, dtypes)


def not_traced() -> None:
    """Refuses ``torch.jit.trace`` and ``make_fx``: what they record would hold the outputs' allocation
    and not the call that writes them."""
    if _is_tracing() or (_dispatch_modes() and _fx_tracing()):
        raise RuntimeError("this operator cannot be traced (torch.jit.trace, make_fx)")


def _fx_tracing() -> bool:
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def written(output: torch.Tensor) -> torch.Tensor:
    """A given output after the call: autograd learns that its values changed, so that a backward pass
    which saved them raises instead of using the new ones."""
    _increment_version(output)
    return output


def ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def call(name: str, index: int, *args) -> None:
    """One library call on CUDA device ``index`` and its current stream; raises on an error code."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_lib.load(), name)
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def first_order_only() -> None:
    """Called in a backward pass: refuses to be recorded itself (``create_graph=True``), since the
    library's gradients have no gradient of their own."""
    if torch.is_grad_enabled():
        raise RuntimeError("this operator has no second derivative (create_graph=True)")


def no_gradient(what: str) -> None:
    """Refuses a call that autograd would have to record: its result would be cut off."""
    raise ValueError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def recording(*tensors) -> bool:
    """Whether autograd records a call on these tensors (None among them allowed). Refuses dual
    tensors: the library would drop their tangents, which need neither ``requires_grad`` nor grad
    mode."""
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("this operator has no forward-mode derivative")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False

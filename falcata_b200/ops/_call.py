"""Argument checks and native calls shared by the operators that run on the caller's stream."""
from __future__ import annotations

import ctypes
from typing import Callable, Optional, Tuple

import torch
from torch.autograd import forward_ad

from ..basic import _lib

_TYPE_CODE = {torch.float32: 0, torch.float16: 6, torch.bfloat16: 16}
_BOUND: dict = {}


def bind(name: str, argtypes: tuple):
    """The native entry point with its argument types set (once)."""
    fn = _BOUND.get(name)
    if fn is None:
        fn = getattr(_lib(), name)
        fn.argtypes = argtypes; fn.restype = ctypes.c_int
        _BOUND[name] = fn
    return fn


def check(ret: int) -> None:
    if ret != 0:
        lib = _lib()
        lib.FB_OpsLastError.restype = ctypes.c_char_p
        raise RuntimeError(lib.FB_OpsLastError().decode())


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def type_code(name: str, t: torch.Tensor) -> int:
    code = _TYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: float32, float16 or bfloat16 is wanted, got {t.dtype}")
    return code


def require_tensor(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is wanted, got {type(t).__name__}")


def one_device(**tensors: Optional[torch.Tensor]) -> None:
    """All of them on one CUDA device (that of the first)."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        where = t.device
        if where != device:
            if where.type != "cuda":
                raise ValueError(f"{name}: a CUDA tensor is wanted, got one on {where}")
            if device is not None:
                raise ValueError(f"{name}: on {where}, the other tensors are on {device}")
            device = where


def no_tangents(operator: str, *tensors: Optional[torch.Tensor]) -> None:
    """Forward-mode derivatives are refused, not dropped."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # outside forward-mode differentiation: nothing to look for
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{operator}: forward-mode derivatives are not available")


class _NoDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, operator, compute, *tensors):
        ctx.operator = operator
        return compute()

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.operator}: its result has no derivative; detach it or the inputs")


def without_derivative(operator: str, compute: Callable[[], torch.Tensor], *tensors: Optional[torch.Tensor]) -> torch.Tensor:
    """``compute()``; where a gradient is wanted in one of the tensors, a backward pass through the result raises."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _NoDerivative.apply(operator, compute, *tensors)
    return compute()


# The stream's handle without the Python object around it, where torch offers that (1 us less per call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def device_and_stream(device: torch.device) -> Tuple[int, int]:
    index = device.index
    return index, _raw_stream(index)

"""Matrix products of rows grouped by leaf: one linear map per leaf, leaves of any number of rows.

``leaf_begin`` [leaves + 1] (int32 / int64, on the device, non-decreasing) gives leaf g the rows [leaf_begin[g], leaf_begin[g + 1]): the
rows lie leaf by leaf. For the leaf numbers that ``Booster.predict(..., pred_leaf=True)`` gives in row order,
``order = torch.argsort(leaf, stable=True)`` groups the rows, and ``torch.searchsorted(leaf[order], torch.arange(leaves + 1))``, of
one type and on the device, gives their boundaries. Sums are fp32, rounded once to the output's type.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._call import bind, check, device_and_stream, no_tangents, one_device, ptr, require_tensor, type_code, without_derivative

__all__ = ["leaf_gram", "leaf_products"]


MAX_COLUMNS = MAX_LEAVES = 1 << 28      # the native call counts them, and a row's bytes, in 32 bits


def _begin(leaf_begin: torch.Tensor) -> None:
    require_tensor("leaf_begin", leaf_begin)
    if leaf_begin.dtype not in (torch.int32, torch.int64) or leaf_begin.dim() != 1 or leaf_begin.numel() < 2:
        raise ValueError(f"leaf_begin: int32 or int64 of [leaves + 1], at least one leaf, is wanted, got {leaf_begin.dtype} {tuple(leaf_begin.shape)}")
    if leaf_begin.numel() - 1 > MAX_LEAVES:
        raise ValueError(f"leaf_begin: at most {MAX_LEAVES} leaves are covered, got {leaf_begin.numel() - 1}")


def _rows(name: str, t: torch.Tensor) -> None:
    require_tensor(name, t)
    type_code(name, t)
    if t.dim() != 2 or t.shape[1] < 1:
        raise ValueError(f"{name}: [rows, columns] with at least one column is wanted, got shape {tuple(t.shape)}")
    if t.shape[1] > MAX_COLUMNS:
        raise ValueError(f"{name}: at most {MAX_COLUMNS} columns are covered, got {t.shape[1]}")


def _inner_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _products(x: torch.Tensor, weight: torch.Tensor, leaf_begin: torch.Tensor) -> torch.Tensor:
    x, leaf_begin = _inner_contiguous(x), leaf_begin.contiguous()
    if weight.stride(2) != 1 and weight.stride(1) != 1:
        weight = weight.contiguous()
    n, f = x.shape
    leaves, outputs = weight.shape[0], weight.shape[1]
    y = x.new_empty((n, outputs))
    if n:
        _run(_fwd(), (ptr(x), x.stride(0), ptr(weight), weight.stride(0), weight.stride(1), weight.stride(2), ptr(leaf_begin), 8 * leaf_begin.element_size(), leaves, n, f, outputs,
                      type_code("x", x), ptr(y)), x.device)
    return y


def _run(entry, args: tuple, device: torch.device) -> None:
    """The native call with the workspace that it asks for; the workspace belongs to the current stream, as every tensor made here."""
    floats = ctypes.c_longlong(0)      # in: no workspace yet; out: the floats that are wanted, 0 when the call has run
    where = device_and_stream(device)
    check(entry(*args, None, ctypes.byref(floats), *where))
    if floats.value:
        workspace = torch.empty(floats.value, dtype=torch.float32, device=device)
        check(entry(*args, workspace.data_ptr(), None, *where))


class _LeafProducts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, leaf_begin):
        ctx.save_for_backward(x, weight, leaf_begin)
        return _products(x, weight, leaf_begin)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, leaf_begin = ctx.saved_tensors
        grad_x = leaf_products(grad, weight.transpose(1, 2), leaf_begin) if ctx.needs_input_grad[0] else None
        grad_weight = leaf_gram(grad, x, leaf_begin) if ctx.needs_input_grad[1] else None
        return grad_x, grad_weight, None


def leaf_products(x: torch.Tensor, weight: torch.Tensor, leaf_begin: torch.Tensor) -> torch.Tensor:
    """``y[i] = weight[leaf of row i] @ x[i]``: [rows, outputs] from ``x`` [rows, features] and ``weight`` [leaves, outputs, features].

    float32 / float16 / bfloat16, one type. ``weight`` may have any strides (a transposed view gives the gradient in ``x``). Rows
    before the first and behind the last leaf get zeros. Boundaries outside the rows are clamped to them; where boundaries fall
    again, a row that several leaves claim belongs to the first of them. Differentiable in ``x`` and ``weight`` (once); runs on
    the current stream.
    """
    _rows("x", x)
    require_tensor("weight", weight)
    if weight.dtype != x.dtype:
        raise TypeError(f"weight: the type of x ({x.dtype}) is wanted, got {weight.dtype}")
    _begin(leaf_begin)
    if weight.dim() != 3 or weight.shape[0] != leaf_begin.numel() - 1 or weight.shape[1] < 1 or weight.shape[2] != x.shape[1]:
        raise ValueError(f"weight: [{leaf_begin.numel() - 1} leaves, outputs, {x.shape[1]} features] is wanted, got shape {tuple(weight.shape)}")
    if weight.shape[1] > MAX_COLUMNS:
        raise ValueError(f"weight: at most {MAX_COLUMNS} outputs are covered, got {weight.shape[1]}")
    no_tangents("leaf_products", x, weight)
    one_device(x=x, weight=weight, leaf_begin=leaf_begin)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _LeafProducts.apply(x, weight, leaf_begin)
    return _products(x, weight, leaf_begin)


def leaf_gram(a: torch.Tensor, b: torch.Tensor, leaf_begin: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``out[g] = sum over the rows i of leaf g of a[i] b[i]^T``: [leaves, columns of a, columns of b], leaves without rows zero.

    With the gradient of ``leaf_products`` for ``a`` and its ``x`` for ``b`` this is the gradient in the weights; with ``h * x`` and
    ``x`` the normal equations of linear leaves. ``dtype``: the inputs' type (default) or float32. Boundaries are clamped to the
    rows; where they fall again, the sums of the leaves concerned are unspecified. Not differentiable (a backward
    pass through the result raises); runs on the current stream, the same sums on every run.
    """
    _rows("a", a); _rows("b", b)
    if a.dtype != b.dtype:
        raise TypeError(f"b: the type of a ({a.dtype}) is wanted, got {b.dtype}")
    if a.shape[0] != b.shape[0]:
        raise ValueError(f"b: {a.shape[0]} rows are wanted, got {b.shape[0]}")
    dtype = dtype or a.dtype
    if dtype not in (a.dtype, torch.float32):
        raise TypeError(f"dtype: {a.dtype} or float32 is wanted, got {dtype}")
    _begin(leaf_begin)
    no_tangents("leaf_gram", a, b)
    one_device(a=a, b=b, leaf_begin=leaf_begin)
    return without_derivative("leaf_gram", lambda: _sums(a, b, leaf_begin, dtype), a, b)


def _sums(a: torch.Tensor, b: torch.Tensor, leaf_begin: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    a, b, leaf_begin = _inner_contiguous(a), _inner_contiguous(b), leaf_begin.contiguous()
    leaves = leaf_begin.numel() - 1
    out = a.new_empty((leaves, a.shape[1], b.shape[1]), dtype=dtype)
    _run(_gram(), (ptr(a), a.stride(0), ptr(b), b.stride(0), ptr(leaf_begin), 8 * leaf_begin.element_size(), leaves, a.shape[0], a.shape[1], b.shape[1], type_code("a", a),
                   type_code("dtype", out), ptr(out)), a.device)
    return out


_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


def _fwd():
    return bind("FB_OpLeafProducts", (_P, _L, _P, _L, _L, _L, _P, _I, _I, _L, _I, _I, _I, _P, _P, ctypes.POINTER(_L), _I, _P))


def _gram():
    return bind("FB_OpLeafGram", (_P, _L, _P, _L, _P, _I, _I, _L, _I, _I, _I, _I, _P, _P, ctypes.POINTER(_L), _I, _P))

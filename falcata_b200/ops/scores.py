"""Log probabilities of class scores on the device, and their gradient.

For scores ``s`` of shape [rows, classes] (what ``Booster.predict(..., raw_score=True)`` returns, or the class-major training
scores that a custom objective sees), per row:

    log_norm = log sum_j exp(s_j)          log p_j = s_j - log_norm          entropy = -sum_j p_j log p_j

and the alternatives: the classes of the largest scores, equal scores by rising class. Statistics are fp32 whatever the type of
the scores. A class of score -inf is ruled out: probability 0, never an alternative. A row whose classes are all ruled out has
log_norm and log probabilities -inf, entropy 0, no alternatives (class -1, log probability -inf) and gradient 0. A row with a NaN
or +inf gives NaN, no alternatives, and NaN gradients.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from ._call import bind, check, device_and_stream, no_tangents, one_device, ptr, require_tensor, type_code, without_derivative

MAX_TOP_CLASSES = 32

__all__ = ["ClassLogProbs", "class_log_probs", "class_log_probs_grad"]


class ClassLogProbs(NamedTuple):
    """Per row: log probability of the label (None without labels), log of the normaliser, entropy, and the alternatives
    [rows, top_k] (None for ``top_k=0``)."""

    log_prob: Optional[torch.Tensor]
    log_norm: torch.Tensor
    entropy: torch.Tensor
    top_log_prob: Optional[torch.Tensor]
    top_class: Optional[torch.Tensor]


def _labels(labels: Optional[torch.Tensor], scores: torch.Tensor) -> Optional[torch.Tensor]:
    if labels is None:
        return None
    require_tensor("labels", labels)
    if labels.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"labels: int32 or int64 class numbers are wanted, got {labels.dtype}")
    if labels.shape != (scores.shape[0],):
        raise ValueError(f"labels: one per row is wanted ({scores.shape[0]}), got shape {tuple(labels.shape)}")
    return labels


def _scores(scores: torch.Tensor) -> None:
    require_tensor("scores", scores)
    type_code("scores", scores)
    if scores.dim() != 2 or scores.shape[1] < 1:
        raise ValueError(f"scores: [rows, classes] with at least one class is wanted, got shape {tuple(scores.shape)}")


def _row_values(name: str, t: Optional[torch.Tensor], shape) -> Optional[torch.Tensor]:
    if t is None:
        return None
    require_tensor(name, t)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(shape)} is wanted, got {tuple(t.shape)}")
    return t


def _forward(scores: torch.Tensor, labels: Optional[torch.Tensor], top_k: int) -> ClassLogProbs:
    n, k = scores.shape
    labels = None if labels is None else labels.contiguous()
    new = scores.new_empty
    log_prob = None if labels is None else new(n, dtype=torch.float32)
    log_norm, entropy = new(n, dtype=torch.float32), new(n, dtype=torch.float32)
    top_log_prob, top_class = (new((n, top_k), dtype=torch.float32), new((n, top_k), dtype=torch.int32)) if top_k else (None, None)
    if n:
        row_stride, class_stride = scores.stride()
        check(_fwd()(scores.data_ptr(), type_code("scores", scores), n, k, row_stride, class_stride, ptr(labels), 0 if labels is None else 8 * labels.element_size(), top_k,
                     ptr(log_prob), log_norm.data_ptr(), entropy.data_ptr(), ptr(top_log_prob), ptr(top_class), *device_and_stream(scores.device)))
    return ClassLogProbs(log_prob, log_norm, entropy, top_log_prob, top_class)


class _ClassLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, labels, top_k):
        out = _forward(scores, labels, top_k)
        ctx.save_for_backward(scores, labels, out.log_norm, out.entropy, out.top_class)
        ctx.set_materialize_grads(False)
        if out.top_class is not None:
            ctx.mark_non_differentiable(out.top_class)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_log_prob, g_log_norm, g_entropy, g_top, _):
        scores, labels, log_norm, entropy, top_class = ctx.saved_tensors
        if all(g is None for g in (g_log_prob, g_log_norm, g_entropy, g_top)):
            return None, None, None
        return class_log_probs_grad(scores, log_norm, entropy, labels=labels, top_class=top_class, grad_log_prob=g_log_prob, grad_log_norm=g_log_norm,
                                    grad_entropy=g_entropy, grad_top_log_prob=g_top), None, None


def class_log_probs(scores: torch.Tensor, labels: Optional[torch.Tensor] = None, top_k: int = 0) -> ClassLogProbs:
    """Log probability of each row's label, log of the normaliser, entropy and the ``top_k`` best classes of class scores.

    ``scores``: CUDA tensor [rows, classes], float32 / float16 / bfloat16, any strides (rows contiguous, or class-major as the
    training scores are). ``labels``: int32 / int64 [rows]; a negative one means "no label" (log probability 0, no gradient), one
    past the last class gives NaN. ``top_k``: 0 to 32, at most the number of classes. Differentiable in ``scores`` (once); the
    call runs on the current stream and does not wait.
    """
    _scores(scores)
    labels = _labels(labels, scores)
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP_CLASSES, scores.shape[1]):
        raise ValueError(f"top_k: 0 to {min(MAX_TOP_CLASSES, scores.shape[1])} alternatives of {scores.shape[1]} classes, got {top_k}")
    no_tangents("class_log_probs", scores)
    one_device(scores=scores, labels=labels)
    if scores.requires_grad and torch.is_grad_enabled():
        return ClassLogProbs(*_ClassLogProbs.apply(scores, labels, top_k))
    return _forward(scores, labels, top_k)


def class_log_probs_grad(scores: torch.Tensor, log_norm: torch.Tensor, entropy: torch.Tensor, labels: Optional[torch.Tensor] = None, top_class: Optional[torch.Tensor] = None,
                         grad_log_prob: Optional[torch.Tensor] = None, grad_log_norm: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                         grad_top_log_prob: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient in ``scores`` of a loss whose gradients in the results of ``class_log_probs`` are given (None: zero).

    ``log_norm``, ``entropy``, ``top_class``: those results. The gradient has the type of the scores and their order in memory
    (class-major scores give a class-major gradient, whose transpose is what ``Booster.update`` takes from a custom objective).
    It has no derivative itself: a backward pass through it raises.
    """
    _scores(scores)
    labels = _labels(labels, scores)
    n, k = scores.shape
    log_norm, entropy = _row_values("log_norm", log_norm, (n,)), _row_values("entropy", entropy, (n,))
    if log_norm is None or entropy is None:
        raise ValueError("log_norm and entropy: the results of class_log_probs are wanted")
    if grad_log_prob is not None and labels is None:
        raise ValueError("grad_log_prob needs the labels")
    if (top_class is None) != (grad_top_log_prob is None) and grad_top_log_prob is not None:
        raise ValueError("grad_top_log_prob needs top_class")
    top_k = 0
    if grad_top_log_prob is not None:
        require_tensor("top_class", top_class)
        if top_class.dtype != torch.int32 or top_class.dim() != 2 or top_class.shape[0] != n or top_class.shape[1] > min(MAX_TOP_CLASSES, k):
            raise ValueError(f"top_class: int32 [{n}, at most {min(MAX_TOP_CLASSES, k)}] is wanted, got {top_class.dtype} {tuple(top_class.shape)}")
        top_k = top_class.shape[1]
        grad_top_log_prob = _row_values("grad_top_log_prob", grad_top_log_prob, (n, top_k))
    else:
        top_class = None
    grads = [_row_values(name, t, (n,)) for name, t in (("grad_log_prob", grad_log_prob), ("grad_log_norm", grad_log_norm), ("grad_entropy", grad_entropy))]
    inputs = (scores, log_norm, entropy, *grads, grad_top_log_prob)
    no_tangents("class_log_probs_grad", *inputs)
    one_device(scores=scores, labels=labels, log_norm=log_norm, entropy=entropy, top_class=top_class, grad_log_prob=grads[0], grad_log_norm=grads[1], grad_entropy=grads[2],
               grad_top_log_prob=grad_top_log_prob)
    return without_derivative("class_log_probs_grad", lambda: _gradient(scores, labels, top_k, top_class, log_norm, entropy, grad_top_log_prob, *grads), *inputs)


def _gradient(scores: torch.Tensor, labels: Optional[torch.Tensor], top_k: int, top_class: Optional[torch.Tensor], *values: Optional[torch.Tensor]) -> torch.Tensor:
    n, k = scores.shape
    log_norm, entropy, grad_top_log_prob, *grads = (None if t is None else (t if t.dtype is torch.float32 else t.float()).contiguous() for t in values)
    labels, top_class = (None if t is None else t.contiguous() for t in (labels, top_class))
    by_class = scores.stride(0) < scores.stride(1)
    out = scores.new_empty((k, n)).t() if by_class else scores.new_empty((n, k))
    if n:
        check(_bwd()(ptr(scores), type_code("scores", scores), n, k, scores.stride(0), scores.stride(1), ptr(labels), 0 if labels is None else 8 * labels.element_size(), top_k,
                     ptr(log_norm), ptr(entropy), ptr(top_class), *map(ptr, grads), ptr(grad_top_log_prob), ptr(out), out.stride(0), out.stride(1), *device_and_stream(scores.device)))
    return out


_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


def _fwd():
    return bind("FB_OpClassLogProbs", (_P, _I, _L, _L, _L, _L, _P, _I, _I, _P, _P, _P, _P, _P, _I, _P))


def _bwd():
    return bind("FB_OpClassLogProbsGrad", (_P, _I, _L, _L, _L, _L, _P, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P, _L, _L, _I, _P))

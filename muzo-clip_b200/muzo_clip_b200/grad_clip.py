"""The norm over all gradients of a model, and clipping by it.

``clip_grad_norm_`` is torch's function of that name for CUDA gradients: two launches for a whole
model, whatever the number of tensors (up to 1150 per launch), no host synchronisation, equal bits
for equal gradients. ``clip_grads`` writes the scaled gradients elsewhere instead, in their own type
or as fp32; ``grad_norm`` is the norm alone. Tensors of fp32, bf16 and fp16 mix freely, on one
device. None of the three is differentiable (as torch's clip_grad_norm_ is not). The native
module checks the tensors (ValueError, TypeError) and makes the calls.
"""

from __future__ import annotations

import math
from collections.abc import Iterable

import torch

from . import _lib

_native = _lib.native
_flat = _native.flat   # (tensor) -> whether its elements fill its memory, in whatever order


def _tensors(tensors) -> list[torch.Tensor]:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return tensors if isinstance(tensors, list) else list(tensors)


def _is_inf(norm_type) -> bool:
    norm_type = float(norm_type)
    if norm_type == 2.0:
        return False
    if norm_type == math.inf:
        return True
    raise ValueError(f"gradient norms of type 2 and inf are supported, not {norm_type}")


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


def grad_norm(grads: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, for ``norm_type=inf``, the largest magnitude) over all elements of all
    ``grads``, as a 0-dim fp32 tensor on their device. Squares are summed beyond fp32's range and
    precision. No tensors: 0."""
    return _native.grad_norm(_tensors(grads), _is_inf(norm_type))


def clip_grads(grads: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Iterable[torch.Tensor] | None = None) -> tuple[list[torch.Tensor], torch.Tensor]:
    """``grads`` times min(1, max_norm / (norm + 1e-6)), written to ``out`` (new tensors of the
    gradients' types by default), and their norm before. An ``out`` tensor has its gradient's shape,
    and its type or fp32 (the gradients an fp32 optimizer state takes); it may be the gradient
    itself, and otherwise must not share memory with any tensor of the call."""
    grads = _tensors(grads)
    out = [torch.empty_like(t) for t in grads] if out is None else _tensors(out)
    return out, _native.clip_grads(grads, None if out is grads else out, _max_norm(max_norm), _is_inf(norm_type))


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ on the library's kernels: scales the gradients of
    ``parameters`` in place so that their norm is at most ``max_norm`` and returns the norm before.
    The gradients are on one device and the norm is the 2-norm or the maximum; ``foreach``, torch's
    choice between its own implementations, changes nothing here.
    A non-finite norm scales as in torch (inf: finite gradients become 0; NaN: all become NaN), or
    raises with ``error_if_nonfinite``, which forms the norm first, waits for it and leaves the
    gradients alone."""
    grads = [p.grad for p in _tensors(parameters) if p.grad is not None]
    if error_if_nonfinite:
        _max_norm(max_norm)
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it "
                               "cannot be clipped. To disable this error and scale the gradients by the non-finite norm "
                               "anyway, set `error_if_nonfinite=False`")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]

"""The norm over all gradients of a model, and clipping by it.

``clip_grad_norm_`` is torch's function of that name for CUDA gradients: two launches for a whole
model, whatever the number of tensors (up to 1150 per launch), no host synchronisation, equal bits
for equal gradients. ``clip_grads`` writes the scaled gradients elsewhere instead, in their own type
or as fp32; ``grad_norm`` is the norm alone. Tensors of fp32, bf16 and fp16 mix freely.
"""

from __future__ import annotations

import math
from array import array
from collections.abc import Iterable

import torch

from . import _lib

_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _tensors(tensors) -> list[torch.Tensor]:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return tensors if isinstance(tensors, list) else list(tensors)


def _inf_norm(norm_type) -> int:
    norm_type = float(norm_type)
    if norm_type == math.inf:
        return 1
    if norm_type == 2.0:
        return 0
    raise ValueError(f"gradient norms of type 2 and inf are supported, not {norm_type}")


def _flat(t: torch.Tensor) -> bool:
    """Whether t's elements fill its memory from data_ptr() on, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda x: x[1]):
        if size == 1:
            continue
        if stride != expected:
            return False
        expected *= size
    return True


def _check(tensors: list[torch.Tensor], what: str) -> torch.device | None:
    device = None
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {type(t).__name__}")
        if t.layout is not torch.strided:
            raise ValueError(f"{what}: sparse gradients are not supported")
        if t.dtype not in _CODES:
            raise TypeError(f"{what} supports float32, bfloat16 and float16, not {t.dtype}")
        if device is None:
            device = t.device
            if device.type != "cuda":
                raise ValueError("muzo_clip_b200 gradient kernels run on CUDA tensors only")
        elif t.device != device:
            raise ValueError(f"{what}: the tensors are on different devices")
    return device


def _column(values, kind: str):
    a = array(kind, values)
    return a, a.buffer_info()[0]


def _workspace(sizes, device):
    size = _lib.lib.muzo_grad_workspace(len(sizes), sum(sizes))
    return torch.empty(size, dtype=torch.uint8, device=device), size


def grad_norm(grads: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, for ``norm_type=inf``, the largest magnitude) over all elements of all
    ``grads``, as a 0-dim fp32 tensor on their device. Squares are summed beyond fp32's range and
    precision. No tensors: 0."""
    inf = _inf_norm(norm_type)
    grads = _tensors(grads)
    device = _check(grads, "grad_norm")
    if device is None:
        return torch.tensor(0.0)
    with torch.no_grad():
        grads = [t if _flat(t) else t.contiguous() for t in grads]
        sizes = [t.numel() for t in grads]
        src, src_p = _column([t.data_ptr() for t in grads], "Q")
        num, num_p = _column(sizes, "q")
        kinds, kinds_p = _column([_CODES[t.dtype] for t in grads], "i")
        norm = torch.empty((), dtype=torch.float32, device=device)
        with _lib.on_device(device):
            work, size = _workspace(sizes, device)
            _lib.launch("muzo_grad_norm", src_p, num_p, kinds_p, len(grads), inf, norm.data_ptr(), work.data_ptr(), size,
                        _lib.stream_ptr(device))
    return norm


def _clip(grads, outs, max_norm: float, inf: int, device) -> torch.Tensor:
    sizes = [t.numel() for t in grads]
    src, src_p = _column([t.data_ptr() for t in grads], "Q")
    dst, dst_p = _column([t.data_ptr() for t in outs], "Q") if outs is not grads else (src, src_p)
    num, num_p = _column(sizes, "q")
    kinds, kinds_p = _column([_CODES[t.dtype] for t in grads], "i")
    to, to_p = _column([_CODES[t.dtype] for t in outs], "i") if outs is not grads else (kinds, kinds_p)
    norm = torch.empty((), dtype=torch.float32, device=device)
    with _lib.on_device(device):
        work, size = _workspace(sizes, device)
        status = _lib.lib.muzo_grad_clip(src_p, dst_p, num_p, kinds_p, to_p, len(grads), inf, max_norm, norm.data_ptr(),
                                         work.data_ptr(), size, _lib.stream_ptr(device))
        if status == _lib.ERR_ARG:
            raise ValueError("gradient clipping: tensors that are written overlap in memory (the same one twice?)")
        _lib.check(status, "muzo_grad_clip")
        _lib.launch_count += _lib.KERNELS_PER_CALL["muzo_grad_clip"]
    return norm


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


def clip_grads(grads: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Iterable[torch.Tensor] | None = None) -> tuple[list[torch.Tensor], torch.Tensor]:
    """``grads`` times min(1, max_norm / (norm + 1e-6)), written to ``out`` (new tensors of the
    gradients' types by default), and their norm before. An ``out`` tensor has its gradient's shape
    and strides, and its type or fp32 (the gradients an fp32 optimizer state takes); it may be the
    gradient itself, and otherwise must not share memory with any tensor of the call."""
    inf, max_norm = _inf_norm(norm_type), _max_norm(max_norm)
    grads = _tensors(grads)
    device = _check(grads, "clip_grads")
    with torch.no_grad():
        if out is None:
            out = [torch.empty_like(t) for t in grads]
        else:
            out = _tensors(out)
            if len(out) != len(grads):
                raise ValueError(f"clip_grads: {len(grads)} gradients but {len(out)} outputs")
            _check(out, "clip_grads")
        if device is None:
            return out, torch.tensor(0.0)
        for g, o in zip(grads, out):
            if o.device != device or o.shape != g.shape or (o.dtype != g.dtype and o.dtype != torch.float32):
                raise ValueError("clip_grads: an output must have its gradient's shape and device, and its type or fp32")
        # what does not fill its memory, or lies in another order than its output, takes a detour
        plain = [(g.stride() == o.stride() or g.numel() <= 1) and _flat(g) for g, o in zip(grads, out)]
        if all(plain):
            norm = _clip(grads, out, max_norm, inf, device)
        else:
            src = [g if p else g.contiguous() for g, p in zip(grads, plain)]
            dst = [o if p else torch.empty(o.shape, dtype=o.dtype, device=device) for o, p in zip(out, plain)]
            norm = _clip(src, dst, max_norm, inf, device)
            for o, d, p in zip(out, dst, plain):
                if not p:
                    o.copy_(d)
        torch.autograd.graph.increment_version([o for o in out if not o.is_inference()])
    return out, norm


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ on the library's kernels: scales the gradients of
    ``parameters`` in place so that their norm is at most ``max_norm`` and returns the norm before.
    A non-finite norm scales as in torch (inf: finite gradients become 0; NaN: all become NaN), or
    raises with ``error_if_nonfinite``, which waits for the norm and leaves the gradients alone."""
    parameters = _tensors(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite:
        _max_norm(max_norm)
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it "
                               "cannot be clipped. To disable this error and scale the gradients by the non-finite norm "
                               "anyway, set `error_if_nonfinite=False`")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]

"""Tensor-core attention that records the per-head maxima QK-Clip needs, and its backward pass.

``attention_max`` is differentiable: with gradients enabled it keeps each row's log-sum-exp, and
the backward pass recomputes the probabilities from it (``attention_max_backward``, also callable
on its own). Both run on the current stream of the tensors' device, allocate their outputs and
workspace from torch's allocator and give equal bits for equal calls.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

# ---------------------------------------------------------------- status words

_ATTN_STATUS: dict[int, torch.Tensor] = {}


def attention_status(device: torch.device) -> torch.Tensor:
    """Two device int32 words per GPU: [0] the first nonzero timeout code of an attention launch,
    [1] the stall request (0; tests set a role's code to make its first wait expire)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    t = _ATTN_STATUS.get(idx)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            # the words outlive any graph: they are cleared now, on a stream that is not captured
            side = torch.cuda.Stream(device=idx)
            with torch.cuda.stream(side):
                t = torch.zeros(2, dtype=torch.int32, device=torch.device("cuda", idx))
        else:
            t = torch.zeros(2, dtype=torch.int32, device=torch.device("cuda", idx))
            torch.cuda.current_stream(idx).synchronize()   # cleared before another stream's launch reads them
        _ATTN_STATUS[idx] = t
    return t


def check_attention_status(device: torch.device) -> None:
    """Raise if an attention launch on `device` reported an expired wait (reads one word)."""
    if device.type != "cuda" or not _ATTN_STATUS:
        return
    idx = device.index if device.index is not None else torch.cuda.current_device()
    t = _ATTN_STATUS.get(idx)
    if t is not None and int(t[0].item()) != 0:
        code = int(t[0].item())
        t[0].zero_()
        raise _lib.MuzoError(f"fused attention reported status {code} (a bounded wait expired); the outputs of "
                             "the forward that ran it are unspecified")


# ---------------------------------------------------------------- arguments


def _check(query, key, value, scaling, key_lo, key_hi) -> float:
    """Refuse what the kernels do not compute; returns the scaling."""
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not isinstance(t, torch.Tensor) or t.ndim != 4:
            raise ValueError(f"attention_max expects a 4-D {name} [B, H, S, D]")
    dev = query.device
    if dev.type != "cuda":
        raise ValueError("muzo_clip_b200 attention kernels run on CUDA tensors only")
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"attention_max supports bfloat16 and float16, not {query.dtype}")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError("attention_max: query, key and value differ in type")
    if key.device != dev or value.device != dev:
        raise ValueError("attention_max: query, key and value are on different devices")
    b, hq, _, d = query.shape
    if key.shape != value.shape or key.shape[0] != b or key.shape[3] != d:
        raise ValueError(f"attention_max: key {tuple(key.shape)} and value {tuple(value.shape)} do not fit "
                         f"query {tuple(query.shape)}")
    if hq == 0 or key.shape[1] == 0 or hq % key.shape[1] != 0:
        raise ValueError(f"attention_max: {hq} query heads are not a multiple of {key.shape[1]} key heads")
    if d % 8 != 0 or not 8 <= d <= 128:
        raise ValueError(f"attention_max supports head dimensions that are multiples of 8 up to 128, not {d}")
    for name, t in (("key_lo", key_lo), ("key_hi", key_hi)):
        if t is not None and (t.dtype != torch.int32 or t.device != dev or t.shape != (b,) or not t.is_contiguous()):
            raise ValueError(f"attention_max: {name} must be a contiguous int32 tensor of {b} values on {dev}")
    scaling = d ** -0.5 if scaling is None else float(scaling)
    if not (scaling > 0.0 and math.isfinite(scaling)):
        raise ValueError(f"attention_max: the scaling must be positive and finite, not {scaling}")
    return scaling


def _readable(t: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """``t`` [.., .., .., D], copied where the kernels' 16-byte tile loads could not read it in
    place (D strided, unaligned, or expanded along a dimension), and the strides of its leading
    dimensions (a dimension of size 1 is never stepped over: its stride is any valid one)."""
    for _ in range(2):
        strides = tuple(int(s) if n > 1 else int(t.shape[-1]) for s, n in zip(t.stride()[:3], t.shape[:3]))
        if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 or s == 0 for s in strides):
            return t, strides
        t = t.clone(memory_format=torch.contiguous_format)
    return t, strides


def _ptr(t: torch.Tensor | None):
    return t.data_ptr() if t is not None and t.numel() else None


# ---------------------------------------------------------------- forward


def _forward(query, key, value, scaling, causal, key_lo, key_hi, record, keep_lse):
    b, hq, sq, d = (int(v) for v in query.shape)
    hkv, sk = int(key.shape[1]), int(key.shape[2])
    dev = query.device
    out = torch.empty((b, sq, hq, d), dtype=query.dtype, device=dev)
    lse = torch.empty((b, hq, sq), dtype=torch.float32, device=dev) if keep_lse else None
    smax = valid = None
    if out.numel() == 0:
        if record:
            smax = torch.full((hq,), float("-inf"), dtype=torch.float32, device=dev)
            valid = torch.ones(1, dtype=torch.int32, device=dev)
        return out, lse, smax, valid
    if record:
        smax = torch.empty(hq, dtype=torch.float32, device=dev)
        valid = torch.empty(1, dtype=torch.int32, device=dev)
    query, qs = _readable(query)
    key, ks = _readable(key)
    value, vs = _readable(value)
    with _lib.on_device(dev):
        _lib.launch("muzo_attention_max_lse", query.data_ptr(), _ptr(key), _ptr(value), out.data_ptr(), _ptr(lse),
                    _lib.dtype_code(query.dtype), b, hq, hkv, sq, sk, d, *qs, *ks, *vs, sq * hq * d, d, hq * d,
                    1 if causal else 0, scaling, _ptr(key_lo), _ptr(key_hi), _ptr(smax), _ptr(valid),
                    attention_status(dev).data_ptr(), _lib.stream_ptr(dev))
    return out, lse, smax, valid


class _AttentionMax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, scaling, causal, key_lo, key_hi, record):
        out, lse, smax, valid = _forward(query, key, value, scaling, causal, key_lo, key_hi, record, True)
        ctx.save_for_backward(query, key, value, out, lse, key_lo, key_hi)
        ctx.scaling, ctx.causal = scaling, causal
        if record:
            ctx.mark_non_differentiable(smax, valid)
        return out, smax, valid

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, _smax, _valid):
        query, key, value, out, lse, key_lo, key_hi = ctx.saved_tensors
        grads = _backward(grad_out, query, key, value, out, lse, ctx.scaling, ctx.causal, key_lo, key_hi,
                          ctx.needs_input_grad[:3])
        return (*grads, None, None, None, None, None)


def attention_max(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: float | None = None,
                  causal: bool = True, key_lo: torch.Tensor | None = None, key_hi: torch.Tensor | None = None,
                  record: bool = True) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """softmax(scaling * Q K^T) V on the tensor cores for Q [B, Hq, Sq, D], K, V [B, Hkv, Sk, D]
    (transformers' transposed views; bf16 or fp16, D a multiple of 8 up to 128), returned as
    [B, Sq, Hq, D] (the layout attention functions return); with ``record``, also the per-head max
    of the eager pre-softmax logits and a validity word, on the device.

    ``causal``: query i sees the keys j <= i + Sk - Sq. ``key_lo`` / ``key_hi`` (int32 per batch)
    bound the visible keys to [key_lo, key_hi); what lies outside is not read into any result, not
    even when it is not finite. A query that sees no key gets zeros. ``scaling`` defaults to
    D ** -0.5.

    Differentiable once in query, key and value (the maxima are not): the products of the backward
    pass take the probabilities and their gradients in the inputs' type, as the forward does, and
    sum in fp32."""
    scaling = _check(query, key, value, scaling, key_lo, key_hi)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        return _AttentionMax.apply(query, key, value, scaling, bool(causal), key_lo, key_hi, bool(record))
    out, _, smax, valid = _forward(query, key, value, scaling, causal, key_lo, key_hi, record, False)
    return out, smax, valid


# ---------------------------------------------------------------- backward


def _backward(grad_out, query, key, value, out, lse, scaling, causal, key_lo, key_hi, wanted):
    b, hq, sq, d = (int(v) for v in query.shape)
    hkv, sk = int(key.shape[1]), int(key.shape[2])
    dev = query.device

    def grad(s, h, want):   # [B, H, S, D] over the projections' [B, S, H, D] memory
        return torch.empty((b, s, h, d), dtype=query.dtype, device=dev).transpose(1, 2) if want else None

    dq, dk, dv = grad(sq, hq, wanted[0]), grad(sk, hkv, wanted[1]), grad(sk, hkv, wanted[2])
    made = [t for t in (dq, dk, dv) if t is not None]
    if query.numel() == 0 or key.numel() == 0:   # no pair of a query and a key
        for t in made:
            t.zero_()
        return dq, dk, dv
    if not made:
        return dq, dk, dv
    query, qs = _readable(query)
    key, ks = _readable(key)
    value, vs = _readable(value)
    out, os_ = _readable(out)
    grad_out, gs = _readable(grad_out)
    strides = (*qs, *ks, *vs, os_[0], os_[2], os_[1], gs[0], gs[2], gs[1],
               sq * hq * d, d, hq * d, sk * hkv * d, d, hkv * d, sk * hkv * d, d, hkv * d)
    code = _lib.dtype_code(query.dtype)
    with _lib.on_device(dev):
        size = _lib.lib.muzo_attention_backward_workspace(code, b, hq, hkv, sq, sk, d)
        workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
        _lib.launch("muzo_attention_backward", query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(),
                    grad_out.data_ptr(), lse.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), code, b, hq, hkv, sq, sk, d,
                    (ctypes.c_int64 * 24)(*strides), 1 if causal else 0, scaling, _ptr(key_lo), _ptr(key_hi),
                    workspace.data_ptr(), size, attention_status(dev).data_ptr(), _lib.stream_ptr(dev))
    return dq, dk, dv


def attention_max_backward(grad_out: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                           out: torch.Tensor, lse: torch.Tensor, scaling: float | None = None, causal: bool = True,
                           key_lo: torch.Tensor | None = None, key_hi: torch.Tensor | None = None,
                           ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients (dQ, dK, dV) of ``attention_max`` for callers that run their own autograd:
    ``out`` and ``grad_out`` are [B, Sq, Hq, D], ``lse`` [B, Hq, Sq] fp32 is the natural logarithm
    of each row's sum of exp(scaled logit) over the keys it sees (-inf where it sees none). The
    other arguments are the forward's. The gradients have the shapes of query, key and value (dK and
    dV summed over the query heads of each key head)."""
    scaling = _check(query, key, value, scaling, key_lo, key_hi)
    b, hq, sq, d = query.shape
    for name, t in (("out", out), ("grad_out", grad_out)):
        if t.shape != (b, sq, hq, d) or t.dtype != query.dtype or t.device != query.device:
            raise ValueError(f"attention_max_backward: {name} must be [B, Sq, Hq, D] = {(b, sq, hq, d)} of the query's "
                             "type and device")
    if lse.shape != (b, hq, sq) or lse.dtype != torch.float32 or lse.device != query.device:
        raise ValueError(f"attention_max_backward: lse must be fp32 [B, Hq, Sq] = {(b, hq, sq)} on {query.device}")
    with torch.no_grad():
        return _backward(grad_out, query, key, value, out, lse.contiguous(), scaling, causal, key_lo, key_hi,
                         (True, True, True))

"""Tensor-core attention that records the per-head maxima QK-Clip needs, and its backward pass.

``attention_max`` is differentiable: with gradients enabled it keeps each row's log-sum-exp, and
the backward pass recomputes the probabilities from it (``attention_max_backward``, also callable
on its own). Both run on the current stream of the tensors' device, allocate their outputs and
workspace from torch's allocator and give equal bits for equal calls. The native module checks the
arguments (ValueError, TypeError) and makes the calls.
"""

from __future__ import annotations

import torch

from . import _lib

_native = _lib.native

# (query, key, value, scaling, causal, key_lo, key_hi, record, keep_lse) -> (out, lse, smax, valid)
_forward = _native.attention_forward
# (tensor) -> (the tensor or a copy that tile loads can read, its three leading strides)
_readable = _native.readable


def _index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def attention_status(device: torch.device) -> torch.Tensor:
    """Two device int32 words per GPU: [0] the first nonzero timeout code of an attention launch,
    [1] the stall request (0; tests set a role's code to make its first wait expire)."""
    return _native.attention_status(_index(device))


def check_attention_status(device: torch.device) -> None:
    """Raise if an attention launch on ``device`` reported an expired wait, which leaves NaN in the
    rows of the output or of the gradients that it concerns. Reads one word from the device, and
    nothing where no attention has been launched."""
    if device.type != "cuda" or _lib.native_error is not None or not _native.attention_used(_index(device)):
        return
    t = attention_status(device)
    code = int(t[0].item())
    if code != 0:
        t[0].zero_()
        raise _lib.MuzoError(f"fused attention reported status {code} (a bounded wait expired); outputs of the forward, "
                             "or gradients of the backward pass, that were computed then are NaN")


def attention_max(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: float | None = None,
                  causal: bool = True, key_lo: torch.Tensor | None = None, key_hi: torch.Tensor | None = None,
                  record: bool = True) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """softmax(scaling * Q K^T) V on the tensor cores for Q [B, Hq, Sq, D], K, V [B, Hkv, Sk, D]
    (transformers' transposed views; bf16 or fp16, D a multiple of 8 up to 128), returned as
    [B, Sq, Hq, D] (the layout attention functions return); with ``record``, also the per-head max
    of the eager pre-softmax logits and a validity word, on the device.

    ``causal``: query i sees the keys j <= i + Sk - Sq. ``key_lo`` / ``key_hi`` (int32 per batch)
    bound the visible keys to [key_lo, key_hi); what lies outside is not read into any result, not
    even when it is not finite (a key that only causality hides is multiplied by a probability of 0, so
    a NaN in it does reach queries of its tile). A query that sees no key gets zeros, and gives nothing
    to any gradient. ``scaling`` defaults to
    D ** -0.5.

    Differentiable once, in reverse mode, in query, key and value (the maxima are not; forward-mode
    derivatives and torch.func's transforms are refused): the products of the backward pass take the
    probabilities and their gradients in the inputs' type, as the forward does, and sum in fp32;
    dO . O is taken from the output as it is returned, rounded to the inputs' type. That rounding is
    what a row of query's gradient loses most by where one key has nearly all of its probability:
    dP - dO . O cancels, and the row, small itself, may be off by its own size.

    A backward pass can be captured into a CUDA graph while no graph of the same leaves that was built
    on another stream is alive (torch ends such a capture with an error)."""
    return _native.attention(query, key, value, scaling, causal, key_lo, key_hi, record)


def attention_max_backward(grad_out: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                           out: torch.Tensor, lse: torch.Tensor, scaling: float | None = None, causal: bool = True,
                           key_lo: torch.Tensor | None = None, key_hi: torch.Tensor | None = None,
                           ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients (dQ, dK, dV) of ``attention_max`` for callers that run their own autograd:
    ``out`` and ``grad_out`` are [B, Sq, Hq, D], ``lse`` [B, Hq, Sq] fp32 is the natural logarithm
    of each row's sum of exp(scaled logit) over the keys it sees (-inf where it sees none). The
    other arguments are the forward's. The gradients have the shapes of query, key and value (dK and
    dV summed over the query heads of each key head)."""
    return _native.attention_backward(grad_out, query, key, value, out, lse, scaling, causal, key_lo, key_hi,
                                      (True, True, True))

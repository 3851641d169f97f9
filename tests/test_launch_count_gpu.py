"""The package's count of the kernels it enqueued is what the device ran."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _states(device, hq, hkv, s, dtype=torch.bfloat16):
    g = torch.Generator(device="cpu").manual_seed(s)
    return [torch.randn((1, h, s, 64), generator=g).to(dtype).to(device).requires_grad_(True) for h in (hq, hkv, hkv)]


def _attention(device, *shape, dtype=torch.bfloat16, record=True):
    from muzo_clip_b200 import attention_max

    x = _states(device, *shape, dtype)

    def run():
        out = attention_max(*x, record=record)[0]
        torch.autograd.grad(out, x, out.detach())

    return run


def _clip(device, count):
    from muzo_clip_b200 import clip_grads, grad_norm

    grads = [torch.ones(5, device=device) for _ in range(count)]

    def run():
        grad_norm(grads)
        clip_grads(grads, 1.0)

    return run


def _qk(device):
    from muzo_clip_b200 import _qk

    q, k, _ = (x.detach() for x in _states(device, 4, 2, 130))
    return lambda: _qk.qk_head_max(q, k, 0.125, True, None)


CALLS = {
    "attention": (lambda d: _attention(d, 4, 2, 100), 5),
    "attention without maxima": (lambda d: _attention(d, 4, 2, 100, record=False), 3),
    "divided key tiles": (lambda d: _attention(d, 8, 1, 1024, record=False), 4),
    "divided key tiles, fp16": (lambda d: _attention(d, 8, 1, 1024, dtype=torch.float16), 6),
    "norm and clip": (lambda d: _clip(d, 3), 4),
    "norm and clip of 2500 tensors": (lambda d: _clip(d, 2500), 10),
    "maximum logit": (_qk, 3),
}


@pytest.mark.parametrize("name", CALLS)
def test_count(device, name):
    from muzo_clip_b200 import _lib

    make, expected = CALLS[name]
    run = make(device)
    run()
    torch.cuda.synchronize()
    before = _lib.launches()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        run()
        torch.cuda.synchronize()
    counted = _lib.launches() - before
    ran = [e.name for e in prof.events() if "muzo::" in e.name]
    assert counted == expected
    if prof.events():      # where the profiler may read the device's activity
        assert len(ran) == counted, ran

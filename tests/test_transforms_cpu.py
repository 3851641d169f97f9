"""Function transforms that the gradient operators do not take are refused, not answered without their part:
forward-mode derivatives, torch.func's gradients and vmap."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from muzo_clip_b200 import attention_max, attention_max_backward, clip_grads, grad_norm


def _states():
    g = torch.Generator().manual_seed(0)
    return [torch.randn((2, 2, 8, 64), generator=g).bfloat16() for _ in range(3)]


@pytest.mark.parametrize("place", range(3))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(place, grad):
    x = _states()
    with fwAD.dual_level():
        x[place] = fwAD.make_dual(x[place], torch.ones_like(x[place]))
        if grad:
            x[(place + 1) % 3].requires_grad_(True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention_max(*x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            attention_max(*x)
        out = x[0].detach().transpose(1, 2)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention_max_backward(out, *x, out, torch.zeros((2, 2, 8)))


def test_forward_mode_in_the_other_arguments_is_refused():
    x = _states()
    out = x[0].transpose(1, 2)
    with fwAD.dual_level():
        dual = fwAD.make_dual(out, torch.ones_like(out))
        lse = fwAD.make_dual(torch.zeros((2, 2, 8)), torch.ones((2, 2, 8)))
        for args in ((dual, *x, out, torch.zeros((2, 2, 8))), (out, *x, dual, torch.zeros((2, 2, 8))), (out, *x, out, lse)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                attention_max_backward(*args)


def test_forward_mode_gradients_are_refused():
    with fwAD.dual_level():
        g = fwAD.make_dual(torch.ones(5), torch.ones(5))
        for call in (lambda: grad_norm([torch.ones(3), g]), lambda: clip_grads([g], 1.0), lambda: clip_grads([torch.ones(5)], 1.0, out=[g])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_torch_func_is_refused():
    q, k, v = _states()

    def f(x):
        return attention_max(x, k, v)[0].float().sum()

    for call in (lambda: torch.func.grad(f)(q), lambda: torch.func.jvp(f, (q,), (q,)),
                 lambda: torch.func.vmap(lambda x: attention_max(x, k, v)[0])(q[None]),
                 lambda: torch.func.vmap(lambda x: grad_norm([x]))(torch.ones(2, 3)),
                 lambda: torch.func.grad(lambda x: grad_norm([x]))(torch.ones(3))):
        with pytest.raises(NotImplementedError, match="torch.func|forward-mode"):
            call()

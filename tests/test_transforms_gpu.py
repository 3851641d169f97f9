"""Forward-mode derivatives of CUDA tensors are refused: an output without its tangent would be taken for one
that does not depend on the input."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def test_a_tangent_is_not_dropped(device):
    from muzo_clip_b200 import attention_max, grad_norm

    x = torch.randn((1, 2, 16, 64), device=device).bfloat16()
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention_max(x, dual, x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            grad_norm([dual])
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.vmap(lambda q: attention_max(q, x, x)[0])(x[None])
    assert bool(torch.isfinite(attention_max(x, x, x)[0]).all())

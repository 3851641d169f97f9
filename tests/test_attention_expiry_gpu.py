"""What a program sees of an attention launch whose bounded wait expired: outputs and gradients that are
not finite, without having asked, and the status word with its message."""

from __future__ import annotations

import pytest
import torch

from test_attention_backward_gpu import _states

pytestmark = pytest.mark.gpu

SHAPES = [  # b, hq, hkv, sq, sk, d
    (1, 2, 2, 300, 300, 64),
    (2, 4, 2, 150, 270, 128),
    (1, 8, 1, 520, 520, 128),     # key tiles divided: the sums of their parts are joined
    (1, 2, 1, 130, 130, 40),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("role", [1, 2, 3])
@pytest.mark.parametrize("shape", SHAPES)
def test_an_expired_launch_leaves_nan(device, dtype, role, shape):
    """Every CTA of a stalled launch gives up: all of the output, the row statistics and the gradients are
    NaN, whatever their memory held, and the call after it is right."""
    from muzo_clip_b200 import _lib, attention_max_backward, check_attention_status
    from muzo_clip_b200.attention import _forward, attention_status

    q, k, v, dout = _states(device, dtype, *shape, seed=80)

    def forward():
        return _forward(q, k, v, 0.125, True, None, None, True, True)

    out, lse, smax, _ = forward()
    want = attention_max_backward(dout, q, k, v, out, lse, 0.125, True)
    status = attention_status(device)
    status.zero_()
    status[1] = role
    try:
        lost, lost_lse, _, valid = forward()
        torch.cuda.synchronize()
        assert int(status[0].item()) == role and int(valid) == 0
        assert bool(torch.isnan(lost).all()) and bool(torch.isnan(lost_lse).all())
        with pytest.raises(_lib.MuzoError, match="expired"):
            check_attention_status(device)
        gone = attention_max_backward(dout, q, k, v, out, lse, 0.125, True)
        torch.cuda.synchronize()
        assert int(status[0].item()) == role
        for name, g in zip(("dq", "dk", "dv"), gone):
            assert bool(torch.isnan(g).all()), name
        with pytest.raises(_lib.MuzoError, match="gradients"):
            check_attention_status(device)
    finally:
        status[1] = 0
    again = forward()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse) and torch.equal(again[2], smax)
    got = attention_max_backward(dout, q, k, v, out, lse, 0.125, True)
    check_attention_status(device)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_training_step_sees_it(device):
    """Forward and backward through autograd, nothing asked: the loss and the gradient norm are NaN."""
    from muzo_clip_b200 import attention_max, grad_norm
    from muzo_clip_b200.attention import attention_status

    q, k, v, _ = _states(device, torch.bfloat16, 1, 4, 2, 200, 200, 64, seed=81)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    status = attention_status(device)
    status.zero_()
    status[1] = 2
    try:
        loss = attention_max(*leaves, record=False)[0].float().square().sum()
        loss.backward()
        torch.cuda.synchronize()
    finally:
        status.zero_()
    assert bool(torch.isnan(loss)) and bool(torch.isnan(grad_norm([x.grad for x in leaves])))

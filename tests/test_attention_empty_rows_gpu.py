"""Query rows that see no key (left padding under causality, more queries than keys) may hold anything in
Q and in the output's gradient: nothing of them reaches the output, the maxima or any gradient, bit for bit,
and their own output and gradient are zero."""

from __future__ import annotations

import math

import pytest
import torch

from test_attention_backward_gpu import _range, _states, _visible

pytestmark = pytest.mark.gpu

CASES = [  # b, hq, hkv, sq, sk, d, lo, hi: causal, rows in front of the first visible key see nothing
    (3, 4, 2, 300, 300, 128, [0, 37, 150], [300, 300, 290]),      # left padding, inside and behind a tile
    (2, 4, 4, 140, 140, 64, [5, 128], [140, 140]),                # the rows of a whole tile
    (1, 2, 2, 300, 140, 64, None, None),                          # Sq > Sk
    (1, 2, 1, 200, 129, 128, None, [100]),                        # both ends
    (1, 8, 1, 520, 520, 128, [201], None),                        # divided key tiles
    (1, 3, 3, 99, 99, 40, [98], None),                            # one row is left
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 60000.0])
@pytest.mark.parametrize("b,hq,hkv,sq,sk,d,lo,hi", CASES)
def test_rows_without_a_key_reach_nothing(device, dtype, bad, b, hq, hkv, sq, sk, d, lo, hi):
    from muzo_clip_b200 import attention_max
    from muzo_clip_b200.attention import check_attention_status

    q, k, v, dout = _states(device, dtype, b, hq, hkv, sq, sk, d, seed=70)
    lo_t, hi_t = _range(device, b, lo, hi)
    empty = ~_visible(b, sq, sk, True, lo, hi, device)[:, 0].any(-1)          # [B, Sq]
    assert bool(empty.any()) and not bool(empty.all())
    results = []
    for fill in (0.0, bad):
        leaves = [q.masked_fill(empty[:, None, :, None], fill).requires_grad_(True)] + \
                 [x.clone().requires_grad_(True) for x in (k, v)]
        out, smax, valid = attention_max(*leaves, d ** -0.5, True, lo_t, hi_t)
        g = dout.masked_fill(empty[:, :, None, None], fill)
        results.append([out.detach(), smax, valid, *torch.autograd.grad(out, leaves, g)])
    check_attention_status(device)
    for name, a, c in zip(("out", "smax", "valid", "dq", "dk", "dv"), *results):
        assert bool(torch.isfinite(c).all()), name
        assert torch.equal(a, c), name
    out, dq = results[1][0], results[1][3]
    assert not bool(out[empty].any()) and not bool(dq.transpose(1, 2)[empty].any())
    assert bool(results[1][4].any()) and bool(results[1][5].any())

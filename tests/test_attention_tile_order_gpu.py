"""Long walks over tiles in the backward kernel, where every tensor-memory column is taken again and again: P
and dS of one tile, S and dP of the next. A product that read its operand after the next tile had taken the
columns would show against the formulas, or between runs beside other work."""

from __future__ import annotations

import pytest
import torch

from test_attention_backward_gpu import _assert_within, _exact, _states, _visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,hkv,sq,sk,d,causal", [
    (1, 4, 4, 2500, 130, 128, False),     # key CTAs with twenty tiles each
    (1, 4, 4, 2500, 130, 64, False),
    (1, 2, 2, 130, 2500, 128, False),     # query CTAs with twenty
    (1, 2, 2, 130, 2500, 64, False),
    (1, 6, 1, 1400, 1400, 128, True),     # divided key tiles
    (1, 6, 1, 1400, 1400, 40, True),
])
def test_long_walks(device, dtype, b, hq, hkv, sq, sk, d, causal):
    from muzo_clip_b200 import attention_max_backward
    from muzo_clip_b200.attention import _forward, check_attention_status

    q, k, v, dout = _states(device, dtype, b, hq, hkv, sq, sk, d, seed=90)
    scale = d ** -0.5
    out, lse, _, _ = _forward(q, k, v, scale, causal, None, None, False, True)
    first = attention_max_backward(dout, q, k, v, out, lse, scale, causal)
    ref = _exact(q, k, v, dout, scale, _visible(b, sq, sk, causal, None, None, device), out)
    _assert_within(first, ref)
    # the same bits beside other work on the same SMs' tensor cores and memory
    side = torch.cuda.Stream(device)
    a = torch.randn((2048, 2048), device=device, dtype=dtype)
    for _ in range(10):
        with torch.cuda.stream(side):
            a = (a @ a) * 2.0 ** -6
        got = attention_max_backward(dout, q, k, v, out, lse, scale, causal)
        assert all(torch.equal(x, y) for x, y in zip(got, first))
    torch.cuda.current_stream(device).wait_stream(side)
    check_attention_status(device)

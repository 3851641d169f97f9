"""The norm over many gradients and clipping by it (muzo_grad_norm, muzo_grad_clip) against 64-bit
sums and torch's own clip_grad_norm_.

The norm's tolerance: eight squares are added in fp32 (8 * 2^-24 of their sum at worst), the rest in
fp64, and the root halves a relative error: 4 * 2^-24, plus the rounding to fp32, 2^-24. A scaled
gradient is one fp32 product with a factor that is off by the norm's error and two fp32 roundings
(8 * 2^-24 in all), rounded to its type (eps / 2).
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

NORM_TOL = 5 * 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _exact_norm(grads, inf=False):
    if inf:
        return max((float(g.double().abs().max()) for g in grads if g.numel()), default=0.0)
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def _grads(device, dtype, sizes, seed=0, gain=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return [(torch.randn(s, generator=g) * gain).to(dtype).to(device) for s in sizes]


SIZES = [
    [1], [7], [8], [2047], [2048], [2049], [1, 3, 0, 5], [16385, 1, 70000],
    [(33, 65), (1024, 688), (0, 4), (5,)], [3_000_017], [13] * 139, [13] * 141, [(17, 3)] * 1200, [0], [0, 0],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_norm_and_clip(device, dtype, sizes):
    from muzo_clip_b200 import clip_grads, grad_norm

    grads = _grads(device, dtype, sizes, len(sizes))
    want = _exact_norm(grads)
    norm = grad_norm(grads)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.device == device
    assert abs(float(norm) - want) <= NORM_TOL * want
    assert float(grad_norm(grads, math.inf)) == _exact_norm(grads, True)
    for max_norm in (0.5 * want, 0.0, 2 * want + 1):
        factor = min(1.0, max_norm / (want + 1e-6))
        for out_dtype in {dtype, torch.float32}:
            dest = [torch.full_like(x, 7.0, dtype=out_dtype) for x in grads]
            before = [x.clone() for x in grads]
            out, got = clip_grads(grads, max_norm, out=dest)
            assert torch.equal(got, norm) and all(a is b for a, b in zip(out, dest))
            tol = (torch.finfo(out_dtype).eps / 2 if out_dtype != torch.float32 else 0.0) + 8 * 2.0 ** -24
            tiny = 2.0 ** -24 if out_dtype == torch.float16 else 0.0
            for g, o, c in zip(grads, out, before):
                assert torch.equal(g, c)
                assert bool(((o.double() - g.double() * factor).abs() <= tol * (g.double() * factor).abs() + tiny).all())
                if factor == 1.0:
                    assert torch.equal(o.to(dtype), g)
    fresh, got = clip_grads(grads, 0.5 * want)
    in_place = [x.clone() for x in grads]
    out, again = clip_grads(in_place, 0.5 * want, out=in_place)
    assert torch.equal(got, again) and all(torch.equal(a, c) for a, c in zip(fresh, in_place))


def test_types_mix(device):
    from muzo_clip_b200 import clip_grads, grad_norm

    grads = [x for d in DTYPES for x in _grads(device, d, [5, (100, 33), 40000], 3)]
    want = _exact_norm(grads)
    assert abs(float(grad_norm(grads)) - want) <= NORM_TOL * want
    out, _ = clip_grads(grads, 1.0)
    assert [o.dtype for o in out] == [g.dtype for g in grads]
    assert abs(_exact_norm(out) - 1.0) <= 2.0 ** -8


@pytest.mark.parametrize("gain", [1e-30, 1e-21, 1e18, 1e25, 3e37])
def test_squares_beyond_fp32(device, gain):
    """Values whose squares leave fp32's range, and small values beside large ones. The norm itself
    is an fp32 value: sqrt(14103) * 3e37 = 3.6e39 lies above the largest one, 3.4e38, and is inf."""
    from muzo_clip_b200 import grad_norm

    grads = _grads(device, torch.float32, [10007, (64, 64)], 1, gain)
    for more in ([], [torch.ones(100, device=device)]):
        want = _exact_norm(grads + more)
        got = float(grad_norm(grads + more))
        if want > torch.finfo(torch.float32).max:
            assert got == math.inf
        else:
            assert abs(got - want) <= NORM_TOL * want


def test_zeros_and_subnormals(device):
    from muzo_clip_b200 import clip_grads, grad_norm

    z = [torch.zeros(5000, device=device), torch.zeros(33, device=device, dtype=torch.bfloat16)]
    assert float(grad_norm(z)) == 0.0 and float(grad_norm(z, math.inf)) == 0.0
    out, _ = clip_grads(z, 1.0)
    assert not any(bool(o.any()) for o in out)
    s = [torch.full((1000,), 2.0 ** -24, dtype=torch.float16, device=device)]
    want = 2.0 ** -24 * math.sqrt(1000)
    assert abs(float(grad_norm(s)) - want) <= NORM_TOL * want
    z[0][4999] = -3.0
    assert float(grad_norm(z)) == 3.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_nonfinite_gradients_as_in_torch(device, dtype, bad, norm_type):
    from muzo_clip_b200 import clip_grad_norm_

    params = [torch.nn.Parameter(torch.zeros(s, device=device, dtype=dtype)) for s in (5, 3000, 40000)]
    for p, g in zip(params, _grads(device, dtype, [5, 3000, 40000], 2)):
        p.grad = g
    params[1].grad[2999] = bad
    with pytest.raises(RuntimeError):
        kept = [p.grad.clone() for p in params]
        clip_grad_norm_(params, 1.0, norm_type, error_if_nonfinite=True)
    assert all(torch.equal(torch.nan_to_num(p.grad), torch.nan_to_num(k)) for p, k in zip(params, kept))
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for t, p in zip(twins, params):
        t.grad = p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(twins, 1.0, norm_type)
    got = clip_grad_norm_(params, 1.0, norm_type)
    assert torch.equal(torch.isnan(want), torch.isnan(got)) and (torch.isnan(got) or float(got) == float(want))
    for t, p in zip(twins, params):
        assert torch.equal(torch.isnan(t.grad), torch.isnan(p.grad))
        assert torch.equal(torch.nan_to_num(t.grad), torch.nan_to_num(p.grad))


def test_in_place_against_torch(device):
    """Parameters without gradients are skipped; the version counters of the gradients move."""
    from muzo_clip_b200 import clip_grad_norm_

    params = [torch.nn.Parameter(torch.zeros(s, device=device)) for s in (7, (50, 60), 9, 100000)]
    for i, g in zip((0, 1, 3), _grads(device, torch.float32, [7, (50, 60), 100000], 6)):
        params[i].grad = g
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for t, p in zip(twins, params):
        t.grad = None if p.grad is None else p.grad.clone()
    versions = [params[i].grad._version for i in (0, 1, 3)]
    got = clip_grad_norm_((p for p in params), 2.0)
    want = torch.nn.utils.clip_grad_norm_(twins, 2.0)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want) and params[2].grad is None
    for i in (0, 1, 3):
        assert torch.allclose(params[i].grad, twins[i].grad, rtol=1e-5, atol=0.0)
    assert all(params[i].grad._version > v for i, v in zip((0, 1, 3), versions))
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    assert float(clip_grad_norm_(torch.nn.Parameter(torch.zeros(3, device=device)), 1.0)) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(device, dtype):
    """Views into a flat bucket at odd offsets, transposed, sliced and channels-last gradients: the
    values of contiguous ones, and nothing beside them is written."""
    from muzo_clip_b200 import clip_grads, grad_norm

    bucket = _grads(device, dtype, [100003], 4)[0]
    cuts = [0, 1, 38, 5001, 5004, 60000, 100003]
    views = [bucket[a:z] for a, z in zip(cuts, cuts[1:])]
    big = _grads(device, dtype, [(60, 90)], 5)[0]
    image = _grads(device, dtype, [(2, 3, 8, 8)], 7)[0].contiguous(memory_format=torch.channels_last)
    others = [big[3:50, 1:77], big.t(), image, big[::2, ::3]]
    for grads in (views, others[:1] + views, [others[1]], [others[2]], [others[3]]):
        copies = [g.clone(memory_format=torch.contiguous_format) for g in grads]
        assert torch.allclose(grad_norm(grads), grad_norm(copies), rtol=2 * NORM_TOL, atol=0.0)
        base = [bucket.clone(), big.clone()]
        want, norm = clip_grads(copies, 0.25 * float(grad_norm(copies)))
        got, norm2 = clip_grads(grads, 0.25 * float(grad_norm(copies)))
        assert all(torch.allclose(a.float(), c.float(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -24) for a, c in zip(got, want))
        assert torch.equal(base[0], bucket) and torch.equal(base[1], big)
        # in place: only the views' elements change
        clip_grads(grads, 0.25 * float(grad_norm(copies)), out=grads)
        assert all(torch.allclose(a.float(), c.float(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -24) for a, c in zip(grads, want))
        if grads is views:
            assert torch.equal(torch.cat(views), bucket) and torch.equal(base[1], big)
        else:
            touched = torch.zeros_like(big, dtype=torch.bool)
            touched[3:50, 1:77] = grads[0].shape == (47, 76)
            touched |= grads[0].shape == (90, 60)
            if grads[0].shape == others[3].shape:
                touched[::2, ::3] = True
            assert torch.equal(big[~touched], base[1][~touched])
        bucket.copy_(base[0])
        big.copy_(base[1])


def test_equal_calls_give_equal_bits(device):
    from muzo_clip_b200 import clip_grads, grad_norm

    grads = _grads(device, torch.bfloat16, [5_000_011, 77, (3000, 700)], 12)
    first, outs = grad_norm(grads), clip_grads(grads, 3.0)[0]
    for _ in range(10):
        assert torch.equal(grad_norm(grads), first)
        assert all(torch.equal(a, c) for a, c in zip(clip_grads(grads, 3.0)[0], outs))


def test_streams_and_graphs(device):
    """Two streams at once, and two captured graphs replayed in turn on new gradients."""
    from muzo_clip_b200 import clip_grads

    held = [_grads(device, torch.float32, [200000 + i, 33], i) for i in range(2)]
    want = [clip_grads(h, 1.0) for h in held]
    streams = [torch.cuda.Stream(device) for _ in held]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream(device))
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = clip_grads(held[i], 1.0)
    torch.cuda.synchronize()
    for (a, n), (c, m) in zip(got, want):
        assert torch.equal(n, m) and all(torch.equal(x, y) for x, y in zip(a, c))
    graphs, results = [], []
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(clip_grads(h, 1.0))
        graphs.append(graph)
    for trial in range(3):
        for i, h in enumerate(held):
            for x, y in zip(h, _grads(device, torch.float32, [200000 + i, 33], 30 + trial + i, 2.0)):
                x.copy_(y)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for h, (a, n) in zip(held, results):
            c, m = clip_grads(h, 1.0)
            assert torch.equal(n, m) and all(torch.equal(x, y) for x, y in zip(a, c))


def test_more_than_32_bits_of_elements(device):
    """A gradient of more than 2^32 bytes: the far end counts and is scaled."""
    from muzo_clip_b200 import clip_grads, grad_norm

    g = torch.zeros((1 << 31) + 4099, dtype=torch.bfloat16, device=device)
    g[-1], g[0], g[1 << 31] = 3.0, 4.0, 12.0
    assert float(grad_norm([g])) == 13.0
    clip_grads([g], 6.5, out=[g])
    assert abs(float(g[-1]) - 1.5) <= 2.0 ** -7 and abs(float(g[1 << 31]) - 6.0) <= 2.0 ** -5
    assert float(g[5]) == 0.0


def test_refusals(device):
    from muzo_clip_b200 import clip_grad_norm_, clip_grads, grad_norm

    g = torch.ones(100, device=device)
    for call, kind in ((lambda: grad_norm([g], 1.0), ValueError), (lambda: grad_norm([g.double()]), TypeError),
                       (lambda: grad_norm([g.cpu()]), ValueError), (lambda: grad_norm([g, g.cpu()]), ValueError),
                       (lambda: grad_norm([1.0]), TypeError), (lambda: grad_norm([g.to_sparse()]), ValueError),
                       (lambda: clip_grads([g], -1.0), ValueError), (lambda: clip_grads([g], math.nan), ValueError),
                       (lambda: clip_grads([g], 1.0, out=[]), ValueError),
                       (lambda: clip_grads([g], 1.0, out=[g[:50]]), ValueError),
                       (lambda: clip_grads([g], 1.0, out=[g.half()]), ValueError),
                       (lambda: clip_grads([g, g], 1.0, out=[g, g]), ValueError),          # the same one twice
                       (lambda: clip_grads([g[:60], g[50:]], 1.0, out=[g[:60], g[50:]]), ValueError),
                       (lambda: clip_grads([g[:50], g[50:]], 1.0, out=[g[50:], g[:50]]), ValueError)):
        with pytest.raises(kind):
            call()
    assert bool((g == 1.0).all())
    p = torch.nn.Parameter(torch.ones(4, device=device))
    p.grad = torch.ones(1, device=device).expand(4)
    with pytest.raises((RuntimeError, ValueError)):
        clip_grad_norm_(p, 0.5)

"""The backward pass of attention_max (muzo_attention_backward) and the row statistics the forward
keeps for it, against the formulas in 64 bits.

Tolerances are the rounding steps the kernels take, summed worst case with |.| in place of every
factor: P and dS enter the products rounded to the input type (half a step u = eps / 2, relative;
fp16 has subnormals, half a step of which is 2^-25: of 2^10 P, and of dS times the power of two
that brings 2 max|dO_i| max|v_j| to between 2^14 and 2^15), results are rounded once more (u), and fp32 dot
products of n terms are off by at most n * 2^-23 of the sum of their terms' magnitudes (2^-16 for the
128 products of a logit). With autograd, delta = dO . O uses the forward's O, which is rounded (u) and
took P rounded (u sum P |v|).
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _visible(b, sq, sk, causal, lo, hi, device):
    i = torch.arange(sq, device=device)[:, None] + (sk - sq)
    j = torch.arange(sk, device=device)[None, :]
    vis = torch.ones((b, sq, sk), dtype=torch.bool, device=device)
    if causal:
        vis &= j <= i
    for bi in range(b):
        if lo is not None:
            vis[bi] &= j >= int(lo[bi])
        if hi is not None:
            vis[bi] &= j < int(hi[bi])
    return vis[:, None]


def _exact(q, k, v, dout, scale, vis, out=None):
    """O, lse, dQ, dK, dV in 64 bits and a bound on the kernels' error in each gradient. `out`: the
    O that delta is taken from (otherwise the exact one, whose rounding the bound then counts)."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    s_p = s_ds = 0.0
    if dtype == FP16:
        s_p = 2.0 ** -35
        largest = 2 * float(dout.double().norm(dim=-1).max()) * float(torch.nan_to_num(v.double(), 0.0, 0.0, 0.0).norm(dim=-1).max())
        s_ds = 2.0 ** -25 * max(largest / 2.0 ** 14, 2.0 ** -40)
    b, hq, sq, d = q.shape
    hkv, sk = k.shape[1], k.shape[2]
    group = hq // hkv
    qd, kd, vd = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    hidden_keys = ~vis.any(dim=-2).expand(b, 1, sk)          # keys nobody sees: whatever they hold is not read
    kd = kd.masked_fill(hidden_keys[..., None], 0.0)
    vd = vd.masked_fill(hidden_keys[..., None], 0.0)
    g = dout.double().transpose(1, 2)
    logits = (qd @ kd.transpose(2, 3) * scale).masked_fill(~vis, -math.inf)
    lse = torch.logsumexp(logits, dim=-1)
    p = torch.exp(logits - torch.where(lse == -math.inf, 0.0, lse)[..., None]).masked_fill(~vis, 0.0)
    o = p @ vd
    used = o if out is None else out.double().transpose(1, 2)
    delta = (g * used).sum(-1, keepdim=True)
    dp = g @ vd.transpose(2, 3)
    ds = p * (dp - delta)
    dq = ds @ kd * scale
    dk = (ds.transpose(2, 3) @ qd * scale).view(b, hkv, group, sk, d).sum(2)
    dv = (p.transpose(2, 3) @ g).view(b, hkv, group, sk, d).sum(2)
    # the bounds
    ga, ka, va, qa = g.abs(), kd.abs(), vd.abs(), qd.abs()
    rel_p = 2.0 ** -16 * (1 + scale * (qa @ ka.transpose(2, 3))) + 2.0 ** -22 * torch.where(lse == -math.inf, 0.0, lse.abs())[..., None]
    err_delta = (ga * used.abs()).sum(-1, keepdim=True) * 2.0 ** -16
    if out is None:
        err_delta = err_delta + (ga * (u * used.abs() + (u + 2.0 ** -16) * (p @ va))).sum(-1, keepdim=True)
    err_dp = 2.0 ** -16 * (ga @ va.transpose(2, 3))
    err_p = p * (rel_p + u) + s_p * vis
    err_ds = (ds.abs() * (u + rel_p) + p * (err_dp + err_delta)) * 1.01 + s_ds * vis
    n = 2.0 ** -23 * max(sq * group, sk)
    t_dq = ((err_ds + n * ds.abs()) @ ka) * scale + u * dq.abs()
    t_dk = ((err_ds + n * ds.abs()).transpose(2, 3) @ qa * scale).view(b, hkv, group, sk, d).sum(2) + u * dk.abs()
    t_dv = ((err_p + n * p).transpose(2, 3) @ ga).view(b, hkv, group, sk, d).sum(2) + u * dv.abs()
    extra = 2.0 ** -25 if dtype == FP16 else 0.0     # a result among the subnormals of fp16
    return {"out": o.transpose(1, 2), "lse": lse, "dq": dq, "dk": dk, "dv": dv,
            "t_dq": t_dq * 1.05 + 1e-30 + extra, "t_dk": t_dk * 1.05 + 1e-30 + extra, "t_dv": t_dv * 1.05 + 1e-30 + extra}


def _states(device, dtype, b, hq, hkv, sq, sk, d, seed=0, gain=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed + 7 * sq + 3 * sk + d + hq)

    def x(s, h, f):
        return (torch.randn((b, s, h, d), generator=g) * f).to(dtype).to(device).transpose(1, 2)

    return x(sq, hq, 1.2 * gain), x(sk, hkv, 1.2 * gain), x(sk, hkv, 1.0), x(sq, hq, 0.5).transpose(1, 2)


def _range(device, b, lo, hi):
    def t(x):
        return None if x is None else torch.tensor(x, dtype=torch.int32, device=device)

    return t(lo), t(hi)


def _assert_within(got, ref, names=("dq", "dk", "dv")):
    for name, t in zip(names, got):
        err = (t.double() - ref[name]).abs()
        over = err - ref["t_" + name]
        assert bool(torch.isfinite(t).all()), name
        assert float(over.max()) <= 0.0, (name, float(err.max()), float((err / ref["t_" + name]).max()))


CASES = [  # b, hq, hkv, sq, sk, d, causal, lo, hi
    (1, 1, 1, 1, 2, 64, True, None, None),
    (2, 2, 1, 1, 300, 128, True, None, None),          # one query against many keys
    (4, 4, 4, 64, 64, 64, True, None, None),           # the tiny Llama's heads
    (2, 6, 2, 77, 77, 128, True, None, None),
    (1, 4, 4, 128, 128, 64, False, None, None),        # exactly one tile
    (1, 2, 2, 129, 257, 128, False, None, None),       # one row beyond a tile
    (2, 8, 2, 300, 300, 64, True, None, None),
    (1, 4, 2, 100, 356, 128, True, None, None),        # end-aligned causal window
    (1, 2, 2, 300, 140, 64, True, None, None),         # Sq > Sk: the first rows see no key
    (1, 8, 1, 520, 520, 128, True, None, None),        # one key head for all: the work is divided
    (3, 4, 2, 300, 300, 128, True, [0, 37, 150], [300, 300, 290]),
    (3, 4, 2, 300, 300, 128, False, [0, 137, 299], [1, 260, 300]),
    (3, 2, 2, 200, 200, 64, False, [0, 50, 120], [0, 50, 90]),     # ranges that leave nothing
    (2, 4, 4, 70, 190, 64, True, None, [190, 121]),
    (1, 2, 1, 130, 130, 32, True, None, None),         # head dimensions below a tile's
    (2, 2, 2, 150, 150, 8, False, None, None),
    (1, 4, 2, 140, 270, 96, True, [128], None),
    (1, 3, 3, 99, 99, 104, True, None, None),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,hq,hkv,sq,sk,d,causal,lo,hi", CASES)
def test_backward_against_the_formula(device, dtype, b, hq, hkv, sq, sk, d, causal, lo, hi):
    from muzo_clip_b200 import attention_max, attention_max_backward
    from muzo_clip_b200.attention import _forward, check_attention_status

    q, k, v, dout = _states(device, dtype, b, hq, hkv, sq, sk, d)
    lo_t, hi_t = _range(device, b, lo, hi)
    scale = d ** -0.5
    vis = _visible(b, sq, sk, causal, lo, hi, device)

    out, lse, _, _ = _forward(q, k, v, scale, causal, lo_t, hi_t, False, True)
    got = attention_max_backward(dout, q, k, v, out, lse, scale, causal, lo_t, hi_t)
    check_attention_status(device)
    ref = _exact(q, k, v, dout, scale, vis, out)
    # lse: fp32 logits of d products, an fp32 sum of sk terms, the exponential's 2^-22
    assert torch.equal(lse == -math.inf, ref["lse"] == -math.inf)
    seen = ref["lse"] != -math.inf
    top = float((q.double().abs() @ k.double().abs().repeat_interleave(hq // hkv, 1).transpose(2, 3)).max()) * scale
    assert float((lse.double() - ref["lse"])[seen].abs().max() if seen.any() else 0.0) <= 2.0 ** -16 * (1 + top) + 2.0 ** -23 * sk
    assert [tuple(t.shape) for t in got] == [tuple(q.shape), tuple(k.shape), tuple(v.shape)]
    _assert_within(got, ref)
    # rows that see nothing and keys that nobody sees have no gradient at all
    empty = ~vis.any(-1).expand(b, 1, sq).expand(b, hq, sq)
    assert not bool(got[0][empty].any())
    unseen = ~vis.any(-2).expand(b, 1, sk).expand(b, hkv, sk)
    assert not bool(got[1][unseen].any()) and not bool(got[2][unseen].any())

    # the same through autograd, where delta comes from the forward's rounded output
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    o2, smax, valid = attention_max(*leaves, scale, causal, lo_t, hi_t)
    assert not smax.requires_grad and int(valid) == 1 and torch.equal(o2, out)
    grads = torch.autograd.grad(o2, leaves, dout)
    _assert_within(grads, _exact(q, k, v, dout, scale, vis))
    for a, c in zip(grads, got):
        assert torch.equal(a, c)   # and the same bits as the direct call


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gradient_against_differences(device, dtype):
    """The directional derivative of sum(w * O) along a random direction of each input, by central
    differences of the 64-bit forward (error of order h^2: 1e-9 here), against the kernel's gradient;
    the gradient's own bound, summed along the direction, is the tolerance."""
    from muzo_clip_b200 import attention_max

    b, hq, hkv, sq, sk, d, scale = 1, 4, 2, 90, 150, 64, 0.125
    q, k, v, w = _states(device, dtype, b, hq, hkv, sq, sk, d, seed=11)
    vis = _visible(b, sq, sk, True, None, None, device)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    out, _, _ = attention_max(*leaves, scale, True, record=False)
    grads = torch.autograd.grad(out, leaves, w)
    ref = _exact(q, k, v, w, scale, vis)
    gen = torch.Generator(device="cpu").manual_seed(5)

    def f(xs):
        kd, vd = (x.repeat_interleave(hq // hkv, 1) for x in xs[1:])
        logits = (xs[0] @ kd.transpose(2, 3) * scale).masked_fill(~vis, -math.inf)
        return float((w.double() * (torch.softmax(logits, -1) @ vd).transpose(1, 2)).sum())

    base = [x.double() for x in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        direction = torch.randn(base[i].shape, generator=gen, dtype=torch.float64).to(device)
        h = 1e-5
        plus, minus = list(base), list(base)
        plus[i], minus[i] = base[i] + h * direction, base[i] - h * direction
        want = (f(plus) - f(minus)) / (2 * h)
        got = float((grads[i].double() * direction).sum())
        assert abs(got - want) <= float((ref["t_" + name] * direction.abs()).sum()) + 1e-6 * (1 + abs(want)), name


@pytest.mark.parametrize("gain", [2.0 ** -14, 2.0 ** -6, 2.0 ** 6])
def test_fp16_small_and_large_gradients(device, gain):
    """Gradients whose dS would be subnormal in fp16 (or overflow) without its power of two: as exact,
    relative to the largest result, as ordinary ones. V large too, for the bound's other factor."""
    from muzo_clip_b200 import attention_max_backward
    from muzo_clip_b200.attention import _forward

    b, hq, hkv, s, d, scale = 1, 4, 2, 700, 64, 0.125
    q, k, v, dout = _states(device, FP16, b, hq, hkv, s, s, d, seed=60)
    dout, v = dout * gain, v * (64.0 if gain > 1 else 1.0)
    vis = _visible(b, s, s, True, None, None, device)
    out, lse, _, _ = _forward(q, k, v, scale, True, None, None, False, True)
    got = attention_max_backward(dout, q, k, v, out, lse, scale, True)
    ref = _exact(q, k, v, dout, scale, vis, out)
    _assert_within(got, ref)
    for g, name in zip(got, ("dq", "dk", "dv")):
        err = (g.double() - ref[name]).abs()
        # P, dS and the result rounded: 2^-11 each of terms that sum to less than four times the largest result
        assert float(err.max()) <= 2.0 ** -9 * float(ref[name].abs().max()) + 2.0 ** -25, name


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("causal", [True, False])
def test_nonfinite_keys_outside_the_range_reach_nothing(device, bad, causal):
    """K and V behind key_hi and before key_lo hold NaN or infinities: the output and every gradient
    are bit for bit those with zeros there, and the padded keys' own gradients are zero."""
    from muzo_clip_b200 import attention_max

    b, hq, hkv, s, d = 3, 4, 2, 300, 128
    q, k, v, dout = _states(device, BF16, b, hq, hkv, s, s, d, seed=3)
    lo, hi = _range(device, b, [0, 37, 128], [200, 300, 299])
    j = torch.arange(s, device=device)
    outside = ((j < lo[:, None]) | (j >= hi[:, None]))[:, None, :, None].expand_as(k)
    results = []
    for fill in (0.0, bad):
        leaves = [q.clone().requires_grad_(True)] + [x.masked_fill(outside, fill).requires_grad_(True) for x in (k, v)]
        out, smax, valid = attention_max(*leaves, d ** -0.5, causal, lo, hi)
        results.append([out, smax, valid, *torch.autograd.grad(out, leaves, dout)])
    for a, c in zip(*results):
        assert torch.equal(a, c) and bool(torch.isfinite(a).all())
    assert not bool(results[1][4][outside].any()) and not bool(results[1][5][outside].any())


def test_nonfinite_logits_make_their_rows_nan(device):
    """A NaN among the keys a row sees gives that row NaN (not zeros), and leaves earlier rows of
    other tiles alone."""
    from muzo_clip_b200 import attention_max

    q, k, v, dout = _states(device, BF16, 1, 2, 2, 300, 300, 64, seed=4)
    k = k.clone()
    k[0, 0, 290, 3] = float("nan")
    out, _, valid = attention_max(q, k, v, 0.125, True)
    assert int(valid) == 0
    assert bool(torch.isnan(out[0, 290:, 0]).all()) and bool(torch.isfinite(out[0, :256]).all())
    assert bool(torch.isfinite(out[0, :, 1]).all())
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    o, _, _ = attention_max(*leaves, 0.125, True)
    dq, dk, dv = torch.autograd.grad(o, leaves, dout)
    assert bool(torch.isnan(dq[0, 0, 290:]).all()) and bool(torch.isfinite(dq[0, 1]).all())


def _layouts(t):
    """The same values in other memory: strided, not aligned to 16 bytes, D not contiguous."""
    b, h, s, d = t.shape
    wide = torch.zeros((b, h, s, 2 * d), dtype=t.dtype, device=t.device)
    wide[..., :d] = t
    yield wide[..., :d]
    flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    yield flat[1:].view(b, h, s, d)
    yield t.transpose(2, 3).contiguous().transpose(2, 3)
    odd = torch.zeros((b, h, s, d + 3), dtype=t.dtype, device=t.device)
    odd[..., :d] = t
    yield odd[..., :d]


def test_layouts_give_the_same_bits(device):
    from muzo_clip_b200 import attention_max

    q, k, v, dout = _states(device, BF16, 2, 4, 2, 150, 150, 64, seed=8)

    def run(q, k, v, g):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out, smax, _ = attention_max(*leaves, None, True)
        return [out.detach(), smax, *torch.autograd.grad(out, leaves, g)]

    want = run(q, k, v, dout)
    for ql, kl, vl, gl in zip(_layouts(q), _layouts(k), _layouts(v), _layouts(dout)):
        assert torch.equal(ql, q) and torch.equal(gl, dout)
        for a, c in zip(run(ql, kl, vl, gl), want):
            assert torch.equal(a, c)
    # expanded along the batch: one key sequence for both rows
    e = run(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), dout)
    c = run(q, k[:1].repeat(2, 1, 1, 1), v[:1].repeat(2, 1, 1, 1), dout)
    assert all(torch.equal(x, y) for x, y in zip(e, c))
    # out.sum() sends an expanded scalar back
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    attention_max(*leaves)[0].sum().backward()
    ones = run(q, k, v, torch.ones_like(dout))
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, ones[2:]))


@pytest.mark.parametrize("shape", [(1, 8, 1, 700, 700, 128), (2, 4, 4, 260, 260, 64)])
def test_equal_calls_give_equal_bits(device, shape):
    from muzo_clip_b200 import attention_max_backward
    from muzo_clip_b200.attention import _forward

    q, k, v, dout = _states(device, BF16, *shape, seed=9)
    out, lse, _, _ = _forward(q, k, v, 0.1, True, None, None, False, True)
    first = attention_max_backward(dout, q, k, v, out, lse, 0.1, True)
    for _ in range(5):
        again = attention_max_backward(dout, q, k, v, out, lse, 0.1, True)
        assert all(torch.equal(a, c) for a, c in zip(again, first))


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)])
def test_only_the_wanted_gradients(device, wanted):
    from muzo_clip_b200 import attention_max

    data = _states(device, BF16, 1, 4, 1, 300, 300, 128, seed=10)

    def run(flags):
        leaves = [x.detach().clone().requires_grad_(bool(w)) for x, w in zip(data[:3], flags)]
        out, _, _ = attention_max(*leaves)
        out.backward(data[3])
        return [x.grad for x in leaves]

    full, some = run((1, 1, 1)), run(wanted)
    for a, c, w in zip(some, full, wanted):
        assert (a is None) if not w else torch.equal(a, c)


@pytest.mark.parametrize("b,sq,sk", [(0, 5, 5), (2, 0, 7), (2, 7, 0), (0, 0, 0)])
def test_lengths_of_zero(device, b, sq, sk):
    from muzo_clip_b200 import attention_max

    q, k, v, dout = _states(device, BF16, b, 4, 2, sq, sk, 64)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    out, smax, valid = attention_max(*leaves)
    assert out.shape == (b, sq, 4, 64) and not bool(out.any())
    assert bool((smax == -math.inf).all()) and int(valid) == 1
    for x, g in zip(leaves, torch.autograd.grad(out, leaves, dout)):
        assert g.shape == x.shape and not bool(g.any())


def test_another_stream_and_two_at_once(device):
    from muzo_clip_b200 import attention_max

    sets = [_states(device, BF16, 1, 4, 2, 400, 400, 64, seed=20 + i) for i in range(2)]

    def run(q, k, v, g):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out, _, _ = attention_max(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream(device) for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream(device))
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(*sets[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, c) for a, c in zip(g, w))


def test_a_thread_without_a_context(device):
    """Forward and backward as the first CUDA work of a new thread, whose allocations all come from
    the cache: nothing before the kernels has bound the device's context to it."""
    import threading

    from muzo_clip_b200 import attention_max, attention_max_backward
    from muzo_clip_b200.attention import _forward

    q, k, v, dout = _states(device, BF16, 1, 4, 2, 200, 200, 64, seed=40)

    def run():
        out, lse, _, _ = _forward(q, k, v, 0.125, True, None, None, False, True)
        return [attention_max(q, k, v, 0.125, True)[0], *attention_max_backward(dout, q, k, v, out, lse, 0.125, True)]

    want = run()
    run()          # leaves blocks of every size in the cache
    got = []
    for _ in range(3):
        thread = threading.Thread(target=lambda: got.append(run()))
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(a, c) for g in got for a, c in zip(g, want))


def test_captured_and_replayed(device):
    """Two graphs of forward and backward (torch.autograd.grad, one key head: divided work with a
    workspace), replayed in turn on new inputs."""
    from muzo_clip_b200 import attention_max

    def run(q, k, v, g):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out, _, _ = attention_max(*leaves, None, True)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    held = [[x.clone() for x in _states(device, BF16, 1, 8, 1, 300 + 100 * i, 300 + 100 * i, 128, seed=i)] for i in range(2)]
    run(*held[0])
    graphs, results = [], []
    for h in held:
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            run(*h)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run(*h))
        graphs.append(graph)
    for trial in range(3):
        for i, h in enumerate(held):
            fresh = _states(device, BF16, 1, 8, 1, 300 + 100 * i, 300 + 100 * i, 128, seed=50 + trial)
            for a, c in zip(h, fresh):
                a.copy_(c)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i, h in enumerate(held):
            assert all(torch.equal(a, c) for a, c in zip(results[i], run(*h)))


@pytest.mark.parametrize("role", [1, 2, 3])
def test_backward_bounded_waits_expire(device, role):
    """A stall request makes one role's first wait expire; the kernel records the role's code and
    returns, and the next launch is right."""
    from muzo_clip_b200 import _lib, attention_max_backward
    from muzo_clip_b200.attention import _forward, attention_status, check_attention_status

    q, k, v, dout = _states(device, BF16, 1, 2, 2, 300, 300, 64, seed=30)
    out, lse, _, _ = _forward(q, k, v, 0.125, True, None, None, False, True)
    want = attention_max_backward(dout, q, k, v, out, lse, 0.125, True)
    status = attention_status(device)
    status.zero_()
    status[1] = role
    try:
        attention_max_backward(dout, q, k, v, out, lse, 0.125, True)
        torch.cuda.synchronize()
        assert int(status[0].item()) == role
        with pytest.raises(_lib.MuzoError):
            check_attention_status(device)
    finally:
        status[1] = 0
    got = attention_max_backward(dout, q, k, v, out, lse, 0.125, True)
    check_attention_status(device)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_ranges_beyond_the_sequence(device):
    """key_lo below 0 or behind the keys, key_hi behind them or negative: clamped, or nothing is seen."""
    from muzo_clip_b200 import attention_max

    b, hq, hkv, s, d = 4, 4, 2, 200, 64
    q, k, v, dout = _states(device, BF16, b, hq, hkv, s, s, d, seed=41)
    big = 2 ** 31 - 1

    def run(lo, hi):
        leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
        out, smax, valid = attention_max(*leaves, None, False, *_range(device, b, lo, hi))
        return [out.detach(), smax, *torch.autograd.grad(out, leaves, dout)]

    for a, c in zip(run([-5, 0, big, 3], [big, s, big, -7]), run([0, 0, s, 3], [s, s, s, 3])):
        assert torch.equal(a, c)
    got = run([-5, 0, big, 3], [big, s, big, -7])
    assert not any(bool(g[2:].any()) for g in (got[0], *got[2:]))


def test_one_tensor_as_query_key_and_value(device):
    """The gradients of one leaf in three places add up."""
    from muzo_clip_b200 import attention_max

    x, _, _, dout = _states(device, BF16, 2, 2, 2, 150, 150, 64, seed=42)
    one = x.detach().clone().requires_grad_(True)
    attention_max(one, one, one)[0].backward(dout)
    three = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    attention_max(*three)[0].backward(dout)
    # autograd adds the three in bf16, in an order of its own: two more roundings
    want = sum(t.grad.double() for t in three)
    size = sum(t.grad.double().abs() for t in three)
    assert bool(((one.grad.double() - want).abs() <= 2 * 2.0 ** -8 * size).all())


def test_differentiable_once(device):
    from muzo_clip_b200 import attention_max

    q, k, v, dout = _states(device, BF16, 1, 2, 2, 50, 50, 64, seed=43)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    out, smax, _ = attention_max(*leaves)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out, leaves, dout, create_graph=True)
    with torch.no_grad():
        assert not attention_max(*leaves)[0].requires_grad


@pytest.mark.parametrize("sq,sk", [(270001, 33), (33, 270001)])
def test_offsets_beyond_32_bits(device, sq, sk):
    """More than 2^31 elements of queries, or of keys: the last head's last rows, in a batch of one
    with 64 heads, against the formulas on that head alone."""
    from muzo_clip_b200 import attention_max_backward
    from muzo_clip_b200.attention import _forward

    h, d = 64, 128
    gen = torch.Generator(device=device).manual_seed(3)

    def x(s):
        return torch.randn((1, s, h, d), generator=gen, device=device, dtype=BF16).transpose(1, 2)

    q, k, v, dout = x(sq), x(sk), x(sk), x(sq).transpose(1, 2)
    assert max(q.numel(), k.numel()) > 2 ** 31
    out, lse, _, _ = _forward(q, k, v, 0.05, False, None, None, False, True)
    got = attention_max_backward(dout, q, k, v, out, lse, 0.05, False)
    sub = [t[:, -1:] for t in (q, k, v)] + [dout[:, :, -1:]]
    ref = _exact(*sub, 0.05, torch.ones((1, 1, sq, sk), dtype=torch.bool, device=device), out[:, :, -1:])
    _assert_within([g[:, -1:] for g in got], ref)


def test_first_call_of_a_process_is_captured():
    """A process whose first attention call is being captured: the status words, the kernels' attributes
    and the modules are set up under capture, and the replay computes what an eager call does."""
    import subprocess
    import sys

    from conftest import ROOT

    code = f"""
import sys; sys.path.insert(0, {str(ROOT / "muzo-clip_b200")!r})
import torch
from muzo_clip_b200 import attention_max, clip_grads
g = torch.Generator(device="cuda").manual_seed(0)
x = [torch.randn((1, 4, 200, 64), generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
def run():
    leaves = [t.detach().requires_grad_(True) for t in x]
    out, smax, valid = attention_max(*leaves)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    scaled, norm = clip_grads(list(grads), 0.5)
    return [out.detach(), smax, valid, *grads, *scaled, norm]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
print("the same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stdout + done.stderr


FRESH = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from muzo_clip_b200 import _lib
gen = torch.Generator(device="cuda").manual_seed(5)
q, k, v, dout = (torch.randn((1, 2048, h, 128), generator=gen, device="cuda").bfloat16() for h in (32, 8, 8, 32))
q, k, v = (x.transpose(1, 2) for x in (q, k, v))
native = _lib.native
out, lse, _, _ = native.attention_forward(q, k, v, None, True, None, None, False, True)
def grads(*wanted):
    return native.attention_backward(dout, q, k, v, out, lse, None, True, None, None, wanted)
first = grads(True, True, True)
for wanted in ((True, True, True), (True, False, False), (False, True, True)):
    torch.cuda.empty_cache()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = [grads(*wanted) for _ in range(5)]
    for _ in range(3):
        graph.replay()
    again = grads(*wanted)
    torch.cuda.synchronize()
    split = wanted != (True, True, True)   # without dQ the key tiles may be divided: another order of their sums
    for got in results + [again]:
        for name, a, b in zip(("dq", "dk", "dv"), got, again):
            assert a is None and b is None or torch.equal(a, b), name
        for name, a, b in zip(("dq", "dk", "dv"), got, first):
            assert a is None or (split and name != "dq") or torch.equal(a, b), name
    del graph, results, again
print("same")
"""


@pytest.mark.parametrize("process", range(3))
def test_first_launches_of_fresh_processes(device, process):
    """The first launches of a process, eager and replayed, behind other kernels' data in shared memory and with memory
    mapped and released in between: both kinds of CTA together, and each alone, give the same bits every time."""
    import subprocess
    import sys

    from conftest import ROOT

    done = subprocess.run([sys.executable, "-c", FRESH, str(ROOT / "muzo-clip_b200")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "same", done.stderr[-2000:]


def test_refusals(device):
    from muzo_clip_b200 import attention_max, attention_max_backward

    q, k, v, dout = _states(device, BF16, 2, 4, 2, 20, 20, 64)
    lse = torch.zeros((2, 4, 20), device=device)
    good = torch.zeros(2, dtype=torch.int32, device=device)
    for bad, kind in (((q.float(), k.float(), v.float()), TypeError), ((q, k.half(), v), TypeError),
                      ((q[0], k, v), ValueError), ((q, k[:1], v[:1]), ValueError), ((q, k, v[:, :, :5]), ValueError),
                      ((q[:, :3], k, v), ValueError), ((q.cpu(), k.cpu(), v.cpu()), ValueError),
                      ((q[..., :60], k[..., :60], v[..., :60]), ValueError)):
        with pytest.raises(kind):
            attention_max(*bad)
    for scaling in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            attention_max(q, k, v, scaling)
    for ranges in (good.long(), good[:1], good.cpu()):
        with pytest.raises(ValueError):
            attention_max(q, k, v, key_lo=ranges)
    with pytest.raises(ValueError):
        attention_max_backward(dout, q, k, v, dout, lse[:, :, :19])
    with pytest.raises(ValueError):
        attention_max_backward(dout.transpose(1, 2), q, k, v, dout, lse)
    with pytest.raises(ValueError):
        attention_max_backward(dout.half(), q, k, v, dout, lse)

"""Clipping gradients that do not fill their memory: results that share elements are refused as contiguous
ones are, results that only interleave are taken, and nothing beside them is written."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _base(device, seed=0, shape=(60, 90), dtype=torch.float32):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(device)


SHARED = {   # views of x (and of another tensor, y) as (gradients, outputs)
    "the same one twice": lambda x, y: ([x[:, ::2]] * 2, [x[:, ::2]] * 2),
    "two results in one place": lambda x, y: ([x[:, ::2], x[:, 1::2]], [y[:, ::2], y[:, ::2]]),
    "columns that overlap": lambda x, y: ([x[:, :40], x[:, 30:70]], [x[:, :40], x[:, 30:70]]),
    "a result over another's gradient": lambda x, y: ([x[:, :40], x[:, 50:70]], [y[:, :40], x[:, 20:40]]),
    "a strided one inside a contiguous one": lambda x, y: ([x, x[:, ::3]], [x, x[:, ::3]]),
    "shifted over itself": lambda x, y: ([x[:, :40]], [x[:, 1:41]]),
    "transposed over itself": lambda x, y: ([x[:40, :40]], [x[:40, :40].t()]),
    "an expanded result": lambda x, y: ([x[:, :4]], [y[:, :1].expand(60, 4)]),
}


@pytest.mark.parametrize("name", SHARED)
def test_shared_elements_are_refused(device, name):
    from muzo_clip_b200 import clip_grads

    x, y = _base(device), _base(device, 1)
    grads, outs = SHARED[name](x, y)
    kept = x.clone(), y.clone()
    with pytest.raises(ValueError):
        clip_grads(grads, 0.5, out=outs)
    assert torch.equal(x, kept[0]) and torch.equal(y, kept[1])


def test_other_pitches_are_told_apart(device):
    """Two views of one buffer with rows of 90 and of 100 elements: refused exactly where they meet."""
    from muzo_clip_b200 import clip_grads

    for offset in range(0, 60):
        buffer = torch.ones(2000, device=device)
        a = buffer.as_strided((3, 4), (90, 7), 0)
        c = buffer.as_strided((3, 4), (100, 11), offset)
        mark = torch.zeros(2000, device=device)
        mark.as_strided((3, 4), (90, 7), 0).add_(1.0)
        mark.as_strided((3, 4), (100, 11), offset).add_(1.0)
        if bool((mark > 1.0).any()):
            with pytest.raises(ValueError):
                clip_grads([a, c], 0.5, out=[a, c])
            assert bool((buffer == 1.0).all())
        else:
            clip_grads([a, c], 0.5, out=[a, c])
            assert bool((buffer[mark == 0.0] == 1.0).all()) and bool((buffer[mark == 1.0] < 0.2).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_interleaved_views_are_taken(device, dtype):
    """Columns of one matrix, its even and odd elements, a matrix beside the transpose of another part of it."""
    from muzo_clip_b200 import clip_grads

    cuts = {"columns": lambda x: [x[:, :31], x[:, 31:32], x[:, 32:]], "even and odd": lambda x: [x[:, ::2], x[:, 1::2]],
            "quarters": lambda x: [x[::2, ::2], x[1::2, ::2], x[::2, 1::2], x[1::2, 1::2]],
            "transposed": lambda x: [x[:, :40].t(), x[:, 40:]]}
    for name, cut in cuts.items():
        x = _base(device, 3, dtype=dtype)
        kept = x.clone()
        want, norm = clip_grads([g.clone(memory_format=torch.contiguous_format) for g in cut(x)], 2.0)
        got, same = clip_grads(cut(x), 2.0, out=cut(x))
        assert torch.allclose(same, norm, rtol=1e-6, atol=0.0), name
        assert all(torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=0.0) for a, b in zip(got, want)), name
        assert not torch.equal(x, kept)
        fresh = torch.zeros_like(x)
        clip_grads(cut(kept), 2.0, out=cut(fresh))
        assert torch.equal(fresh, x), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_guards_between_views_stay(device, dtype):
    """Views at odd offsets of one bucket, with elements between them that belong to nobody."""
    from muzo_clip_b200 import clip_grads, grad_norm

    bucket = _base(device, 4, (100003,), dtype)
    spans = [(1, 2), (3, 39), (45, 5001), (5004, 5005), (5006, 60001), (60010, 99990)]
    views = [bucket[a:z] for a, z in spans]
    mine = torch.zeros(bucket.shape, dtype=torch.bool, device=device)
    for a, z in spans:
        mine[a:z] = True
    before = bucket.clone()
    want, norm = clip_grads([x.clone() for x in views], 0.25 * float(grad_norm(views)))
    _, same = clip_grads(views, 0.25 * float(grad_norm(views)), out=views)
    # the same squares in groups of eight that begin elsewhere: each sum in fp32, 8 half steps, halved by the root
    assert abs(float(same) - float(norm)) <= 2 * 5 * 2.0 ** -24 * float(norm)
    for a, c in zip(views, want):
        assert torch.allclose(a.float(), c.float(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -24)
    assert torch.equal(bucket[~mine], before[~mine]) and not torch.equal(bucket[mine], before[mine])

"""Host side of the gradient operators, without a GPU: what the entry points refuse before any
launch, workspace sizes, and the Python functions' checks on CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

_P = 256          # a device address nothing dereferences: every call here ends in a host check
_S = (ctypes.c_int64 * 24)(*([64] * 24))
_ODD = (ctypes.c_int64 * 24)(*([64] * 23 + [63]))


def _bwd(L, q=_P, k=_P, v=_P, out=_P, dout=_P, lse=_P, dq=_P, dk=_P, dv=_P, dtype=1, b=1, hq=4, hkv=2, sq=8, sk=8, d=64,
         strides=_S, scale=0.1, ws=_P, size=1 << 40, status=_P):
    return L.muzo_attention_backward(q, k, v, out, dout, lse, dq, dk, dv, dtype, b, hq, hkv, sq, sk, d, strides, 1, scale,
                                     None, None, ws, size, status, None)


@pytest.mark.parametrize("change, expected", [
    ({"q": None}, 1), ({"lse": None}, 1), ({"dout": None}, 1), ({"ws": None}, 1), ({"strides": None}, 1),
    ({"status": None}, 1), ({"b": -1}, 1), ({"hq": 3}, 1), ({"hkv": 0}, 1), ({"scale": 0.0}, 1), ({"scale": -1.0}, 1),
    ({"scale": float("nan")}, 1), ({"scale": float("inf")}, 1),
    ({"dtype": 0}, 2), ({"dtype": 9}, 2),
    ({"strides": _ODD}, 3), ({"q": _P + 2}, 3), ({"dv": _P + 8}, 3), ({"ws": _P + 4}, 3),
    ({"size": 16}, 5),
    ({"d": 60}, 6), ({"d": 136}, 6), ({"d": 0}, 6), ({"sq": 1 << 31}, 6),
    ({"b": 0}, 0), ({"sq": 0, "sk": 0}, 0),
    ({"dq": None, "dk": None, "dv": None, "sk": 0}, 0),          # nothing to write
])
def test_backward_refuses_before_any_launch(change, expected):
    from muzo_clip_b200 import _lib

    assert _bwd(_lib.lib, **change) == expected


def _fwd(L, q=_P, k=_P, lse=_P, d=64, scale=0.1, smax=None, valid=None, stride=64):
    return L.muzo_attention_max_lse(q, k, _P, _P, lse, 1, 1, 4, 2, 8, 8, d, *([stride] * 12), 1, scale, None, None, smax,
                                    valid, _P, None)


@pytest.mark.parametrize("change, expected", [
    ({"q": None}, 1), ({"k": None}, 1), ({"scale": 0.0}, 1), ({"scale": float("nan")}, 1), ({"smax": _P}, 1),
    ({"d": 12}, 6), ({"d": 256}, 6), ({"stride": 4}, 3), ({"q": _P + 8}, 3),
])
def test_forward_refuses_before_any_launch(change, expected):
    from muzo_clip_b200 import _lib

    assert _fwd(_lib.lib, **change) == expected


def test_backward_workspace_sizes():
    from muzo_clip_b200 import _lib

    size = _lib.lib.muzo_attention_backward_workspace
    assert size(1, 1, 4, 3, 8, 8, 64, 1) < 0 and size(0, 1, 4, 2, 8, 8, 64, 1) < 0 and size(1, 1, 4, 2, 8, 8, 72 + 64, 0) < 0
    # two fp32 values for each query row, padded to tiles of 128
    for b, hq, sq in ((1, 4, 8), (3, 32, 2048), (2, 6, 129)):
        for causal in (0, 1):
            assert size(1, b, hq, 2, sq, sq, 128, causal) >= 8 * b * hq * (-(-sq // 128) * 128)
    # one key head and many queries: sums of dK and dV for each part of the work
    assert size(1, 1, 8, 1, 2048, 2048, 128, 1) >= 8 * 8 * 2048 + 2 * 2048 * 2 * 128 * 4
    # beyond 32 bits
    assert size(1, 64, 128, 128, 1 << 20, 1 << 20, 128, 1) > 1 << 32


def test_python_refuses_cpu_tensors():
    from muzo_clip_b200 import attention_max, attention_max_backward

    q = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention_max(q, q, q)
    with pytest.raises(ValueError):
        attention_max_backward(q.transpose(1, 2), q, q, q, q.transpose(1, 2), torch.zeros((1, 2, 4)))


def test_readable_layouts():
    """Which layouts are read in place: D contiguous, 16-byte aligned, strides of 8 elements; a
    dimension of size 1 may have any stride."""
    from muzo_clip_b200.attention import _readable

    base = torch.zeros((2, 5, 3, 64), dtype=torch.bfloat16)
    t = base.transpose(1, 2)
    same, strides = _readable(t)
    assert same.data_ptr() == base.data_ptr() and strides == (5 * 3 * 64, 64, 3 * 64)
    one = base[:1].as_strided((1, 3, 5, 64), (7, 64, 192, 1))
    same, strides = _readable(one)
    assert same.data_ptr() == base.data_ptr() and strides[0] % 8 == 0 and strides[0] > 0
    for t in (base[:1].expand(4, -1, -1, -1), torch.zeros((2, 3, 5, 68), dtype=torch.bfloat16)[..., :64],
              torch.zeros((2, 3, 64, 5), dtype=torch.bfloat16).transpose(2, 3)):
        copy, strides = _readable(t)
        assert copy.is_contiguous() and torch.equal(copy, t) and not any(s % 8 or s == 0 for s in strides)


def _u64(*v):
    return (ctypes.c_uint64 * len(v))(*v)


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _i32(*v):
    return (ctypes.c_int32 * len(v))(*v)


@pytest.mark.parametrize("change, expected", [
    ({"src": None}, 1), ({"num": None}, 1), ({"kind": None}, 1), ({"norm": None}, 1), ({"ws": None}, 1), ({"n": -1}, 1),
    ({"num": _i64(-1)}, 1), ({"src": _u64(0)}, 1), ({"kind": _i32(7)}, 2), ({"src": _u64(257)}, 3),
    ({"src": _u64(258), "kind": _i32(0)}, 3), ({"ws": _P + 4}, 3), ({"size": 64}, 5), ({"num": _i64(1 << 41)}, 6),
])
def test_norm_refuses_before_any_launch(change, expected):
    from muzo_clip_b200 import _lib

    a = {"src": _u64(256), "num": _i64(64), "kind": _i32(1), "n": 1, "norm": _P, "ws": _P, "size": 1 << 30, **change}
    assert _lib.lib.muzo_grad_norm(a["src"], a["num"], a["kind"], a["n"], 0, a["norm"], a["ws"], a["size"], None) == expected


@pytest.mark.parametrize("change, expected", [
    ({"dst": None}, 1), ({"to": None}, 1), ({"to": _i32(2, 1)}, 2), ({"max": -1.0}, 1), ({"max": float("nan")}, 1),
    ({"dst": _u64(1024, 1024)}, 1),                                  # two results in one place
    ({"dst": _u64(256 + 64, 4096)}, 1),                              # a result over another element of its own source
    ({"dst": _u64(256, 300)}, 1),                                    # a result over another tensor's source
    ({"dst": _u64(0, 512)}, 1),
    ({"to": _i32(0, 1)}, 1),                                         # in place, but wider
    ({"size": 64}, 5),                                               # separate results pass the overlap check
    ({"dst": _u64(2048, 4096), "size": 64}, 5),
])
def test_clip_refuses_before_any_launch(change, expected):
    from muzo_clip_b200 import _lib

    a = {"src": _u64(256, 512), "dst": _u64(256, 512), "num": _i64(64, 64), "kind": _i32(1, 1), "to": _i32(1, 1), "max": 1.0,
         "size": 1 << 30, **change}
    assert _lib.lib.muzo_grad_clip(a["src"], a["dst"], a["num"], a["kind"], a["to"], 2, 0, a["max"], _P, _P, a["size"],
                                   None) == expected


def test_flat_layouts():
    from muzo_clip_b200.grad_clip import _flat

    t = torch.zeros(4, 6, 8)
    assert _flat(t) and _flat(t.transpose(0, 2)) and _flat(t[1:3]) and _flat(t[:, :1, :1][:1]) and _flat(torch.zeros(0, 3))
    assert not _flat(t[:, 1:3]) and not _flat(t[..., ::2]) and not _flat(torch.zeros(1).expand(5))


def test_gradient_functions_refuse_cpu_tensors():
    from muzo_clip_b200 import clip_grads, grad_norm

    with pytest.raises(ValueError):
        grad_norm([torch.zeros(4)])
    with pytest.raises(ValueError):
        clip_grads([torch.zeros(4)], 1.0)
    assert float(grad_norm([])) == 0.0

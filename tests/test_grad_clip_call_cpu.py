"""clip_grad_norm_ takes torch's arguments, by name and by place."""

from __future__ import annotations

import inspect

import pytest
import torch

from muzo_clip_b200 import clip_grad_norm_


def test_arguments_are_torchs():
    mine, theirs = (inspect.signature(f).parameters for f in (clip_grad_norm_, torch.nn.utils.clip_grad_norm_))
    assert list(mine) == list(theirs)
    assert [p.default for p in mine.values()] == [p.default for p in theirs.values()]


@pytest.mark.parametrize("foreach", [None, True, False])
def test_foreach_is_taken(foreach):
    parameter = torch.nn.Parameter(torch.zeros(3))      # no gradient: the norm of nothing
    assert float(clip_grad_norm_([parameter], 1.0, 2.0, False, foreach)) == 0.0
    assert float(clip_grad_norm_([parameter], max_norm=1.0, foreach=foreach)) == 0.0

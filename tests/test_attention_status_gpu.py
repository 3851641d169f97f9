"""The attention kernels' status words: created by a device's first launch, outside any graph, and not by a
check of them."""

from __future__ import annotations

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


UNUSED = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import muzo_clip_b200 as m
dev = torch.device("cuda", 0)
torch.zeros(1, device=dev)
before = torch.cuda.memory_stats(dev)["allocation.all.allocated"]
m.check_attention_status(dev)
m.check_attention_status(torch.device("cuda"))
m.check_attention_status(torch.device("cpu"))
assert torch.cuda.memory_stats(dev)["allocation.all.allocated"] == before
print("nothing")
"""


def test_no_attention_launch_nothing_to_check(device):
    """Without an attention launch on the device the check neither allocates nor waits."""
    from conftest import ROOT

    done = subprocess.run([sys.executable, "-c", UNUSED, str(ROOT / "muzo-clip_b200")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "nothing", done.stdout + done.stderr[-2000:]

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


WORDS = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import muzo_clip_b200 as m
from muzo_clip_b200.attention import attention_status
dev = torch.device("cuda", 0)
gen = torch.Generator(device=dev).manual_seed(0)
x = [torch.randn((1, 4, 200, 64), generator=gen, device=dev, dtype=torch.bfloat16) for _ in range(3)]
torch.cuda.synchronize()
# the capture runs on a stream of torch's pool of 32, and the pool's next one is that stream again
first = torch.cuda.Stream()
others = [torch.cuda.Stream() for _ in range(31)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=first):
    out, smax, valid = m.attention_max(*x)
words = attention_status(dev)
assert words.tolist() == [0, 0], words.tolist()      # clear before the first replay
words[0] = 2                                           # a launch before has reported an expired wait
graph.replay()
torch.cuda.synchronize()
assert words.tolist() == [2, 0], words.tolist()      # and a replay leaves that standing
words.zero_()
again = m.attention_max(*x)
torch.cuda.synchronize()
assert torch.equal(out, again[0]) and torch.equal(smax, again[1])
print("kept")
"""


def test_status_words_of_a_captured_first_call(device):
    from conftest import ROOT

    done = subprocess.run([sys.executable, "-c", WORDS, str(ROOT / "muzo-clip_b200")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "kept", done.stdout + done.stderr[-2000:]


INFERENCE = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import muzo_clip_b200 as m
from muzo_clip_b200 import _lib
from muzo_clip_b200.attention import attention_status
dev = torch.device("cuda", 0)
x = torch.zeros((1, 2, 8, 64), dtype=torch.bfloat16, device=dev)
with torch.inference_mode():
    m.attention_max(x, x, x)
m.check_attention_status(dev)
attention_status(dev)[0] = 3
try:
    m.check_attention_status(dev)
except _lib.MuzoError:
    m.check_attention_status(dev)
    print("cleared")
"""


def test_status_words_of_a_first_call_in_inference_mode(device):
    from conftest import ROOT

    done = subprocess.run([sys.executable, "-c", INFERENCE, str(ROOT / "muzo-clip_b200")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "cleared", done.stdout + done.stderr[-2000:]

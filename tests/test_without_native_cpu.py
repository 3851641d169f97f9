"""The optimizer, QK-Clip's own kernels and Newton-Schulz reach the library through its C ABI: where the
compiled module over torch tensors does not load (another torch version), the package still imports and works,
and only the operators behind that module refuse, with the reason."""

from __future__ import annotations

import subprocess
import sys

from conftest import ROOT

CODE = """
import sys
sys.path.insert(0, sys.argv[1])

class Broken:
    def find_spec(self, name, path=None, target=None):
        if name == "muzo_clip_b200._native":
            raise ImportError("undefined symbol: of another torch version")
        return None

sys.meta_path.insert(0, Broken())
import torch
import muzo_clip_b200 as m
from muzo_clip_b200 import _lib, _qk

assert m.prng.hash64_seed(1, "a.weight", (2, 3), 0) == _lib.hash64_seed_native(1, "a.weight", (2, 3), 0)
model = torch.nn.Sequential()
model.q_proj = torch.nn.Linear(8, 8, bias=False)
opt = m.MuZOClipOptimizer(model, seed=3)
assert len(m.select_muzo_parameters(model)) == 1
m.check_attention_status(torch.device("cuda", 0))        # nothing of it can have run
x = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16)
for call in (lambda: m.attention_max(x, x, x), lambda: m.grad_norm([torch.ones(3)]), lambda: m.clip_grads([torch.ones(3)], 1.0),
             lambda: m.attention_max_backward(x, x, x, x, x, x)):
    try:
        call()
    except ImportError as e:
        assert "another torch version" in str(e) and "build.py" in str(e), e
    else:
        raise AssertionError("answered without its module")
print("works")
"""


def test_the_package_without_its_torch_module():
    done = subprocess.run([sys.executable, "-c", CODE, str(ROOT / "muzo-clip_b200")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "works", done.stdout + done.stderr[-3000:]

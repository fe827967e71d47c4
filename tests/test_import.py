"""The package's host-side parts (routing sort, checkpoints, synthetic data) need no CUDA build of torch."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# torch without what only its CUDA builds bind
CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import vpipe_b200
from vpipe_b200 import checkpoint, moe, ops, synth
q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
try:
    ops.qk_norm_rope(q, q)
except ValueError as e:
    assert "no CPU path" in str(e), e
else:
    raise AssertionError("rows on the CPU were taken")
print("imported")
"""


def test_the_package_imports_with_a_torch_that_has_no_cuda():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr[-2000:]

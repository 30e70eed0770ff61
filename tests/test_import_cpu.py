"""The package on a torch that was built without CUDA.  No GPU is touched."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys
sys.path.insert(0, {root!r})
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:      # what such a torch lacks
    delattr(torch._C, name)
import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import dense, ep, layout, moe, synth
x = torch.zeros((2, 64))
weight = torch.zeros((8, 64), dtype=torch.int8), torch.ones(8)
for call in (lambda: okc.quantize_rows(x), lambda: okc.int8_linear(x, weight), lambda: okc.int8_linear(weight, weight), lambda: okc.int8_gated(x, weight),
             lambda: okc.block_norm(x, x), lambda: okc.block_norm(x[:0], pre_gain=torch.ones(64)), lambda: okc.int8_rows(*weight)):
    try:
        call()
    except ValueError as e:
        assert "CUDA" in str(e), e
    else:
        raise SystemExit("not refused")
print("fine")
"""


def test_the_package_imports_on_a_torch_without_cuda():
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(root=ROOT)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-2000:]

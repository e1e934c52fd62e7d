"""The package imports, and its calls refuse tensors, whatever torch offers to ask for the current device with."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys, torch
sys.path.insert(0, %r)
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
def current_device():
    raise %s("no device here")
torch.cuda.current_device = current_device
import __graft_entry__ as ge
pkg = ge.import_package()
x = torch.zeros(2, 64)
try:
    pkg.add_rmsnorm(x, x, x.bfloat16(), 2, 64, o=x)
except ValueError as e:
    assert "expected a tensor on the current device" in str(e), e
    print("refused")
"""


@pytest.mark.parametrize("error", ["RuntimeError", "AssertionError"])
def test_without_the_private_names(error):
    r = subprocess.run([sys.executable, "-c", PROGRAM % (ROOT, error)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "refused", r.stderr

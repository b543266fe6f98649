"""When ftb._pycall is loaded: at the first call that goes through it, not with the package."""
import os
import subprocess
import sys

import pytest

from tests.conftest import PKG, ROOT

NEEDED = """
import sys
import torch
import ftb
from ftb import synth, banks, experts, fused_nvfp4
synth.make_bank(2, 128, 128)
assert "ftb._pycall" not in sys.modules
assert "_pycall" not in open("/proc/self/maps").read()
x = torch.zeros(4, 64, dtype=torch.bfloat16)
try:
    ftb.rms_norm(x, x[0])
except ValueError as e:
    assert "CUDA" in str(e)
assert "ftb._pycall" in sys.modules
assert set(vars(ftb._runtime._pycall)) >= {"key", "call", "empty"}
"""

MISSING = """
import sys
sys.modules["ftb._pycall"] = None  # (an import of it fails)
import torch
import ftb
x = torch.zeros(4, 64, dtype=torch.bfloat16)
for _ in range(2):
    try:
        ftb.rms_norm(x, x[0])
    except ftb._lib.FtbLibraryError as e:
        assert "make -C" in str(e)
    else:
        assert False
"""


@pytest.mark.parametrize("program", [NEEDED, MISSING], ids=["needed", "missing"])
def test_loading(program):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, PKG]))
    out = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, env=env,
                         timeout=300)
    assert out.returncode == 0, out.stderr

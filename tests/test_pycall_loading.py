"""When ftb._pycall is loaded: at the first call that goes through it, not with the package. When it
is built: again for another torch."""
import os
import shutil
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

OTHER = """
import torch
import ftb
x = torch.zeros(4, 64, dtype=torch.bfloat16)
torch.__version__ = "2.0.1+other"
try:
    ftb.rms_norm(x, x[0])
except ftb._lib.FtbLibraryError as e:
    assert "2.0.1+other" in str(e) and "make -C" in str(e)
else:
    assert False
"""


@pytest.mark.parametrize("program", [NEEDED, MISSING, OTHER], ids=["needed", "missing", "other"])
def test_loading(program):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, PKG]))
    out = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, env=env,
                         timeout=300)
    assert out.returncode == 0, out.stderr


@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_another_torch_builds_it_again(tmp_path):
    """The Makefile's rule, with compilers that only touch their output and a python that names a
    torch version."""
    csrc = tmp_path / "package" / "csrc"
    shutil.copytree(os.path.join(PKG, "csrc"), csrc)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    (tmp_path / "package" / "ftb").mkdir()

    def tool(name, text):
        path = tmp_path / name
        path.write_text("#!/bin/sh\n" + text)
        path.chmod(0o755)
        return str(path)

    touch = tool("touch_output", 'while [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n')
    log = tmp_path / "built"
    cxx = tool("cxx", f'echo built >> {log}\nexec {touch} "$@"\n')

    def make(version):
        python = tool("python", f"echo {version}\n")
        out = subprocess.run(["make", "-C", str(csrc), f"NVCC={touch}", f"CXX={cxx}",
                              f"PYTHON={python}", f"BUILD={tmp_path}/build"],
                             capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr
        return len(log.read_text().splitlines())

    assert [make(v) for v in ("2.11.0", "2.11.0", "2.12.0", "2.12.0", "2.11.0")] == [1, 1, 2, 2, 3]

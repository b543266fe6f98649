"""examples/decoder_layers.py on prompts of any length: its rotary table goes by them."""
import os
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 8300])
def test_example_at_other_lengths(tokens):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "decoder_layers.py"),
                          "--tokens", str(tokens), "--steps", "2"], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0, out.stderr
    assert "step 2: 4 new tokens over" in out.stdout

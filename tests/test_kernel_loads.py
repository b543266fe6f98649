"""How the attention kernels load: what can be seen of it in their sources.

A kernel may be resident while the one before it on the stream still writes (programmatic launches): the
append's codes, scales and q, the plan's pieces. The wait for that kernel makes its writes visible to
ordinary loads. Non-coherent ones (ld.global.nc, __ldg) are for memory that nobody writes while the kernel
lives, so the attention has none of them."""
import glob
import os
import re

import pytest

from tests.conftest import PKG

SOURCES = sorted(glob.glob(os.path.join(PKG, "csrc", "attn*.cu*")))


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_the_attention_loads_coherently(path):
    with open(path) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"ld\.global(?:\.\w+)*\.nc\b[^\"]*|__ldg\s*\([^;]*", text)


def test_the_sources_are_there():
    assert {"attn.cu", "attn.cuh", "attn_chunk.cu", "attn_stream.cu"} <= set(map(os.path.basename, SOURCES))

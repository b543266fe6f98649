"""Waits that end: what can be seen of it in the kernels' sources.

A named barrier has no limit, so no warp of its group may leave before it. The attention kernels'
waits on copies give up after a limit; where warps share named barriers, one that gave up has to
pass them all the same, so their function has no return of its own."""
import glob
import os
import re

import pytest

from tests.conftest import PKG

SOURCES = sorted(glob.glob(os.path.join(PKG, "csrc", "attn_*.cu")))


def functions(text):
    """(name, body) of the device functions at namespace level, without comments."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"^(?:__device__|__global__|template)[^;{}]*?(\w+)\s*\([^;{}]*\)\s*\{", text,
                         re.M):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at - 1]


def without_lambdas(body):
    while True:
        m = re.search(r"\[[&=\w, ]*\]\s*(?:\([^()]*\))?\s*\{", body)
        if not m:
            return body
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(body[at], 0)
            at += 1
        body = body[:m.start()] + body[at:]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_no_warp_leaves_before_a_named_barrier(path):
    with open(path) as f:
        found = dict(functions(f.read()))
    assert found, path
    for name, body in found.items():
        if "named_bar(" in body:
            assert not re.search(r"\breturn\b", without_lambdas(body)), name


def test_the_streaming_consumers_share_named_barriers():
    """(the test above looks at the function that has them)"""
    with open(os.path.join(PKG, "csrc", "attn_stream.cu")) as f:
        body = dict(functions(f.read()))["stream_consumer"]
    assert body.count("named_bar(") > 4
    assert re.search(r"l\[0\] = l\[1\] = NAN", body)  # rows without all their keys are not numbers

"""Calls of ftb.paged_attention from threads that have made no call of CUDA's runtime before: the tensor maps
need the device's context current to the thread."""
import threading

import pytest
import torch

import ftb
from tests.attn_cases import AttnCase, build, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [[(1, 700), (1, 90)], [(500, 1200)]])
def test_a_threads_first_call(pairs):
    c = AttnCase(pairs, q_heads=16, page=32)
    ref, bound, _ = reference(c, *build(c))
    out = torch.empty_like(c.t["q"])
    ftb.paged_attention(**c.t, out=out)  # (the workspace is there)
    seen = []

    def work():
        try:
            ftb.paged_attention(**c.t, out=out)
            seen.append(None)
        except Exception as e:  # noqa: BLE001
            seen.append(e)

    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert ((out.double().cpu() - ref).abs() <= bound).all()
    assert seen == [None] * 3

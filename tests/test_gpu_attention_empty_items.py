"""Items without keys in the tensor-core kernel of ftb.paged_attention: sequences that have none, and new
tokens before every key. They end the list of a call's items, so a block may meet many in a row behind one
with keys, whose last product is issued with the step that follows it: without one it is issued when an
item without keys is met. (Before that, four in a row stopped the block until its waits gave up.)"""
import pytest
import torch

import ftb
from tests.attn_cases import AttnCase, build, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("empty", [1, 40, 400])
def test_many_items_without_keys(empty, head):
    c = AttnCase([(300, 1500), (280, 280)] + [(1, 0)] * empty + [(500, 200)], q_heads=24, kv_heads=8,
                 head=head, page=32)
    q, keys = build(c)
    ref, bound, ref_lse = reference(c, q, keys)
    for _ in range(20):
        out, lse = ftb.paged_attention(**c.t, return_lse=True, check_status=True)
        assert ((out.double().cpu() - ref).abs() <= bound).all()
        assert torch.equal(torch.isinf(lse).cpu(), torch.isinf(ref_lse))

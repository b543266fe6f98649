"""ftb.DecoderLayer on steps without tokens, as a rank of a group may have them."""
import pytest
import torch

import ftb
from tests.test_gpu_decoder import build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages,past,new", [([], [], []), ([[0]], [0], [0]), ([[0, 1], [2]], [33, 4], [0, 0])])
@pytest.mark.parametrize("residual", [torch.bfloat16, torch.float32])
def test_a_step_without_tokens(pages, past, new, residual):
    layer, cache = build(), ftb.PagedKvCache(3, 32, 2, 64)
    step = ftb.AttnStep.build(pages, past, new, 32)
    x = torch.empty(0, 512, dtype=residual, device="cuda")
    for next_norm in (layer.input_norm, None):
        r, h = layer(x, None, step, cache, next_norm)
        assert r.shape == (0, 512) and r.dtype == residual
        assert h is None if next_norm is None else h.shape == (0, 512)
    assert (cache.k == 0).all() and (cache.v == 0).all()

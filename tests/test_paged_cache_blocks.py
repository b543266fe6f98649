"""The tokens per scale that an 8-bit ftb.PagedKvCache has by default."""
import pytest
import torch

import ftb

FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("page,size", [(16, 16), (32, 32), (48, 16), (64, 64), (80, 16), (96, 32), (128, 128),
                                       (192, 64), (256, 128), (384, 128), (1024, 128)])
def test_the_largest_that_divides_the_page(page, size):
    c = ftb.PagedKvCache(3, page, 2, 32, dtype=FP8, device="cpu")
    assert c.k_scale.shape == c.v_scale.shape == (3, page // size, 2)


@pytest.mark.parametrize("page", [1, 8, 24, 40, 100])
def test_pages_that_none_divides(page):
    with pytest.raises(ValueError):
        ftb.PagedKvCache(3, page, 2, 32, dtype=FP8, device="cpu")

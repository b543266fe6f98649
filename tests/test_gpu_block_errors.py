"""What the block operators raise: the kinds of error a caller can tell apart."""
import pytest
import torch

import ftb

pytestmark = pytest.mark.gpu


def test_an_output_that_does_not_fit_is_an_out_of_memory_error():
    """The input is one row, seen 2^31 - 1 times; the output would be 17 TB."""
    x = torch.zeros(1, 4096, dtype=torch.bfloat16, device="cuda").expand(2 ** 31 - 1, 4096)
    w = torch.ones(4096, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(torch.cuda.OutOfMemoryError):
        ftb.rms_norm(x, w)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        ftb.block_norm(x, x, pre_weight=w)


def test_block_norm_without_a_block_output():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="rms_norm"):
        ftb.block_norm(x, None, pre_weight=x[0])

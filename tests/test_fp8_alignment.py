"""Pointers of the 8-bit cache's calls that their elements' loads could not use are refused before any launch
(no GPU needed)."""
import ctypes

import pytest

from ftb import _lib
from tests.test_fp8_refusals import attention, copy
from tests.test_fp8_shared_scales import rope

ALIGN = _lib.FTB_ERR_ALIGN


@pytest.mark.parametrize("kw", [dict(k_scale=18), dict(v_scale=33), dict(k_scale=17)])
def test_scales(kw):
    assert rope(**kw) == ALIGN
    assert attention(max_q=1, **kw) == ALIGN


@pytest.mark.parametrize("kw", [dict(src=18), dict(dst=17)])
def test_ids_of_32_bits(kw):
    assert copy(n=3, **kw) == ALIGN


@pytest.mark.parametrize("kw", [dict(src=20), dict(dst=36)])
def test_ids_of_64_bits(kw):
    s = _lib.PagesArgsStruct(n=3, num_pages=4, n_caches=1, src=kw.get("src", 16), dst=kw.get("dst", 16),
                             id64=1)
    s.caches[0], s.page_strides[0], s.page_bytes[0] = 256, 64, 64
    assert _lib.load().ftb_copy_pages(ctypes.byref(s), None) == ALIGN

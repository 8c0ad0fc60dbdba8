"""The 8-bit block cache without a GPU: refusals that the other tests of it do not reach."""
import math

import pytest

from test_blocks import _view


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_scales_that_are_no_number_are_refused(pkg, bad):
    lib, view = pkg._lib.load(), _view(pkg)
    assert lib.sphkv_blocks_decode(view, 4096, 1, 512, 128, None, 4096, 1, None, 4096, 1 << 30, 4, bad, None) == -1
    assert b"sm_scale" in lib.sphkv_last_error()
    assert lib.sphkv_blocks_attend(view, 4096, 1, 512, 128, None, 2, None, 4096, 1, 4096, 1 << 30, 4, bad, None) == -1
    assert b"sm_scale" in lib.sphkv_last_error()

"""Refusals of the cache attention's scalar arguments at the C entry, before any launch."""
import ctypes
import math

import pytest

from instinctflash_b200 import _lib


@pytest.mark.parametrize("scale,cap,status", [
    (1.0, math.inf, -1), (1.0, 1e-39, -1), (1.0, -0.5, -1), (1.0, math.nan, -1), (math.inf, 0.0, -1), (-math.inf, 0.0, -1), (math.nan, 0.0, -1),
    (1.0, 0.0, 0), (-3.0, 1.2e-38, 0), (1e38, 3e38, 0)])
def test_scalars_that_are_refused(scale, cap, status):
    p = ctypes.c_void_p(4096)   # never dereferenced
    got = _lib.lib().iflb200_cache_attention(p, 1, 64, 64, 64, p, p, p, p, 4, 16, 80, p, 2, 2, p, None, None, None, 1, 1, 2, 1, scale, cap, 1,
                                             p, 64, 64, 64, None, 0, None)
    assert got == -2            # head_dim is looked at first
    got = _lib.lib().iflb200_cache_attention(p, 1, 64, 64, 64, p, p, p, p, 4, 16, 64, p, 2, 2, p, None, None, None, 0, 1, 2, 1, scale, cap, 1,
                                             p, 64, 64, 64, None, 0, None)
    assert got == status        # (no sequence: nothing to launch)

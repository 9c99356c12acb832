"""cache_append, what needs no GPU: calls without rows."""
import ctypes

import pytest

from test_host_ragged import P, cache_desc
from test_host_window import rope


@pytest.mark.parametrize("axes", [1, 3, 8])
def test_no_rows_need_no_positions(pkg, axes):
    """(An empty tensor's address is null.)"""
    append = lambda **over: pkg._lib.load_library().cosmos_attn_cache_append(ctypes.byref(cache_desc(pkg, cu=P, **over)), ctypes.byref(rope(pkg, axes=axes, positions=None)), None)
    assert append(rows=0, k_rows=None, v_rows=None, q=None, o=None) == pkg._lib.ST_OK
    if axes > 1:
        assert append(rows=4) == pkg._lib.ST_BAD_ARG

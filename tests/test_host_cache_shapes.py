"""One token over a window of the cache: which calls take one kernel, and no workspace, goes by the time of a workgroup's tiles (head dim, codes, rows)."""
import ctypes

import pytest

from test_host_ragged import P, cache_desc

CASES = [(64, "CACHE_SAME", 4, 6), (64, "CACHE_E4M3", 4, 5), (64, "CACHE_INT8", 4, 5), (128, "CACHE_SAME", 4, 5), (128, "CACHE_E4M3", 4, 4), (128, "CACHE_INT8", 4, 4),
         (64, "CACHE_SAME", 32, 5), (64, "CACHE_INT8", 32, 4), (128, "CACHE_SAME", 32, 4), (128, "CACHE_INT8", 32, 3)]


@pytest.mark.parametrize("D, kind, group, most", CASES)
def test_windows_of_few_tiles_are_taken_whole(pkg, D, kind, group, most):
    lib, page, heads = pkg._lib.load_library(), 32, 2
    whole = []
    for tiles in range(2, 9):
        strides = (heads * page * D, page * D, D)
        d = cache_desc(pkg, o=P + (1 << 30), kind=getattr(pkg._lib, kind), D=D, Hq=heads * group, width=400, table_stride=400, k_stride=strides, v_stride=strides, q_stride=(heads * group * D, D), o_stride=(heads * group * D, D))
        window = (tiles - 1) * 128 - 60            # (a window may begin anywhere in its first tile)
        whole.append(lib.cosmos_attn_cache_window_workspace_bytes(ctypes.byref(d), window, 0) == 0)
        assert (lib.cosmos_attn_cache_window_workspace_bytes(ctypes.byref(d), window - 128, 1) == 0) == whole[-1] or tiles == 2      # (a tile of first keys counts as well)
    assert whole == [t <= most for t in range(2, 9)]

"""Windows, chunks over the cache and appending to it, what needs no GPU: status codes, refusals, sizes of workspaces."""
import ctypes

import pytest
import torch

from test_host_ragged import P, cache_desc, on, ragged_desc


def test_window_status_codes(pkg):
    L, lib = pkg._lib, pkg._lib.load_library()
    fwd = lambda D, w, s: lib.cosmos_attn_ragged_window(ctypes.byref(D), w, s, P, 1 << 40, None)
    bwd = lambda D, w, s: lib.cosmos_attn_ragged_window_bwd(ctypes.byref(D), w, s, P, 1 << 40, None)
    for call in (fwd, bwd):
        assert call(ragged_desc(pkg), -1, 0) == call(ragged_desc(pkg), 5, -1) == L.ST_BAD_ARG
        assert call(ragged_desc(pkg, causal=0), 5, 0) == L.ST_UNSUPPORTED
        assert call(ragged_desc(pkg, D=96), 5, 0) == L.ST_UNSUPPORTED and call(ragged_desc(pkg, q=None), 5, 0) == L.ST_BAD_ARG
    assert fwd(ragged_desc(pkg, Tq=0, q=None, o=None), 5, 0) == L.ST_OK
    for window, sinks in ((-1, 0), (5, -1)):
        assert lib.cosmos_attn_ragged_window_workspace_bytes(ctypes.byref(ragged_desc(pkg)), window, sinks) == lib.cosmos_attn_ragged_window_bwd_workspace_bytes(ctypes.byref(ragged_desc(pkg)), window, sinks) == 0
    assert lib.cosmos_attn_ragged_window_bwd(ctypes.byref(ragged_desc(pkg)), 5, 0, None, 0, None) == L.ST_WORKSPACE


def test_window_workspaces(pkg):
    """None or all of the keys: as without; a short window's tiles are not cut."""
    lib = pkg._lib.load_library()
    D = ragged_desc(pkg, Tq=4096, Tk=4096)
    of = lambda w, s: lib.cosmos_attn_ragged_window_workspace_bytes(ctypes.byref(D), w, s)
    assert of(0, 0) == of(4096, 0) == of(5, 4096) == of(1 << 62, 1 << 62) == lib.cosmos_attn_ragged_workspace_bytes(ctypes.byref(D)) > 0
    assert of(100, 4) == 0
    assert pkg.ragged._workspace_bytes(False, 3, 8, 2, 128, 4096, 4096) == of(0, 0) and pkg.ragged._workspace_bytes(False, 3, 8, 2, 128, 4096, 4096, 100, 4) == 0


def test_window_arguments(pkg, monkeypatch):
    def no_launch(*a):
        raise AssertionError("launched")

    for module in (pkg.ragged, pkg.kv_cache):
        monkeypatch.setattr(module, "on_device", no_launch)
    new = lambda *shape, dtype=torch.bfloat16: on(torch.zeros(*shape, dtype=dtype))
    q, k, cu, lse = new(4, 6, 64), new(4, 2, 64), new(2, dtype=torch.int32), new(6, 4, dtype=torch.float32)
    for over, error in [(dict(window=0), AssertionError), (dict(window=-3), AssertionError), (dict(window=5, sinks=-1), AssertionError), (dict(sinks=2), AssertionError), (dict(window=2.5), TypeError),
                        (dict(window=5, causal=False), NotImplementedError)]:
        over = {"causal": True, **over}
        for call in (lambda: pkg.ragged_fwd(q, k, k, cu, **over), lambda: pkg.ragged_bwd(q, k, k, q, lse, q, cu, **over), lambda: pkg.attention_ragged(q, k, k, cu, **over)):
            with pytest.raises(error, match="" if error is not AssertionError else "window|sinks|first keys"):
                call()

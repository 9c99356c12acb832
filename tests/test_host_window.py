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


def test_cache_window_and_chunk_status_codes(pkg):
    L, lib = pkg._lib, pkg._lib.load_library()
    one = lambda D, w=0, s=0: lib.cosmos_attn_cache_window(ctypes.byref(D), w, s, P, 1 << 40, None)
    more = lambda D, w=0, s=0: lib.cosmos_attn_cache_chunk(ctypes.byref(D), w, s, P, 1 << 40, None)
    for call in (one, more):
        assert call(cache_desc(pkg, cu=P), -1, 0) == call(cache_desc(pkg, cu=P), 5, -1) == L.ST_BAD_ARG
        for over, status in [(dict(abi_version=1), L.ST_BAD_ARG), (dict(kind=3), L.ST_UNSUPPORTED), (dict(D=32), L.ST_UNSUPPORTED), (dict(page_size=8), L.ST_BAD_SHAPE), (dict(Hq=0), L.ST_BAD_ARG),
                             (dict(Hq=7), L.ST_BAD_SHAPE), (dict(lens=None), L.ST_BAD_ARG), (dict(q=None), L.ST_BAD_ARG), (dict(o_stride=(512, 0)), L.ST_BAD_STRIDE), (dict(o_stride=(64, 64)), L.ST_BAD_STRIDE),
                             (dict(q=P + 2), L.ST_BAD_STRIDE), (dict(sm_scale=float("inf")), L.ST_BAD_ARG), (dict(table=None), L.ST_BAD_ARG)]:
            assert call(cache_desc(pkg, **{"cu": P, **over}), 5, 1) == status, over
    for over, status in [(dict(cu=None), L.ST_BAD_ARG), (dict(rows=-1), L.ST_BAD_ARG), (dict(rows=1 << 29), L.ST_UNSUPPORTED), (dict(rows=1 << 32), L.ST_UNSUPPORTED), (dict(B=1 << 24, Hkv=8), L.ST_UNSUPPORTED),
                         (dict(q_stride=((1 << 22) + 8, 64)), L.ST_BAD_STRIDE)]:
        assert more(cache_desc(pkg, **{"cu": P, **over})) == status, over
    assert more(cache_desc(pkg, cu=P, rows=0, q=None, o=None)) == L.ST_OK == one(cache_desc(pkg, B=0))
    long = cache_desc(pkg, cu=P, width=100, table_stride=100)
    assert lib.cosmos_attn_cache_chunk_workspace_bytes(ctypes.byref(long), 0, 0) > 0 == lib.cosmos_attn_cache_chunk_workspace_bytes(ctypes.byref(long), 64, 4)
    assert lib.cosmos_attn_cache_chunk(ctypes.byref(long), 0, 0, None, 0, None) == L.ST_WORKSPACE
    assert lib.cosmos_attn_cache_window_workspace_bytes(ctypes.byref(long), 0, 0) > 0 == lib.cosmos_attn_cache_window_workspace_bytes(ctypes.byref(long), 64, 4)


def test_refusals_of_pieces(pkg, monkeypatch):
    def no_launch(*a):
        raise AssertionError("launched")

    monkeypatch.setattr(pkg.kv_cache, "on_device", no_launch)
    new = lambda *shape, dtype=torch.bfloat16: on(torch.zeros(*shape, dtype=dtype))
    cache = pkg.KVCache(new(5, 2, 16, 64), new(5, 2, 16, 64))
    table, lens, cu, q = new(3, 2, dtype=torch.int32), new(3, dtype=torch.int32), new(4, dtype=torch.int32), new(9, 4, 64)
    for call, error in [
        (lambda: pkg.cache_attention(q, cache, table, lens), AssertionError),                       # nine rows for three sequences, no offsets
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=lens), AssertionError),
        (lambda: pkg.cache_attention(q, cache, table, cu, cu=cu), AssertionError),
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=new(4)), AssertionError),
        (lambda: pkg.cache_attention(new(9, 5, 64), cache, table, lens, cu=cu), AssertionError),
        (lambda: pkg.cache_attention(new(9, 4, 64, dtype=torch.float16), cache, table, lens, cu=cu), AssertionError),
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=cu, window=0), AssertionError),
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=cu, sinks=4), AssertionError),
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=cu, window=1.5), TypeError),
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=cu, out=new(8, 4, 64)), AssertionError),
        (lambda: pkg.cache_attention(q, cache, table, lens, cu=cu, out=on(torch.zeros(9, 4, 128, dtype=torch.bfloat16)[:, :, ::2])), ValueError),
    ]:
        with pytest.raises(error):
            call()


def rope(pkg, **over):
    R = pkg._lib.CacheRope()
    R.freqs, R.pairs, R.axes, R.eps = P, 32, 1, 1e-6
    for k, v in over.items():
        setattr(R, k, v)
    return R


def test_append_layout_and_status_codes(pkg):
    L, lib = pkg._lib, pkg._lib.load_library()
    assert ctypes.sizeof(L.CacheRope) == 64 == pkg.kv_cache._ROPE.size and L.CacheRope.pairs.offset == 40 and L.CacheRope.eps.offset == 56
    append = lambda D, R: lib.cosmos_attn_cache_append(ctypes.byref(D), ctypes.byref(R), None)
    for over, status in [(dict(abi_version=1), L.ST_BAD_ARG), (dict(kind=3), L.ST_UNSUPPORTED), (dict(D=32), L.ST_UNSUPPORTED), (dict(rows=5), L.ST_BAD_SHAPE), (dict(lens=None), L.ST_BAD_ARG),
                         (dict(k_rows=None), L.ST_BAD_ARG), (dict(v_rows_stride=(128, 60)), L.ST_BAD_STRIDE), (dict(rows=-1), L.ST_BAD_ARG), (dict(Hq=0), L.ST_BAD_ARG), (dict(o=None), L.ST_BAD_ARG),
                         (dict(q_stride=(512, 60)), L.ST_BAD_STRIDE), (dict(o_stride=(64, 64)), L.ST_BAD_STRIDE), (dict(v=P), L.ST_BAD_ARG), (dict(k_stride=(0, 2048, 64)), L.ST_BAD_STRIDE),
                         (dict(cu=P, rows=1 << 30, Hq=64, Hkv=8, q_stride=(4096, 64), o_stride=(4096, 64), k_stride=(8 * 32 * 64, 32 * 64, 64), v_stride=(8 * 32 * 64, 32 * 64, 64), k_scale_stride=(256, 32),
                               v_scale_stride=(256, 32)), L.ST_UNSUPPORTED)]:
        assert append(cache_desc(pkg, **over), rope(pkg)) == status, over
    for over, status in [(dict(pairs=12), L.ST_BAD_SHAPE), (dict(pairs=40), L.ST_BAD_SHAPE), (dict(pairs=-8), L.ST_BAD_ARG), (dict(axes=0), L.ST_BAD_ARG), (dict(axes=9, positions=P), L.ST_UNSUPPORTED),
                         (dict(axes=2), L.ST_BAD_ARG), (dict(freqs=None), L.ST_BAD_ARG), (dict(freqs=P + 4), L.ST_BAD_STRIDE), (dict(q_weight=P + 8), L.ST_BAD_STRIDE), (dict(positions=P + 2), L.ST_BAD_STRIDE),
                         (dict(positions=P, positions_stride=-1), L.ST_BAD_STRIDE), (dict(eps=float("nan")), L.ST_BAD_ARG), (dict(eps=-1.0), L.ST_BAD_ARG)]:
        assert append(cache_desc(pkg), rope(pkg, **over)) == status, over
    assert append(cache_desc(pkg, rows=0, cu=P, k_rows=None, q=None), rope(pkg)) == L.ST_OK
    assert lib.cosmos_attn_cache_append(ctypes.byref(cache_desc(pkg)), None, None) == L.ST_BAD_ARG


def test_refusals_of_append(pkg, monkeypatch):
    def no_launch(*a):
        raise AssertionError("launched")

    monkeypatch.setattr(pkg.kv_cache, "on_device", no_launch)
    new = lambda *shape, dtype=torch.bfloat16: on(torch.zeros(*shape, dtype=dtype))
    f32 = torch.float32
    cache = pkg.KVCache(new(5, 2, 16, 64), new(5, 2, 16, 64))
    table, lens, q, k, freqs = new(3, 2, dtype=torch.int32), new(3, dtype=torch.int32), new(3, 4, 64), new(3, 2, 64), new(32, dtype=f32)
    for args, over, error in [
        ((q, k, new(4, 2, 64)), {}, AssertionError), ((q, new(4, 2, 64), new(4, 2, 64)), {}, AssertionError), ((new(4, 4, 64), k, k), {}, AssertionError), ((q, new(3, 1, 64), new(3, 1, 64)), {}, AssertionError),
        ((new(3, 4, 64, dtype=torch.float16), k, k), {}, AssertionError), ((new(3, 4, 128), k, k), {}, AssertionError), ((q, k, k), dict(freqs=new(30, dtype=f32)), AssertionError),
        ((q, k, k), dict(freqs=new(40, dtype=f32)), AssertionError), ((q, k, k), dict(freqs=new(2, 32, dtype=f32)), AssertionError), ((q, k, k), dict(freqs=new(32, dtype=torch.int32)), AssertionError),
        ((q, k, k), dict(freqs=freqs, positions=new(4, dtype=torch.int32)), AssertionError), ((q, k, k), dict(freqs=freqs, positions=new(3, 2, dtype=torch.int32)), AssertionError),
        ((q, k, k), dict(freqs=freqs, positions=new(3, dtype=f32)), AssertionError), ((q, k, k), dict(freqs=None, positions=new(3, dtype=torch.int32)), AssertionError),
        ((q, k, k), dict(q_weight=new(32)), AssertionError), ((None, k, k), dict(q_weight=new(64)), AssertionError), ((None, k, k), dict(out=q), AssertionError), ((q, k, k), dict(out=new(3, 2, 64)), AssertionError),
        ((q, k, k), dict(out=on(torch.zeros(3, 4, 128, dtype=torch.bfloat16)[:, :, ::2])), ValueError), ((q, k, k), dict(cu=lens), AssertionError),
    ]:
        with pytest.raises(error):
            pkg.cache_append(cache, *args, table, lens, **{"freqs": freqs, **over})


def test_freqs_without_a_dim_are_refused(pkg, monkeypatch):
    """(by what looks at all arguments at once as well)"""
    def no_launch(*a):
        raise AssertionError("launched")

    monkeypatch.setattr(pkg.kv_cache, "on_device", no_launch)
    new = lambda *shape, dtype=torch.bfloat16: on(torch.zeros(shape, dtype=dtype))
    cache = pkg.KVCache(new(5, 2, 16, 64), new(5, 2, 16, 64))
    with pytest.raises(AssertionError, match="freqs must be"):
        pkg.cache_append(cache, new(3, 4, 64), new(3, 2, 64), new(3, 2, 64), new(3, 2, dtype=torch.int32), new(3, dtype=torch.int32), freqs=new(dtype=torch.float32))

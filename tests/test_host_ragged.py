"""Attention over packed sequences and over a paged cache, what needs no GPU: descriptor layouts and status codes (validation happens before anything touches the device), the Python
operators' refusals, and sizes of workspaces."""
import ctypes

import pytest
import torch

P = 0x7F0000000000      # never dereferenced: validation looks at values alone


def ragged_desc(pkg, **over):
    L = pkg._lib
    D = L.RaggedDesc()
    D.abi_version, D.dtype, D.n_seq, D.Hq, D.Hkv, D.D, D.causal, D.Tq, D.Tk, D.sm_scale = L.ABI_VERSION, L.DTYPE_BF16, 3, 8, 2, 128, 1, 100, 120, 0.1
    for i, name in enumerate(("q", "k", "v", "cu_q", "cu_k", "o", "lse", "dout", "dq", "dk", "dv")):
        setattr(D, name, P + 4096 * i)
    for name, heads in (("q", 8), ("k", 2), ("v", 2), ("o", 8), ("dout", 8), ("dq", 8), ("dk", 2), ("dv", 2)):
        setattr(D, name + "_stride", (ctypes.c_int64 * 2)(heads * 128, 128))
    for k, v in over.items():
        setattr(D, k, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
    return D


def test_ragged_desc_layout_and_status_codes(pkg):
    L, lib = pkg._lib, pkg._lib.load_library()
    assert ctypes.sizeof(L.RaggedDesc) == 8 * 4 + 2 * 8 + 8 + 11 * 8 + 16 * 8 + 8
    assert L.RaggedDesc.Tq.offset == 32 and L.RaggedDesc.q.offset == 56 and L.RaggedDesc.q_stride.offset == 144
    cases = [
        (dict(abi_version=1), L.ST_BAD_ARG), (dict(n_seq=-1), L.ST_BAD_ARG), (dict(Hkv=0), L.ST_BAD_ARG), (dict(q=None), L.ST_BAD_ARG), (dict(cu_k=None), L.ST_BAD_ARG),
        (dict(sm_scale=float("nan")), L.ST_BAD_ARG), (dict(sm_scale=float("inf")), L.ST_BAD_ARG), (dict(Tq=-1), L.ST_BAD_ARG),
        (dict(dtype=7), L.ST_UNSUPPORTED), (dict(D=96), L.ST_UNSUPPORTED), (dict(Tq=1 << 30), L.ST_UNSUPPORTED), (dict(Tk=1 << 31), L.ST_UNSUPPORTED), (dict(Tq=1 << 62), L.ST_UNSUPPORTED),
        (dict(n_seq=1 << 24), L.ST_UNSUPPORTED), (dict(Tk=1 << 30, Hkv=8), L.ST_UNSUPPORTED),
        (dict(Hkv=3), L.ST_BAD_SHAPE),
        (dict(k=P + 8), L.ST_BAD_STRIDE), (dict(cu_q=P + 2), L.ST_BAD_STRIDE), (dict(q_stride=(1020, 128)), L.ST_BAD_STRIDE), (dict(k_stride=(64, 128)), L.ST_BAD_STRIDE),
        (dict(v_stride=(256, -128)), L.ST_BAD_STRIDE), (dict(rest=P + 8), L.ST_BAD_STRIDE), (dict(k_stride=((1 << 22) + 8, 128)), L.ST_BAD_STRIDE), (dict(q_stride=(1024, 1 << 27)), L.ST_BAD_STRIDE),
        (dict(o_stride=(128, 64)), L.ST_BAD_STRIDE),
    ]
    for over, want in cases:
        assert lib.cosmos_attn_ragged(ctypes.byref(ragged_desc(pkg, **over)), P, 1 << 40, None) == want, over
        if "o_stride" not in over:
            assert lib.cosmos_attn_ragged_bwd(ctypes.byref(ragged_desc(pkg, **over)), P, 1 << 40, None) == want, over
        assert lib.cosmos_attn_ragged_bwd_workspace_bytes(ctypes.byref(ragged_desc(pkg, **over))) == 0 or "o_stride" in over
    # outputs whose rows share memory
    for over in (dict(o_stride=(1024, 0)), dict(o_stride=(512, 128))):
        assert lib.cosmos_attn_ragged(ctypes.byref(ragged_desc(pkg, **over)), P, 1 << 40, None) == L.ST_BAD_STRIDE
    for over in (dict(dq_stride=(1024, 0)), dict(dk_stride=(128, 128)), dict(dv=None), dict(dout=None), dict(lse=None)):
        assert lib.cosmos_attn_ragged_bwd(ctypes.byref(ragged_desc(pkg, **over)), P, 1 << 40, None) in (L.ST_BAD_STRIDE, L.ST_BAD_ARG), over
    D = ragged_desc(pkg)
    assert lib.cosmos_attn_ragged_bwd_workspace_bytes(ctypes.byref(D)) >= 100 * 8 * 4
    assert lib.cosmos_attn_ragged_bwd(ctypes.byref(D), None, 0, None) == L.ST_WORKSPACE
    # nothing to do: no launch, whatever the addresses are
    assert lib.cosmos_attn_ragged(ctypes.byref(ragged_desc(pkg, Tq=0, q=None, o=None)), None, 0, None) == L.ST_OK


def cache_desc(pkg, **over):
    L = pkg._lib
    D = L.CacheDesc()
    D.abi_version, D.dtype, D.kind, D.Hkv, D.D, D.page_size, D.pages = L.ABI_VERSION, L.DTYPE_BF16, L.CACHE_INT8, 2, 64, 32, 50
    D.B, D.width, D.table_stride, D.rows, D.Hq, D.sm_scale = 4, 10, 10, 4, 8, 0.1
    for i, name in enumerate(("k", "v", "k_scale", "v_scale", "table", "lens", "k_rows", "v_rows", "q", "o", "lse")):
        setattr(D, name, P + 4096 * i)
    D.k_stride = D.v_stride = (ctypes.c_int64 * 3)(2 * 32 * 64, 32 * 64, 64)
    D.k_scale_stride = D.v_scale_stride = (ctypes.c_int64 * 2)(2 * 32, 32)
    D.k_rows_stride = D.v_rows_stride = (ctypes.c_int64 * 2)(128, 64)
    D.q_stride = D.o_stride = (ctypes.c_int64 * 2)(512, 64)
    for k, v in over.items():
        setattr(D, k, (ctypes.c_int64 * len(v))(*v) if isinstance(v, tuple) else v)
    return D


def test_cache_desc_layout_and_status_codes(pkg):
    L, lib = pkg._lib, pkg._lib.load_library()
    assert ctypes.sizeof(L.CacheDesc) == 24 + 8 + 16 + 48 + 16 + 32 + 8 + 16 + 16 + 8 + 16 + 32 + 16 + 16 + 32 + 8
    assert L.CacheDesc.pages.offset == 24 and L.CacheDesc.table.offset == 152 and L.CacheDesc.q.offset == 256 and L.CacheDesc.lse.offset == 304
    write = lambda D: lib.cosmos_attn_cache_write(ctypes.byref(D), None)
    read = lambda D: lib.cosmos_attn_cache_read(ctypes.byref(D), None)
    attend = lambda D: lib.cosmos_attn_cache_attention(ctypes.byref(D), P, 1 << 40, None)
    for over, want in [
        (dict(abi_version=1), L.ST_BAD_ARG), (dict(pages=0), L.ST_BAD_ARG), (dict(k=None), L.ST_BAD_ARG), (dict(v_scale=None), L.ST_BAD_ARG), (dict(table=None), L.ST_BAD_ARG), (dict(B=-1), L.ST_BAD_ARG),
        (dict(dtype=5), L.ST_UNSUPPORTED), (dict(kind=3), L.ST_UNSUPPORTED), (dict(D=32), L.ST_UNSUPPORTED), (dict(width=1 << 26), L.ST_UNSUPPORTED), (dict(width=(1 << 25) + 1), L.ST_UNSUPPORTED),
        (dict(page_size=8), L.ST_BAD_SHAPE), (dict(page_size=48), L.ST_BAD_SHAPE), (dict(page_size=2048), L.ST_BAD_SHAPE),
        (dict(k=P + 8), L.ST_BAD_STRIDE), (dict(k_stride=(4096, 2048, 72)), L.ST_BAD_STRIDE), (dict(v_stride=(4096, 2048, 48)), L.ST_BAD_STRIDE),
        (dict(k_scale_stride=(64, 30)), L.ST_BAD_STRIDE), (dict(table=P + 1), L.ST_BAD_STRIDE), (dict(table_stride=-10), L.ST_BAD_STRIDE),
    ]:
        for call in (write, attend, lambda D: read(D)):
            D = cache_desc(pkg, cu=P, **over)
            assert call(D) == want, over
        assert lib.cosmos_attn_cache_attention_workspace_bytes(ctypes.byref(cache_desc(pkg, **over))) == 0
    for call in (write, read):
        assert call(cache_desc(pkg, cu=P, rows=1 << 30, Hkv=8)) == L.ST_UNSUPPORTED      # (more workgroups than a launch takes)
    assert attend(cache_desc(pkg, B=1 << 21, width=1, Hq=8)) == L.ST_UNSUPPORTED
    for over, want in [(dict(rows=5), L.ST_BAD_SHAPE), (dict(lens=None), L.ST_BAD_ARG), (dict(k_rows=None), L.ST_BAD_ARG), (dict(v_rows_stride=(128, 60)), L.ST_BAD_STRIDE), (dict(rows=-1), L.ST_BAD_ARG)]:
        assert write(cache_desc(pkg, **over)) == want, over
    for over, want in [(dict(cu=None), L.ST_BAD_ARG), (dict(cu=P, k_rows_stride=(64, 64)), L.ST_BAD_STRIDE), (dict(cu=P, v_rows_stride=(128, 0)), L.ST_BAD_STRIDE)]:
        assert read(cache_desc(pkg, **over)) == want, over
    for over, want in [(dict(Hq=0), L.ST_BAD_ARG), (dict(Hq=7), L.ST_BAD_SHAPE), (dict(lens=None), L.ST_BAD_ARG), (dict(q=None), L.ST_BAD_ARG), (dict(o_stride=(512, 0)), L.ST_BAD_STRIDE),
                       (dict(o_stride=(64, 64)), L.ST_BAD_STRIDE), (dict(q=P + 2), L.ST_BAD_STRIDE), (dict(sm_scale=float("inf")), L.ST_BAD_ARG)]:
        assert attend(cache_desc(pkg, **over)) == want, over
    D = cache_desc(pkg, width=100, table_stride=100)
    assert lib.cosmos_attn_cache_attention_workspace_bytes(ctypes.byref(D)) > 0
    assert lib.cosmos_attn_cache_attention(ctypes.byref(D), None, 0, None) == L.ST_WORKSPACE
    assert write(cache_desc(pkg, rows=0, k_rows=None)) == L.ST_OK and attend(cache_desc(pkg, B=0)) == L.ST_OK


def test_attention_workspace_does_not_grow_with_the_table(pkg):
    """Parts are kept for each workgroup, one of a share of all keys or of a sequence's last ones."""
    of = lambda B, width: pkg.kv_cache._workspace_bytes(8, 128, 64, B, width, 32)
    assert of(3, 1 << 14) == of(3, 1 << 12) > 0 and of(64, 1 << 14) < 2 * of(1, 1 << 14)
    assert pkg.kv_cache._workspace_bytes(8, 128, 16, 64, 32, 32) == 0          # tables of few tiles: nothing is shared


def test_python_argument_checks(pkg, monkeypatch):
    cpu = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: pkg.ragged_fwd(cpu, cpu, cpu, cu), lambda: pkg.attention_ragged(cpu, cpu, cpu, cu), lambda: pkg.KVCache(*[torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)] * 2)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(AssertionError):
        pkg.ragged_fwd(cpu[0], cpu, cpu, cu)
    with pytest.raises(NotImplementedError):
        pkg.KVCache.empty(2, 2, 16, 64, dtype=torch.float32, device="cpu")


class OnGpu(torch.Tensor):
    """A host tensor that says it is a GPU's: for refusals that come before anything is launched."""
    is_cuda = True


def on(x):
    return x.as_subclass(OnGpu)


def test_refusals_before_a_launch(pkg, monkeypatch):
    def no_launch(*a):
        raise AssertionError("launched")

    for module in (pkg.ragged, pkg.kv_cache):
        monkeypatch.setattr(module, "on_device", no_launch)
    new = lambda *shape, dtype=torch.bfloat16: on(torch.zeros(*shape, dtype=dtype))
    q, k, cu = new(4, 6, 64), new(4, 2, 64), new(2, dtype=torch.int32)
    for call, error in [
        (lambda: pkg.ragged_fwd(new(4, 6, 64, dtype=torch.float32), k, k, cu), NotImplementedError),
        (lambda: pkg.ragged_fwd(new(4, 6, 80), new(4, 2, 80), new(4, 2, 80), cu), NotImplementedError),
        (lambda: pkg.ragged_fwd(q, new(4, 2, 64, dtype=torch.float16), k, cu), AssertionError),
        (lambda: pkg.ragged_fwd(q, new(4, 4, 64), new(4, 4, 64), cu), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, new(5, 2, 64), cu), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, new(4, 2, 128), cu), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, k, new(2, 1, dtype=torch.int32)), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, k, cu, new(3, dtype=torch.int32)), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, k, new(2)), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, k, cu, out=new(4, 2, 64)), AssertionError),
        (lambda: pkg.ragged_fwd(q, k, k, cu, out=on(torch.zeros(4, 6, 128, dtype=torch.bfloat16)[:, :, ::2])), ValueError),
        (lambda: pkg.ragged_bwd(q, k, k, q, new(6, 4), q, cu), AssertionError),
        (lambda: pkg.ragged_bwd(q, k, k, k, new(6, 4, dtype=torch.float32), q, cu), AssertionError),
    ]:
        with pytest.raises(error):
            call()
    pages = lambda dtype=torch.bfloat16, page=16: new(5, 2, page, 64, dtype=dtype)
    scales = new(5, 2, 16, dtype=torch.float32)
    for call, error in [
        (lambda: pkg.KVCache(pages(), pages(torch.float16)), AssertionError),
        (lambda: pkg.KVCache(pages(page=24), pages(page=24)), AssertionError),
        (lambda: pkg.KVCache(pages(), pages(), scales, scales), AssertionError),
        (lambda: pkg.KVCache(pages(torch.int8), pages(torch.int8)), AssertionError),
        (lambda: pkg.KVCache(pages(torch.int8), pages(torch.int8), scales, new(5, 2, 16)), AssertionError),
        (lambda: pkg.KVCache(pages().transpose(2, 3), pages().transpose(2, 3)), (AssertionError, NotImplementedError)),
        (lambda: pkg.KVCache(new(5, 2, 16, 32), new(5, 2, 16, 32)), NotImplementedError),
    ]:
        with pytest.raises(error):
            call()
    cache = pkg.KVCache(pages(), pages())
    table, lens, one = new(3, 2, dtype=torch.int32), new(3, dtype=torch.int32), new(3, 2, 64)
    for call, error in [
        (lambda: pkg.cache_write(cache, one, new(4, 2, 64), table, lens), AssertionError),
        (lambda: pkg.cache_write(cache, new(4, 2, 64), new(4, 2, 64), table, lens), AssertionError),          # four rows for three sequences, no offsets
        (lambda: pkg.cache_write(cache, new(3, 1, 64), new(3, 1, 64), table, lens), AssertionError),
        (lambda: pkg.cache_write(cache, new(3, 2, 64, dtype=torch.float16), new(3, 2, 64, dtype=torch.float16), table, lens), AssertionError),
        (lambda: pkg.cache_write(cache, one, one, table, lens, cu=lens), AssertionError),
        (lambda: pkg.cache_write(cache, one, one, lens, lens), AssertionError),
        (lambda: pkg.cache_read(cache, table, lens, 3), AssertionError),
        (lambda: pkg.cache_read(cache, table, new(4, dtype=torch.int32), 3, dtype=torch.float32), NotImplementedError),
        (lambda: pkg.cache_attention(new(3, 5, 64), cache, table, lens), AssertionError),
        (lambda: pkg.cache_attention(new(3, 4, 128), cache, table, lens), AssertionError),
        (lambda: pkg.cache_attention(new(2, 4, 64), cache, table, new(2, dtype=torch.int32)), AssertionError),
        (lambda: pkg.cache_attention(new(3, 4, 64), cache, table, new(2, dtype=torch.int32)), AssertionError),
        (lambda: pkg.cache_attention(new(3, 4, 64), cache, table, lens, out=new(3, 4, 64, dtype=torch.float16)), AssertionError),
    ]:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("which", ["k", "v", "k_scale", "v_scale"])
@pytest.mark.parametrize("how", ["data", "set_", "resize_"])
def test_a_cache_whose_memory_was_exchanged_is_refused(pkg, monkeypatch, which, how):
    """Its descriptor holds addresses: what lies there may be another tensor's by now."""
    launched = []
    monkeypatch.setattr(pkg.kv_cache, "on_device", lambda *a: launched.append(a))
    monkeypatch.setattr(pkg.kv_cache, "plain_int32", lambda *a: True)
    make = lambda: (on(torch.zeros(5, 2, 16, 64, dtype=torch.int8)), on(torch.zeros(5, 2, 16, dtype=torch.float32)))
    (k, k_scale), (v, v_scale) = make(), make()
    cache = pkg.KVCache(k, v, k_scale, v_scale)
    cache._index = -1                 # (where a host tensor says it is)
    table, lens, one = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), on(torch.zeros(3, 2, 64, dtype=torch.bfloat16))
    calls = [lambda: pkg.cache_write(cache, one, one, table, lens), lambda: pkg.cache_read(cache, table, torch.zeros(4, dtype=torch.int32), 3), lambda: pkg.cache_attention(one, cache, table, lens)]
    for call in calls:
        call()
    assert len(launched) == 3
    x = getattr(cache, which)
    if how == "data":
        x.data = torch.zeros_like(x).as_subclass(torch.Tensor).clone()
    elif how == "set_":
        x.set_(torch.zeros_like(x).as_subclass(torch.Tensor).clone())
    else:
        x.resize_(500, *x.shape[1:])
    for call in calls:
        with pytest.raises(RuntimeError, match="exchanged"):
            call()
    assert len(launched) == 3


def test_pages_that_share_memory_are_not_written(pkg):
    """Pages, heads or rows that lie over each other (`expand`), and one memory as keys and values: to be read, but no two workgroups may write one place."""
    L, lib = pkg._lib, pkg._lib.load_library()
    write = lambda D: lib.cosmos_attn_cache_write(ctypes.byref(D), None)
    read = lambda D: lib.cosmos_attn_cache_read(ctypes.byref(D), None)
    good = [dict(), dict(k_stride=(64, 50 * 32 * 64, 50 * 64)), dict(v_stride=(2 * 2 * 32 * 64, 64, 128)), dict(pages=1, k_stride=(0, 2048, 64)), dict(Hkv=1, rows=4, v_stride=(2048, 0, 64)),
            dict(k_scale_stride=(32, 1600)), dict(k_stride=(1 << 40, 1 << 50, 64))]
    for over in good:
        for call in (write, read):
            assert call(cache_desc(pkg, cu=P, **over)) not in (L.ST_BAD_STRIDE, L.ST_BAD_ARG), over
    for over in [dict(k_stride=(0, 2048, 64)), dict(v_stride=(4096, 0, 64)), dict(k_stride=(2048, 2048, 64)), dict(v_stride=(4096, 2032, 64)), dict(k_stride=(4096, 64, 64)), dict(k_stride=(4080, 2048, 64)),
                 dict(k_scale_stride=(0, 32)), dict(v_scale_stride=(64, 28)), dict(k_scale_stride=(32, 32))]:
        assert write(cache_desc(pkg, cu=P, **over)) == L.ST_BAD_STRIDE, over
        assert read(cache_desc(pkg, cu=P, **over)) != L.ST_BAD_STRIDE, over
    for over in [dict(v=P), dict(v_scale=P + 2 * 4096)]:
        assert write(cache_desc(pkg, cu=P, **over)) == L.ST_BAD_ARG, over
        assert read(cache_desc(pkg, cu=P, **over)) != L.ST_BAD_ARG, over


def test_numbers_past_32_bits_stay_out_of_range(pkg):
    """Offsets, lengths and tables of 64 bits: what 32 do not hold is not taken for a number that they do."""
    far = torch.tensor([0, (1 << 32) + 5, 1 << 31, -(1 << 40) + 3, (1 << 31) - 1, -7])
    got = pkg.ragged.int32_on(far, far.device)
    assert got.dtype == torch.int32 and got.tolist() == [0, (1 << 31) - 1, (1 << 31) - 1, -(1 << 31), (1 << 31) - 1, -7]
    assert pkg.ragged.int32_on(torch.tensor([3, 1 << 62], dtype=torch.uint64), far.device).tolist() == [3, (1 << 31) - 1]
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int32):
        assert pkg.ragged.int32_on(torch.tensor([[3, 100], [0, 9]], dtype=dtype), far.device).tolist() == [[3, 100], [0, 9]]
    assert pkg.ragged.int32_on(far[::2], far.device).tolist() == [0, (1 << 31) - 1, (1 << 31) - 1]

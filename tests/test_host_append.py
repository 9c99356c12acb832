"""cache_append, what needs no GPU: calls without rows, outputs that lie over inputs."""
import ctypes

import pytest
import torch

from test_host_ragged import P, cache_desc
from test_host_window import rope


@pytest.mark.parametrize("axes", [1, 3, 8])
def test_no_rows_need_no_positions(pkg, axes):
    """(An empty tensor's address is null.)"""
    append = lambda **over: pkg._lib.load_library().cosmos_attn_cache_append(ctypes.byref(cache_desc(pkg, cu=P, **over)), ctypes.byref(rope(pkg, axes=axes, positions=None)), None)
    assert append(rows=0, k_rows=None, v_rows=None, q=None, o=None) == pkg._lib.ST_OK
    if axes > 1:
        assert append(rows=4) == pkg._lib.ST_BAD_ARG


def brute(a, a_stride, a_heads, b, b_stride, b_heads, rows, D):
    """Elements of two tensors [rows, heads, D], counted one by one (starts in elements)."""
    of = lambda at, stride, heads: {at + r * stride[0] + h * stride[1] + c for r in range(rows) for h in range(heads) for c in range(0, D, 8)}
    return bool(of(a, a_stride, a_heads) & of(b, b_stride, b_heads))


# (what is not refused is launched where there is a device, and the addresses are made up)
no_device = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="for machines without a GPU: calls that pass the checks end there")


def launched(status, L):
    """Neither a refusal of the arguments: there is no device here."""
    assert status in (L.ST_BAD_ARG, L.ST_WRONG_DEVICE), status
    return status == L.ST_WRONG_DEVICE


LAYOUTS = [                       # starts of q, o, k, v and strides of q, o, k, v, in elements; three rows of 4 and 2 heads of 64
    ((0, 0, 256, 384), ((512, 64), (512, 64), (512, 64), (512, 64))),              # queries in place in a fused projection
    ((0, 64, 512, 640), ((768, 64), (768, 64), (768, 64), (768, 64))),             # a head further
    ((0, 768, 256, 384), ((512, 64), (512, 64), (512, 64), (512, 64))),            # a row and a half further
    ((0, 256, 256, 384), ((512, 64), (512, 64), (512, 64), (512, 64))),            # over the keys
    ((0, 384, 256, 384), ((512, 64), (512, 64), (512, 64), (512, 64))),            # over the values
    ((0, 512, 256, 384), ((1024, 64), (1024, 64), (1024, 64), (1024, 64))),        # beside them
    ((0, 4096, 256, 384), ((512, 64), (256, 64), (512, 64), (512, 64))),           # behind all
    ((0, 1600, 256, 384), ((512, 64), (256, 64), (512, 64), (512, 64))),           # behind all, right behind the last element
    ((4096, 4096 + 192, 0, 192), ((64, 768), (64, 768), (64, 384), (64, 384))),    # heads first, a head of rows further
    ((4096, 4096 + 64, 0, 192), ((64, 192), (64, 192), (64, 384), (64, 384))),     # heads first, a row further
    ((8192, 0, 192, 1024), ((256, 64), (384, 64), (384, 64), (384, 64))),          # over the keys' last part of a row
    ((8192, 0, 256, 1024 + 512), ((256, 64), (384, 64), (384, 64), (384, 64))),    # right in front of them
]


@no_device
@pytest.mark.parametrize("at, strides", LAYOUTS)
def test_outputs_over_inputs_are_refused(pkg, at, strides):
    L, lib = pkg._lib, pkg._lib.load_library()
    names, heads = ("q", "o", "k_rows", "v_rows"), (4, 4, 2, 2)
    D = cache_desc(pkg, cu=P, rows=3, Hq=4, **{n: (P | 1 << 30) + 2 * a for n, a in zip(names, at)}, **{n + "_stride": s for n, s in zip(names, strides)})
    over = [brute(at[1], strides[1], 4, at[i], strides[i], h, 3, 64) for i, h in ((0, 4), (2, 2), (3, 2))]
    if at[0] == at[1] and strides[0] == strides[1]:
        over[0] = False
    assert launched(lib.cosmos_attn_cache_append(ctypes.byref(D), ctypes.byref(rope(pkg)), None), L) == (not any(over))
    assert launched(lib.cosmos_attn_cache_chunk(ctypes.byref(D), 0, 0, P, 1 << 40, None), L) == (not over[0])
    D.B = 3
    assert launched(lib.cosmos_attn_cache_window(ctypes.byref(D), 0, 0, P, 1 << 40, None), L) == (not over[0])


@no_device
def test_one_row_has_no_stride(pkg):
    L, lib = pkg._lib, pkg._lib.load_library()
    at = P | 1 << 30
    for o, over in ((at, True), (at + 64 * 2, False), (at + 64 * 6, True), (at + 64 * 8, False), (at - 64 * 2, False)):
        D = cache_desc(pkg, cu=P, rows=1, Hq=1, Hkv=1, q=at + 64 * 100, o=o, k_rows=at, v_rows=at + 64 * 6, q_stride=(8, 0), o_stride=(16, 0), k_rows_stride=(0, 0), v_rows_stride=(0, 0))
        assert launched(lib.cosmos_attn_cache_append(ctypes.byref(D), ctypes.byref(rope(pkg)), None), L) == (not over)

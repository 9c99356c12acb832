"""A paged key-value cache, in 16 or 8 bits, and attention of one new token of each sequence over it (``cosmos_attn_cache_write``, ``_read``, ``_attention``).

A sequence's keys and values lie in pages of a pool, in any order: position j in page ``table[i, j // page_size]``, place ``j % page_size``.  Tables and lengths are int32 tensors on the
device; nothing is copied to the host, and a captured step follows what they hold at the replay.

    cache = KVCache.empty(pages, heads, page_size, head_dim, dtype=torch.int8, device="cuda")
    cache_write(cache, k, v, table, lens, cu)                  # a prompt's keys and values, packed
    keys, values = cache_read(cache, table, cu_known, rows)    # back, in 16 bits: for the next piece of a prompt with ``attention_ragged``
    cache_write(cache, k1, v1, table, lens)                    # one new token of each sequence, ``lens`` with it
    o, _ = cache_attention(q, cache, table, lens)              # its attention over all of them

The reference has no counterpart (its networks see all of a video at once).  No gradients.
"""
from __future__ import annotations

import functools
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _DTYPES
from .ragged import HEAD_DIMS, check_rows, int32_on, on_device, packed, packed_ready, plain_int32

KINDS = {torch.bfloat16: _lib.CACHE_SAME, torch.float16: _lib.CACHE_SAME, torch.float8_e4m3fn: _lib.CACHE_E4M3, torch.int8: _lib.CACHE_INT8}

# struct cosmos_attn_cache_desc in two parts: what the cache says, and what the call does
_CACHE_PART = struct.Struct("=6iq2Q6q2Q4q")
_CALL_PART = struct.Struct("=2iQq2Qq2Q4q2ifi2Q4qQ")


class KVCache:
    """Pages of keys and values, ``[pages, heads, page_size, head_dim]`` each: bf16, fp16, or 8 bits (float8_e4m3fn, int8) with an fp32 scale for each row of a head,
    ``[pages, heads, page_size]``.  Takes the tensors as they are (any page, head and row strides of 16-byte steps) and writes into them:
    ``k``, ``v``, ``k_scale``, ``v_scale`` are theirs, and stay so: once a tensor's memory is exchanged (``.data``, ``set_``, ``resize_``) its cache is refused.
    Pages or heads that share memory (``expand``) can be read and attended to; writing them is refused."""

    __slots__ = ("_k", "_v", "_k_scale", "_v_scale", "pages", "heads", "page_size", "head_dim", "dtype", "device", "kind", "_parts", "_index", "_at")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        assert k.dim() == 4 and v.shape == k.shape, "k and v must be [pages, heads, page_size, head_dim]"
        if not k.is_cuda:
            raise RuntimeError("cosmos attention (HIP) needs tensors on a GPU; there is no CPU path")
        if k.dtype not in KINDS:
            raise NotImplementedError(f"a cache of {k.dtype} is not supported (bf16, fp16, float8_e4m3fn, int8)")
        assert v.dtype == k.dtype and v.device == k.device, "k and v must have one type and device"
        self.pages, self.heads, self.page_size, self.head_dim = k.shape
        if self.head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"head dim {self.head_dim}: the HIP kernels are built for {HEAD_DIMS}")
        assert self.pages >= 1 and self.heads >= 1 and 16 <= self.page_size <= 1024 and self.page_size & (self.page_size - 1) == 0, "page_size must be a power of two, 16 .. 1024"
        self.dtype, self.device, self.kind = k.dtype, k.device, KINDS[k.dtype]
        unit = 16 // k.element_size()
        for x in (k, v):
            assert x.stride(3) == 1 and all(s % unit == 0 for s in x.stride()[:3]) and x.data_ptr() % 16 == 0 and x.stride(2) >= self.head_dim, "rows of 16-byte steps"
        scales = (k_scale, v_scale)
        if self.kind == _lib.CACHE_SAME:
            assert k_scale is None and v_scale is None, "16 bits have no scales"
        else:
            for x in scales:
                assert x is not None and x.shape == k.shape[:3] and x.dtype == torch.float32 and x.device == k.device, "8 bits need fp32 scales [pages, heads, page_size]"
                assert x.stride(2) == 1 and x.stride(0) % 4 == 0 and x.stride(1) % 4 == 0 and x.data_ptr() % 16 == 0, "scales of a head's page lie side by side"
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self._index = k.get_device()
        at = lambda x: 0 if x is None else x.data_ptr()
        self._at = tuple((x, x.data_ptr()) for x in (k, v, k_scale, v_scale) if x is not None)
        steps = lambda x, n: (0,) * n if x is None else x.stride()[:n]
        self._parts = {
            dtype: _CACHE_PART.pack(_lib.ABI_VERSION, code, self.kind, self.heads, self.head_dim, self.page_size, self.pages, at(k), at(v), *steps(k, 3), *steps(v, 3),
                                    at(k_scale), at(v_scale), *steps(k_scale, 2), *steps(v_scale, 2))
            for dtype, code in _DTYPES.items()}

    k, v = property(lambda self: self._k), property(lambda self: self._v)
    k_scale, v_scale = property(lambda self: self._k_scale), property(lambda self: self._v_scale)

    def __reduce__(self):
        """A copy, or what is loaded, is a cache of its own tensors."""
        return type(self), (self._k, self._v, self._k_scale, self._v_scale)

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "KVCache":
        """A cache whose pages hold nothing yet."""
        if dtype not in KINDS:
            raise NotImplementedError(f"a cache of {dtype} is not supported (bf16, fp16, float8_e4m3fn, int8)")
        new = lambda: torch.empty((pages, heads, page_size, head_dim), dtype=dtype, device=device)
        scale = lambda: torch.empty((pages, heads, page_size), dtype=torch.float32, device=device) if KINDS[dtype] != _lib.CACHE_SAME else None
        return cls(new(), new(), scale(), scale())

    def _part(self, dtype: torch.dtype) -> bytes:
        for x, at in self._at:          # (the addresses in `_parts` are what a call writes to)
            if x.data_ptr() != at:
                raise RuntimeError("the memory of this cache's tensors was exchanged: make another KVCache of them")
        if self.kind == _lib.CACHE_SAME:
            assert dtype == self.dtype, f"a cache of {self.dtype} holds rows of that type, not {dtype}"
        return self._parts[dtype]


def _check_table(cache: KVCache, table: torch.Tensor) -> torch.Tensor:
    if plain_int32(table, 2, cache._index):
        return table
    table = int32_on(table, cache.device)
    assert table.dim() == 2, "table must be [sequences, pages of a sequence at most]"
    return table if table.shape[0] <= 1 or table.stride(0) >= 0 else table.contiguous()


def _check_numbers(x: torch.Tensor, count: int, cache: KVCache, what: str) -> torch.Tensor:
    if plain_int32(x, 1, cache._index) and x.shape[0] == count:
        return x
    x = int32_on(x, cache.device)
    assert x.dim() == 1 and x.shape[0] == count, f"{what} numbers are needed"
    return x


def _call(table, lens=0, cu=0, rows=0, k=0, v=0, k_stride=(0, 0), v_stride=(0, 0), fill=0, Hq=0, sm_scale=0.0, q=0, o=0, q_stride=(0, 0), o_stride=(0, 0), lse=0) -> bytes:
    B, width = table.shape
    return _CALL_PART.pack(B, width, table.data_ptr(), table.stride()[0], lens, cu, rows, k, v, *k_stride, *v_stride, fill, Hq, sm_scale, 0, q, o, *q_stride, *o_stride, lse)


def _check_rows(x: torch.Tensor, name: str, cache: KVCache, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of the cache's head dim and device, as the kernels take them."""
    if not (x.is_cuda and x.dim() == 3 and x.dtype in _DTYPES and x.get_device() == cache._index and (like is None or x.dtype is like.dtype)):
        check_rows(x, name, like)
    assert x.device == cache.device and x.shape[2] == cache.head_dim, f"{name} must be [rows, heads, D] of the cache's head dim, on its device"
    return x if packed_ready(x) else packed(x)


def cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, cu: Optional[torch.Tensor] = None) -> None:
    """Packed rows ``k``, ``v`` ``[rows, heads, D]`` into the cache: sequence i's are ``cu[i] .. cu[i + 1] - 1`` (``cu`` None: one for each sequence), its last positions; ``lens[i]`` counts them.

    8 bits: ``scale = max |x| * fp32(1 / 448)`` (e4m3) or ``* fp32(1 / 127)`` (int8), ``code = round(x / scale)``, all in fp32; a row with a value that is not finite reads back as NaN.
    Rows of no sequence, sequences whose ``lens`` is below their rows, positions that the table does not hold and pages outside of the cache: nothing is written.  No two rows of a call
    may have one place."""
    k = _check_rows(k, "k", cache)
    v = _check_rows(v, "v", cache, k)
    assert k.shape == v.shape and k.shape[1] == cache.heads, "k and v must be [rows, heads, D] of the cache"
    part, table = cache._part(k.dtype), _check_table(cache, table)
    B, rows = table.shape[0], k.shape[0]
    lens = _check_numbers(lens, B, cache, "as many lengths as the table has sequences: its")
    if cu is None:
        assert rows == B, "one row for each sequence, or offsets"
    else:
        cu = _check_numbers(cu, B + 1, cache, "one offset more than the table has sequences: its")
    desc = part + _call(table, lens.data_ptr(), 0 if cu is None else cu.data_ptr(), rows, k.data_ptr(), v.data_ptr(), k.stride()[:2], v.stride()[:2])
    on_device(cache._index, _lib.load_library().cosmos_attn_cache_write, desc)


def cache_read(cache: KVCache, table: torch.Tensor, cu: torch.Tensor, rows: int, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, ``[rows, heads, D]``: the first ``cu[i + 1] - cu[i]`` positions of sequence i as the rows from ``cu[i]`` on.  ``dtype``: of the results where the cache has 8 bits
    (bf16 unless said), code times scale rounded.  Rows of no sequence are zeros; what pages outside of the cache or the table would hold is NaN."""
    if dtype is None:
        dtype = cache.dtype if cache.kind == _lib.CACHE_SAME else torch.bfloat16
    if dtype not in _DTYPES:
        raise NotImplementedError(f"dtype={dtype} is not supported (bf16 / fp16)")
    assert rows >= 0
    part, table = cache._part(dtype), _check_table(cache, table)
    cu = _check_numbers(cu, table.shape[0] + 1, cache, "one offset more than the table has sequences: its")
    heads, D = cache.heads, cache.head_dim
    k = torch.empty((rows, heads, D), dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    desc = part + _call(table, 0, cu.data_ptr(), rows, k.data_ptr(), v.data_ptr(), (heads * D, D), (heads * D, D), 1)
    on_device(cache._index, _lib.load_library().cosmos_attn_cache_read, desc)
    return k, v


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(Hkv: int, D: int, page_size: int, B: int, width: int, Hq: int) -> int:
    """What the library asks for, which follows from sizes alone (addresses are never dereferenced)."""
    part = _CACHE_PART.pack(_lib.ABI_VERSION, _lib.DTYPE_BF16, _lib.CACHE_SAME, Hkv, D, page_size, 1, 16, 16, *(page_size * Hkv * D, page_size * D, D) * 2, 0, 0, 0, 0, 0, 0)
    call = _CALL_PART.pack(B, width, 16, width, 16, 0, 0, 0, 0, 0, 0, 0, 0, 0, Hq, 1.0, 0, 16, 16, Hq * D, D, Hq * D, D, 0)
    return _lib.load_library().cosmos_attn_cache_attention_workspace_bytes(part + call)


def cache_attention(
    q: torch.Tensor,
    cache: KVCache,
    table: torch.Tensor,
    lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    need_lse: bool = False,
    out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(o, lse)``: attention of one token of each sequence, ``q [B, Hq, D]``, over the first ``lens[i]`` positions that its row of ``table`` holds; ``lse``: fp32 ``[B, Hq]``.

    ``lens[i] == 0``: o = 0, lse = -inf.  A length that the table does not hold, or a page outside of the cache among a sequence's: NaN.  ``out``: a tensor for o."""
    q = _check_rows(q, "q", cache)
    B, Hq, D = q.shape
    assert Hq >= 1 and Hq % cache.heads == 0, "q must be [B, Hq, D], Hq a multiple of the cache's heads"
    part, table = cache._part(q.dtype), _check_table(cache, table)
    assert table.shape[0] == B, "a row of the table for each sequence"
    lens = _check_numbers(lens, B, cache, "as many lengths as there are sequences: their")
    if out is None:
        o = torch.empty_like(q) if q.is_contiguous() else torch.empty((B, Hq, D), dtype=q.dtype, device=q.device)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must have q's shape, type and device"
        if not packed_ready(out):
            raise ValueError("out: rows of 16-byte steps are written in place, this view cannot be")
        o = out
    lse = q.new_empty((B, Hq), dtype=torch.float32) if need_lse else None
    ws_bytes = _workspace_bytes(cache.heads, D, cache.page_size, B, table.shape[1], Hq)
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    desc = part + _call(table, lens.data_ptr(), 0, 0, 0, 0, (0, 0), (0, 0), 0, Hq, D ** -0.5 if sm_scale is None else sm_scale, q.data_ptr(), o.data_ptr(), q.stride()[:2], o.stride()[:2],
                        0 if lse is None else lse.data_ptr())
    on_device(cache._index, _lib.load_library().cosmos_attn_cache_attention, desc, 0 if workspace is None else workspace.data_ptr(), ws_bytes)
    return o, lse

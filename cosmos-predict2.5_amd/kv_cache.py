"""A paged key-value cache, in 16 or 8 bits, and attention of one new token of each sequence over it (``cosmos_attn_cache_write``, ``_read``, ``_attention``).

A sequence's keys and values lie in pages of a pool, in any order: position j in page ``table[i, j // page_size]``, place ``j % page_size``.  Tables and lengths are int32 tensors on the
device; nothing is copied to the host, and a captured step follows what they hold at the replay.

    cache = KVCache.empty(pages, heads, page_size, head_dim, dtype=torch.int8, device="cuda")
    cache_write(cache, k, v, table, lens, cu)                  # a prompt's keys and values, packed
    o, _ = cache_attention(q, cache, table, lens, cu=cu)       # its attention over them and all before, causal
    q1 = cache_append(cache, q1, k1, v1, table, lens, freqs=freqs)      # one new token of each sequence, ``lens`` with it: queries and keys turned by their positions, keys and values written
    o, _ = cache_attention(q1, cache, table, lens)             # its attention over all of them
    keys, values = cache_read(cache, table, cu_known, rows)    # back, in 16 bits

The reference has no counterpart (its networks see all of a video at once).  No gradients.
"""
from __future__ import annotations

import functools
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _DTYPES
from .ragged import HEAD_DIMS, check_rows, checked_window, int32_on, on_device, packed, packed_ready, plain_int32

KINDS = {torch.bfloat16: _lib.CACHE_SAME, torch.float16: _lib.CACHE_SAME, torch.float8_e4m3fn: _lib.CACHE_E4M3, torch.int8: _lib.CACHE_INT8}

# struct cosmos_attn_cache_desc in two parts: what the cache says, and what the call does
_CACHE_PART = struct.Struct("=6iq2Q6q2Q4q")
_CALL_PART = struct.Struct("=2iQq2Qq2Q4q2ifi2Q4qQ")
# struct cosmos_attn_cache_rope
_ROPE = struct.Struct("=2Qq2Q4ifi")


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


def _check_weight(weight: Optional[torch.Tensor], like: torch.Tensor, name: str) -> Optional[torch.Tensor]:
    """A norm's weight as the kernels take it: fp32, or of the rows' type, at 16 bytes."""
    if weight is None:
        return None
    assert weight.dim() == 1 and weight.shape[0] == like.shape[2] and weight.device == like.device, f"{name} must be [D], on the rows' device"
    if weight.dtype != like.dtype and weight.dtype != torch.float32:
        weight = weight.float()
    return weight if weight.stride(0) == 1 and weight.data_ptr() % 16 == 0 else weight.clone(memory_format=torch.contiguous_format)


def _is_weight(x: Optional[torch.Tensor], D: int, device: int) -> bool:
    return x is None or (x.dim() == 1 and x.shape[0] == D and x.get_device() == device and x.is_contiguous() and not x.data_ptr() & 15)


def _append_as_it_is(cache, q, k, v, table, lens, cu, freqs, positions, interleaved, q_weight, k_weight, eps):
    """:func:`cache_append` of tensors that can be taken as they are, all of it looked at once: None where something is to be converted, copied or refused.  (One new token: 9.6 us, 13 with
    the checks one by one.)"""
    if not (q.dim() == 3 == k.dim() and 1 <= freqs.dim() <= 2 == table.dim()):
        return None
    device, dtype, D = cache._index, k.dtype, cache.head_dim
    (rows, Hq, _), shape, (B, width) = q.shape, k.shape, table.shape
    axes, pairs = freqs.shape if freqs.dim() == 2 else (1, freqs.shape[0])
    pq, pk, pv, pf = q.data_ptr(), k.data_ptr(), v.data_ptr(), freqs.data_ptr()
    if (dtype not in _DTYPES or shape != (rows, cache.heads, D) or v.shape != shape or q.shape[2] != D or q.dtype is not dtype or v.dtype is not dtype or freqs.dtype is not torch.float32
            or not (q.get_device() == k.get_device() == v.get_device() == freqs.get_device() == device) or not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous() and freqs.is_contiguous())
            or (pq | pk | pv | pf) & 15 or Hq < 1 or max(Hq, cache.heads) * D > 1 << 22 or pairs % 8 or 2 * pairs > D or axes < 1
            or not plain_int32(table, 2, device) or table.stride()[0] < 0 or not plain_int32(lens, 1, device) or lens.shape[0] != B
            or (rows != B if cu is None else not plain_int32(cu, 1, device) or cu.shape[0] != B + 1)
            or (axes != 1 if positions is None else positions.shape != (rows, axes) or not plain_int32(positions, 2, device) or not positions.is_contiguous())
            or not _is_weight(q_weight, D, device) or not _is_weight(k_weight, D, device)):
        return None
    weight_16 = 0
    if q_weight is not None or k_weight is not None:
        kinds = {w.dtype for w in (q_weight, k_weight) if w is not None}
        if kinds != {torch.float32} and kinds != {dtype}:
            return None
        weight_16 = 0 if kinds == {torch.float32} else 1
    part, o, own = cache._part(dtype), torch.empty_like(q), cache.heads * D
    desc = part + _CALL_PART.pack(B, width, table.data_ptr(), table.stride()[0], lens.data_ptr(), 0 if cu is None else cu.data_ptr(), rows, pk, pv, own, D, own, D, 1, Hq, 0.0, 0, pq, o.data_ptr(),
                                  Hq * D, D, Hq * D, D, 0)
    rope = _ROPE.pack(pf, 0 if positions is None else positions.data_ptr(), axes, 0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), pairs, axes,
                      1 if interleaved else 0, weight_16, eps, 0)
    on_device(device, _lib.load_library().cosmos_attn_cache_append, desc, rope)
    return o


def cache_append(
    cache: KVCache,
    q: Optional[torch.Tensor],
    k: torch.Tensor,
    v: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    cu: Optional[torch.Tensor] = None,
    *,
    freqs: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    out: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """New tokens, packed as for :func:`cache_write`: keys are normalised and turned by their positions and written with their values; returns the queries, normalised and turned, ``[rows, Hq, D]``
    (``q`` None: None; ``out`` takes them: memory of its own, or ``q`` itself; one that lies over ``k``, ``v`` or other rows of ``q`` is refused).

    ``freqs``: ``[R]`` or ``[axes, R]``, fp32 (others are rounded to it), radians a position, for R pairs of channels (a multiple of 8, ``2 R <= D``): ``(i, i + R)``, or with ``interleaved`` ``(2 i, 2 i + 1)``; the channels behind
    are not turned (None: none are).  The angle of pair i is ``sum_a positions[row, a] * freqs[a, i]``, formed in 64 bits; ``positions``: whole numbers of 32 bits, ``[rows]`` or ``[rows, axes]``, of images and
    videos say; None: the token's place in its sequence.
    ``q_weight``, ``k_weight``: ``[D]`` of the RMS norm (``eps``) of each head's row in front of that; None: no norm.  All of it in fp32, rounded once: to the rows' type, or to the cache's 8 bits.
    Queries of no sequence, and of sequences whose ``lens`` is below their rows, become zeros (in ``out``: left as they are).  As in :func:`cache_write`, what has no place is not written."""
    if q is not None and freqs is not None and out is None:
        made = _append_as_it_is(cache, q, k, v, table, lens, cu, freqs, positions, interleaved, q_weight, k_weight, eps)
        if made is not None:
            return made
    k = _check_rows(k, "k", cache)
    v = _check_rows(v, "v", cache, k)
    assert k.shape == v.shape and k.shape[1] == cache.heads, "k and v must be [rows, heads, D] of the cache"
    part, table = cache._part(k.dtype), _check_table(cache, table)
    B, rows, D = table.shape[0], k.shape[0], cache.head_dim
    lens = _check_numbers(lens, B, cache, "as many lengths as the table has sequences: its")
    if cu is None:
        assert rows == B, "one row for each sequence, or offsets"
    else:
        cu = _check_numbers(cu, B + 1, cache, "one offset more than the table has sequences: its")
    if q is None:
        assert out is None and q_weight is None, "out and q_weight are the queries'"
        o, Hq = None, 0
    else:
        q = _check_rows(q, "q", cache, k)
        Hq = q.shape[1]
        assert q.shape[0] == rows and Hq >= 1, "q must be [rows, Hq, D], a row for each of k's"
        if out is None:
            o = torch.empty_like(q) if q.is_contiguous() else torch.empty((rows, Hq, D), dtype=q.dtype, device=q.device)
        else:
            assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must have q's shape, type and device"
            if not packed_ready(out):
                raise ValueError("out: rows of 16-byte steps are written in place, this view cannot be")
            o = out
    q_weight, k_weight = _check_weight(q_weight, k, "q_weight"), _check_weight(k_weight, k, "k_weight")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        q_weight, k_weight = q_weight.float(), k_weight.float()
    weight_16 = any(w is not None and w.dtype != torch.float32 for w in (q_weight, k_weight))
    axes, pairs = 1, 0
    if freqs is None:
        assert positions is None, "positions need freqs"
    else:
        assert freqs.dim() in (1, 2) and freqs.is_floating_point(), "freqs must be [pairs] or [axes, pairs]"
        if freqs.dtype != torch.float32 or freqs.get_device() != cache._index or not freqs.is_contiguous() or freqs.data_ptr() % 16:
            freqs = freqs.to(device=cache.device, dtype=torch.float32).clone(memory_format=torch.contiguous_format)
        axes, pairs = freqs.shape if freqs.dim() == 2 else (1, freqs.shape[0])
        assert pairs % 8 == 0 and 2 * pairs <= D and axes >= 1, "freqs hold a multiple of 8 pairs, of at most D channels"
        assert positions is not None or axes == 1, "several axes need positions"
    if positions is not None:
        positions = int32_on(positions, cache.device)
        if positions.dim() == 1:
            positions = positions[:, None]
        assert positions.dim() == 2 and positions.shape == (rows, axes), "positions must be [rows, axes]"
        if (axes > 1 and positions.stride(1) != 1) or positions.stride(0) < 0:
            positions = positions.contiguous()
    at = lambda x: 0 if x is None else x.data_ptr()
    desc = part + _call(table, lens.data_ptr(), at(cu), rows, k.data_ptr(), v.data_ptr(), k.stride()[:2], v.stride()[:2], 0 if out is not None else 1, Hq, 0.0, at(q), at(o),
                        (0, 0) if q is None else q.stride()[:2], (0, 0) if q is None else o.stride()[:2])
    rope = _ROPE.pack(at(freqs), at(positions), 0 if positions is None else positions.stride(0), at(q_weight), at(k_weight), pairs, axes, 1 if interleaved else 0, 1 if weight_16 else 0, eps, 0)
    on_device(cache._index, _lib.load_library().cosmos_attn_cache_append, desc, rope)
    return o


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
def _workspace_bytes(Hkv: int, D: int, page_size: int, B: int, width: int, Hq: int, window: int = 0, sinks: int = 0, rows: int = -1, kind: int = _lib.CACHE_SAME) -> int:
    """What the library asks for, which follows from sizes and the cache's kind alone (addresses are never dereferenced).  `rows`: of a call with offsets."""
    part = _CACHE_PART.pack(_lib.ABI_VERSION, _lib.DTYPE_BF16, kind, Hkv, D, page_size, 1, 16, 16, *(page_size * Hkv * D, page_size * D, D) * 2, 16, 16, 0, 0, 0, 0)
    call = _CALL_PART.pack(B, width, 16, width, 16, 16, max(rows, 0), 0, 0, 0, 0, 0, 0, 0, Hq, 1.0, 0, 16, 16, Hq * D, D, Hq * D, D, 0)
    lib = _lib.load_library()
    return (lib.cosmos_attn_cache_window_workspace_bytes if rows < 0 else lib.cosmos_attn_cache_chunk_workspace_bytes)(part + call, window, sinks)


def _attention_as_it_is(q, cache, table, lens, sm_scale, need_lse, cu, window, sinks):
    """:func:`cache_attention` of tensors that can be taken as they are, all of it looked at once: None where something is to be converted, copied or refused.  (One new
    token: 9.9 us, 11.1 with the checks one by one.)"""
    if not q.dim() == 3 == 1 + table.dim():
        return None
    device, dtype, D, pq = cache._index, q.dtype, cache.head_dim, q.data_ptr()
    (rows, Hq, of), (B, width) = q.shape, table.shape
    if (dtype not in _DTYPES or of != D or q.get_device() != device or not q.is_contiguous() or pq & 15 or Hq < 1 or Hq % cache.heads or Hq * D > 1 << 22
            or not plain_int32(table, 2, device) or not plain_int32(lens, 1, device) or lens.shape[0] != B
            or (rows != B if cu is None else not plain_int32(cu, 1, device) or cu.shape[0] != B + 1)):
        return None
    part, o, row = cache._part(dtype), torch.empty_like(q), Hq * D
    lse = q.new_empty((rows, Hq), dtype=torch.float32) if need_lse else None
    desc = part + _CALL_PART.pack(B, width, table.data_ptr(), table.stride()[0], lens.data_ptr(), 0 if cu is None else cu.data_ptr(), rows, 0, 0, 0, 0, 0, 0, _lib.FILL_ALL, Hq,
                                  D ** -0.5 if sm_scale is None else sm_scale, 0, pq, o.data_ptr(), row, D, row, D, 0 if lse is None else lse.data_ptr())
    ws_bytes = _workspace_bytes(cache.heads, D, cache.page_size, B, width, Hq, window, sinks, -1 if cu is None else rows, cache.kind)
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    lib = _lib.load_library()
    on_device(device, lib.cosmos_attn_cache_window if cu is None else lib.cosmos_attn_cache_chunk, desc, window, sinks, 0 if workspace is None else workspace.data_ptr(), ws_bytes)
    return o, lse


def cache_attention(
    q: torch.Tensor,
    cache: KVCache,
    table: torch.Tensor,
    lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    need_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    cu: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(o, lse)``: attention of one token of each sequence, ``q [B, Hq, D]``, over the first ``lens[i]`` positions that its row of ``table`` holds; ``lse``: fp32 ``[B, Hq]``.

    ``cu``: of the sequences' last tokens, packed, ``q [rows, Hq, D]``: sequence i's are the rows ``cu[i] .. cu[i + 1] - 1`` and its last positions of ``lens[i]``, whose keys and values are in the
    cache already; each sees the positions up to its own; keys and values that it does not see have to be finite where another token of its sequence in the call sees them.  ``lse``: ``[rows, Hq]``.  Offsets as in :func:`ragged_fwd`; rows of no sequence become zeros, and -inf (in ``out``: left as they are).
    ``window``: a token sees that many last positions, its own among them, and those below ``sinks``; pages that no token of a sequence sees are not looked up, whatever the table says of them.

    A token that sees nothing (``lens[i] == 0``, or below its rows): o = 0, lse = -inf.  A length that the table does not hold: NaN.  A page outside of the cache: NaN for the tokens that see it.
    ``out``: a tensor for o, of its own memory or ``q`` itself."""
    window, sinks = checked_window(window, sinks)
    if out is None:
        made = _attention_as_it_is(q, cache, table, lens, sm_scale, need_lse, cu, window, sinks)
        if made is not None:
            return made
    q = _check_rows(q, "q", cache)
    rows, Hq, D = q.shape
    assert Hq >= 1 and Hq % cache.heads == 0, "q must be [rows, Hq, D], Hq a multiple of the cache's heads"
    part, table = cache._part(q.dtype), _check_table(cache, table)
    B = table.shape[0]
    lens = _check_numbers(lens, B, cache, "as many lengths as there are sequences: their")
    if cu is None:
        assert rows == B, "a row of the table for each sequence, or offsets"
    else:
        cu = _check_numbers(cu, B + 1, cache, "one offset more than the table has sequences: its")
    if out is None:
        o = torch.empty_like(q) if q.is_contiguous() else torch.empty((rows, Hq, D), dtype=q.dtype, device=q.device)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must have q's shape, type and device"
        if not packed_ready(out):
            raise ValueError("out: rows of 16-byte steps are written in place, this view cannot be")
        o = out
    lse = q.new_empty((rows, Hq), dtype=torch.float32) if need_lse else None
    ws_bytes = _workspace_bytes(cache.heads, D, cache.page_size, B, table.shape[1], Hq, window, sinks, -1 if cu is None else rows, cache.kind)
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    desc = part + _call(table, lens.data_ptr(), 0 if cu is None else cu.data_ptr(), rows, 0, 0, (0, 0), (0, 0), _lib.FILL_ALL if out is None else _lib.FILL_LSE, Hq,
                        D ** -0.5 if sm_scale is None else sm_scale, q.data_ptr(), o.data_ptr(), q.stride()[:2], o.stride()[:2], 0 if lse is None else lse.data_ptr())
    lib = _lib.load_library()
    on_device(cache._index, lib.cosmos_attn_cache_window if cu is None else lib.cosmos_attn_cache_chunk, desc, window, sinks, 0 if workspace is None else workspace.data_ptr(), ws_bytes)
    return o, lse

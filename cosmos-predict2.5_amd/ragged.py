"""Attention over packed sequences of different lengths with grouped heads, and its gradients (``cosmos_attn_ragged``, ``cosmos_attn_ragged_bwd``).

All sequences of a batch lie one behind the other, ``[rows, heads, D]``, and int32 offsets on the device say where each begins: no padding, no copy of the lengths to the host, and a captured
call follows offsets that change between replays.  Each ``Hq / Hkv`` query heads in a row share a key head.  With ``causal`` the masks are aligned at the sequences' ends: the last query sees
every key, so queries may be the last few of a prompt whose first keys come from elsewhere (``kv_cache.cache_read``).  With ``window`` a query looks back on that many keys, its own among them, and
on the first ``sinks`` of its sequence; time goes by what is seen.

The reference has no counterpart: its attention takes one length for the batch (cosmos_predict2/_src/predict2/networks/attention.py:90-181 ignores ``q_lens`` / ``k_lens``).
"""
from __future__ import annotations

import functools
import operator
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPES, _on_device

HEAD_DIMS = (64, 128)
_MOST_ROW_BYTES = 1 << 23

# struct cosmos_attn_ragged_desc in one go
_RAGGED_DESC = struct.Struct("@8i2qfi11Q16qQ")


def packed_ready(x: torch.Tensor) -> bool:
    """Can the kernels read ``[rows, heads, D]`` as it is: elements of a row of a head side by side, 16-byte steps, rows behind each other?"""
    rows, heads, D = x.shape
    row, head, last = x.stride()
    return (last == 1 and row % 8 == 0 and head % 8 == 0 and x.data_ptr() % 16 == 0 and (rows <= 1 or row >= D) and head >= 0
            and 2 * row <= _MOST_ROW_BYTES and (heads <= 1 or 2 * heads * head <= 1 << 30))


def packed(x: torch.Tensor) -> torch.Tensor:
    return x if packed_ready(x) else x.clone(memory_format=torch.contiguous_format)


def check_rows(x: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> None:
    """A GPU's 16-bit ``[rows, heads, D]`` of a head dim that is built, on the device and of the type of ``like``."""
    assert x.dim() == 3, f"{name} must be [rows, heads, D]"
    if not x.is_cuda:
        raise RuntimeError("cosmos attention (HIP) needs tensors on a GPU; there is no CPU path")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"{name}: dtype={x.dtype} is not supported (bf16 / fp16)")
    if x.shape[2] not in HEAD_DIMS:
        raise NotImplementedError(f"{name}: head dim {x.shape[2]}: the HIP kernels are built for {HEAD_DIMS}")
    if like is not None:
        assert x.dtype == like.dtype and x.device == like.device, f"{name} must have the type and device of the others"


def int32_on(x: torch.Tensor, device: torch.device) -> torch.Tensor:
    """Offsets, lengths and tables as the kernels take them: int32 on the device, elements of the last dim side by side."""
    assert not x.is_floating_point() and not x.is_complex() and x.dtype != torch.bool, "offsets, lengths and tables are whole numbers"
    if x.dtype != torch.int32 or x.device != device:
        if x.dtype in (torch.int64, torch.uint64):      # (2^32 + 5 is not 5)
            x = x.to(torch.int64).clamp(-(1 << 31), (1 << 31) - 1)
        x = x.to(device=device, dtype=torch.int32)
    return x if x.dim() == 0 or x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _check(q, k, v, cu_q, cu_k):
    check_rows(q, "q")
    check_rows(k, "k", q)
    check_rows(v, "v", q)
    assert k.shape == v.shape and k.shape[2] == q.shape[2], "k and v have one shape, and q their head dim"
    assert q.shape[1] >= 1 and k.shape[1] >= 1 and q.shape[1] % k.shape[1] == 0, "the query heads are a multiple of the key heads"
    cu_q = int32_on(cu_q, q.device)
    cu_k = cu_q if cu_k is None else int32_on(cu_k, q.device)
    assert cu_q.dim() == 1 and cu_q.shape == cu_k.shape and cu_q.shape[0] >= 1, "cu_q and cu_k hold one offset more than there are sequences"
    return cu_q, cu_k


def checked_window(window: Optional[int], sinks: int, causal: bool = True) -> Tuple[int, int]:
    """``(window, sinks)`` as the library takes them, ``(0, 0)`` where none is asked for."""
    sinks = operator.index(sinks)
    assert sinks >= 0, "sinks counts first keys"
    if window is None:
        assert not sinks, "first keys that stay visible need a window that passes them"
        return 0, 0
    window = operator.index(window)
    assert window >= 1, "window counts keys, a query's own among them (None: all)"
    if not causal:
        raise NotImplementedError("a window needs causal=True")
    return min(window, 1 << 31), min(sinks, 1 << 31)


def plain_int32(x: torch.Tensor, dims: int, device: int) -> bool:
    """Is it as :func:`int32_on` would give it?"""
    return x.dtype is torch.int32 and x.dim() == dims and x.get_device() == device and x.stride()[-1] == 1


def on_device(device: int, launch, desc: bytes, *rest) -> None:
    """``launch(desc, *rest, stream)`` with the device current, on its current stream."""
    if torch._C._cuda_getDevice() == device:      # (there is a tensor on a GPU: nothing is left to be initialised)
        status = launch(desc, *rest, torch._C._cuda_getCurrentRawStream(device))
    else:
        status = _on_device(torch.device("cuda", device), lambda stream: launch(desc, *rest, stream))
    if status:
        _lib.raise_for_status(status)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(backward: bool, n_seq: int, Hq: int, Hkv: int, D: int, Tq: int, Tk: int, window: int = 0, sinks: int = 0) -> int:
    """What the library asks for, which follows from sizes alone (addresses are never dereferenced)."""
    desc = _RAGGED_DESC.pack(_lib.ABI_VERSION, _lib.DTYPE_BF16, n_seq, Hq, Hkv, D, 1, 0, Tq, Tk, 1.0, 0, *(16,) * 11, *(Hq * D, D, Hkv * D, D, Hkv * D, D, Hq * D, D), Hq * D, D, Hq * D, D,
                             Hkv * D, D, Hkv * D, D, 0)
    lib = _lib.load_library()
    return (lib.cosmos_attn_ragged_window_bwd_workspace_bytes if backward else lib.cosmos_attn_ragged_window_workspace_bytes)(desc, window, sinks)


def _fwd_as_it_is(q, k, v, cu_q, cu_k, causal, sm_scale, need_lse, rest, window, sinks):
    """:func:`ragged_fwd` of tensors that can be taken as they are, all of it looked at once: None where something is to be converted, copied or refused.  A small call is as long as what the
    host does for it: one short prompt 11 us, 17 with the checks one by one."""
    if not (q.dim() == 3 == k.dim() and q.is_cuda):
        return None
    (Tq, Hq, D), dtype, device, shape = q.shape, q.dtype, q.get_device(), k.shape
    code, (Tk, Hkv, _) = _DTYPES.get(dtype), shape
    if cu_k is None:
        cu_k = cu_q
    if (code is None or D not in HEAD_DIMS or shape[2] != D or v.shape != shape or k.dtype is not dtype or v.dtype is not dtype or k.get_device() != device or v.get_device() != device
            or Hq < 1 or Hkv < 1 or Hq % Hkv or not plain_int32(cu_q, 1, device) or not (cu_k is cu_q or plain_int32(cu_k, 1, device)) or cu_q.shape != cu_k.shape):
        return None
    (q0, q1, q2), (k0, k1, k2), (v0, v1, v2), pq, pk, pv = q.stride(), k.stride(), v.stride(), q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (q2 != 1 or k2 != 1 or v2 != 1 or (pq | pk | pv) & 15 or (q0 | q1 | k0 | k1 | v0 | v1) & 7 or min(q0, k0, v0) < D or max(q0, k0, v0) > _MOST_ROW_BYTES // 2
            or max(q1 * Hq, k1 * Hkv, v1 * Hkv) > 1 << 29):
        return None
    o = torch.empty_like(q) if q.is_contiguous() else torch.empty((Tq, Hq, D), device=q.device, dtype=dtype)
    lse = q.new_empty((Hq, Tq), dtype=torch.float32) if need_lse else None
    desc = _RAGGED_DESC.pack(_lib.ABI_VERSION, code, cu_q.shape[0] - 1, Hq, Hkv, D, 1 if causal else 0, 1, Tq, Tk, D ** -0.5 if sm_scale is None else sm_scale, 0, pq, pk, pv, cu_q.data_ptr(),
                             cu_k.data_ptr(), o.data_ptr(), 0 if lse is None else lse.data_ptr(), 0, 0, 0, 0, q0, q1, k0, k1, v0, v1, Hq * D, D, 0, 0, 0, 0, 0, 0, 0, 0, 0 if rest is None else rest.data_ptr())
    ws_bytes = _workspace_bytes(False, cu_q.shape[0] - 1, Hq, Hkv, D, Tq, Tk, window, sinks)
    workspace = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
    on_device(device, _lib.load_library().cosmos_attn_ragged_window, desc, window, sinks, 0 if workspace is None else workspace.data_ptr(), ws_bytes)
    return o, lse


def _bwd_as_it_is(q, k, v, o, lse, dout, cu_q, cu_k, causal, sm_scale, rest, window, sinks):
    """:func:`ragged_bwd`, as :func:`_fwd_as_it_is` (forward and gradients of 48 positions through autograd: 131 us, 138 with the checks one by one)."""
    if not (q.dim() == 3 == k.dim() and q.is_cuda and o.is_contiguous() and lse.is_contiguous()):
        return None
    shape, dtype, device, kv = q.shape, q.dtype, q.get_device(), k.shape
    (Tq, Hq, D), (Tk, Hkv, _), code = shape, kv, _DTYPES.get(dtype)
    if cu_k is None:
        cu_k = cu_q
    if (code is None or D not in HEAD_DIMS or kv[2] != D or v.shape != kv or o.shape != shape or dout.shape != shape or lse.shape != (Hq, Tq) or lse.dtype is not torch.float32
            or any(x.dtype is not dtype or x.get_device() != device for x in (k, v, o, dout)) or lse.get_device() != device
            or Hq < 1 or Hkv < 1 or Hq % Hkv or not plain_int32(cu_q, 1, device) or not (cu_k is cu_q or plain_int32(cu_k, 1, device)) or cu_q.shape != cu_k.shape):
        return None
    (q0, q1, q2), (k0, k1, k2), (v0, v1, v2), (g0, g1, g2) = q.stride(), k.stride(), v.stride(), dout.stride()
    pq, pk, pv, po, pg = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr()
    if (not q2 == k2 == v2 == g2 == 1 or (pq | pk | pv | po | pg) & 15 or (q0 | q1 | k0 | k1 | v0 | v1 | g0 | g1) & 7 or min(q0, k0, v0, g0) < D or max(q0, k0, v0, g0, Hq * D) > _MOST_ROW_BYTES // 2
            or max(q1 * Hq, k1 * Hkv, v1 * Hkv, g1 * Hq) > 1 << 29):
        return None
    dq, dk, dv = (torch.empty(x, device=q.device, dtype=dtype) for x in (shape, kv, kv))
    desc = _RAGGED_DESC.pack(_lib.ABI_VERSION, code, cu_q.shape[0] - 1, Hq, Hkv, D, 1 if causal else 0, 1, Tq, Tk, D ** -0.5 if sm_scale is None else sm_scale, 0, pq, pk, pv, cu_q.data_ptr(),
                             cu_k.data_ptr(), po, lse.data_ptr(), pg, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), q0, q1, k0, k1, v0, v1, Hq * D, D, g0, g1, Hq * D, D, Hkv * D, D, Hkv * D, D, 0 if rest is None else rest.data_ptr())
    ws_bytes = _workspace_bytes(True, cu_q.shape[0] - 1, Hq, Hkv, D, Tq, Tk, window, sinks)
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8)
    on_device(device, _lib.load_library().cosmos_attn_ragged_window_bwd, desc, window, sinks, workspace.data_ptr(), ws_bytes)
    return dq, dk, dv


def _check_rest(rest, q):
    assert rest.shape == q.shape and rest.dtype == q.dtype and rest.device == q.device and rest.is_contiguous() and rest.data_ptr() % 16 == 0, "rest must be a contiguous tensor like q"


def _strides(*tensors):
    return [s for x in tensors for s in ((0, 0) if x is None else x.stride()[:2])]


def _pointers(*tensors):
    return [0 if x is None else x.data_ptr() for x in tensors]


def _desc(q, k, v, o, lse, cu_q, cu_k, causal, sm_scale, fill, rest, dout=None, dq=None, dk=None, dv=None) -> bytes:
    return _RAGGED_DESC.pack(
        _lib.ABI_VERSION, _DTYPES[q.dtype], cu_q.shape[0] - 1, q.shape[1], k.shape[1], q.shape[2], 1 if causal else 0, fill, q.shape[0], k.shape[0],
        q.shape[2] ** -0.5 if sm_scale is None else sm_scale, 0, *_pointers(q, k, v, cu_q, cu_k, o, lse, dout, dq, dk, dv), *_strides(q, k, v, o, dout, dq, dk, dv), *_pointers(rest))


def ragged_fwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_q: torch.Tensor,
    cu_k: Optional[torch.Tensor] = None,
    causal: bool = False,
    sm_scale: Optional[float] = None,
    need_lse: bool = True,
    out: Optional[torch.Tensor] = None,
    rest: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(o, lse)``: ``q [Tq, Hq, D]``, ``k``, ``v`` ``[Tk, Hkv, D]``; sequence i has the rows ``cu_q[i] .. cu_q[i + 1] - 1`` of q and ``cu_k[i] ..`` of k and v
    (``cu_k`` None: the same).  ``causal``: query t of Lq sees the keys up to ``t + Lk - Lq``, with ``window`` (causal alone) the last ``window`` of these and those below ``sinks``.
    ``lse``: fp32 ``[Hq, Tq]``.

    A row that sees no key: o = 0, lse = -inf.  Rows of no sequence (before ``cu_q[0]``, from the last offset on) become zeros, and -inf; in ``out``, a tensor that is given for o, they are
    left as they are (lse is -inf there too).  Offsets that do not ascend within the tensors, or a sequence that begins before an earlier one's end: a sequence of such ``cu_q`` is none (its rows are of no
    sequence, unless another one has them), one of such ``cu_k`` has rows of NaN; the sequences before are as ever (zeros behind the last offset, say, are sequences without rows; the last offset
    again is less to look through).  ``out``
    must not overlap the inputs.
    ``rest``, a contiguous tensor like q, takes what rounding o left off, for :func:`ragged_bwd` (rows of no sequence: left as they are).  No gradients:
    :func:`attention_ragged` has them."""
    window, sinks = checked_window(window, sinks, causal)
    if rest is not None:
        _check_rest(rest, q)
    if out is None:
        made = _fwd_as_it_is(q, k, v, cu_q, cu_k, causal, sm_scale, need_lse, rest, window, sinks)
        if made is not None:
            return made
    cu_q, cu_k = _check(q, k, v, cu_q, cu_k)
    q, k, v = packed(q), packed(k), packed(v)
    if out is None:
        o = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must have q's shape, type and device"
        if not packed_ready(out):
            raise ValueError("out: rows of 16-byte steps are written in place, this view cannot be")
        o = out
    lse = torch.empty((q.shape[1], q.shape[0]), device=q.device, dtype=torch.float32) if need_lse else None
    desc = _desc(q, k, v, o, lse, cu_q, cu_k, causal, sm_scale, _lib.FILL_ALL if out is None else _lib.FILL_LSE, rest)
    lib = _lib.load_library()
    ws_bytes = lib.cosmos_attn_ragged_window_workspace_bytes(desc, window, sinks)
    workspace = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
    on_device(q.get_device(), lib.cosmos_attn_ragged_window, desc, window, sinks, 0 if workspace is None else workspace.data_ptr(), ws_bytes)
    return o, lse


def ragged_bwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    o: torch.Tensor,
    lse: torch.Tensor,
    dout: torch.Tensor,
    cu_q: torch.Tensor,
    cu_k: Optional[torch.Tensor] = None,
    causal: bool = False,
    sm_scale: Optional[float] = None,
    rest: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dq, dk, dv)`` of :func:`ragged_fwd` (of the same ``causal``, ``sm_scale``, ``window`` and ``sinks``) for the gradient ``dout`` of o, from its o and lse, and its ``rest``: without it dq and dk of sharp softmaxes, and of rows that see
    few keys, have o's rounding in them.  Rows of no sequence get zeros.  The same results every time (no atomics).  A call takes up to 400 MB of workspace from torch's allocator while it runs
    (the forward up to 200), where tiles are few enough to be cut."""
    window, sinks = checked_window(window, sinks, causal)
    if rest is not None:
        _check_rest(rest, q)
    made = _bwd_as_it_is(q, k, v, o, lse, dout, cu_q, cu_k, causal, sm_scale, rest, window, sinks)
    if made is not None:
        return made
    cu_q, cu_k = _check(q, k, v, cu_q, cu_k)
    for x, name in ((o, "o"), (dout, "dout")):
        assert x.shape == q.shape and x.dtype == q.dtype and x.device == q.device, f"{name} must have q's shape, type and device"
    assert lse.shape == (q.shape[1], q.shape[0]) and lse.dtype == torch.float32 and lse.device == q.device, "lse is the forward's, fp32 [Hq, Tq]"
    q, k, v, o, dout, lse = packed(q), packed(k), packed(v), packed(o), packed(dout), lse.contiguous()
    dq, dk, dv = (torch.empty(x.shape, device=x.device, dtype=x.dtype) for x in (q, k, v))
    desc = _desc(q, k, v, o, lse, cu_q, cu_k, causal, sm_scale, _lib.FILL_ALL, rest, dout, dq, dk, dv)
    lib = _lib.load_library()
    ws_bytes = lib.cosmos_attn_ragged_window_bwd_workspace_bytes(desc, window, sinks)
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8)
    on_device(q.get_device(), lib.cosmos_attn_ragged_window_bwd, desc, window, sinks, workspace.data_ptr(), ws_bytes)
    return dq, dk, dv


class _RaggedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, softmax_scale, window, sinks):
        rest = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        o, lse = ragged_fwd(q, k, v, cu_q, cu_k, causal=causal, sm_scale=softmax_scale, rest=rest, window=window, sinks=sinks)
        ctx.save_for_backward(q, k, v, o, lse, rest, cu_q, cu_k)
        ctx.causal, ctx.softmax_scale, ctx.window, ctx.sinks = causal, softmax_scale, window, sinks
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, o, lse, rest, cu_q, cu_k = ctx.saved_tensors
        grads = ragged_bwd(q, k, v, o, lse, dout, cu_q, cu_k, causal=ctx.causal, sm_scale=ctx.softmax_scale, rest=rest, window=ctx.window, sinks=ctx.sinks)
        return (*grads, None, None, None, None, None, None)


def attention_ragged(q, k, v, cu_q, cu_k=None, softmax_scale=None, causal=False, window=None, sinks=0):
    """Differentiable attention over packed sequences: o of :func:`ragged_fwd`, gradients by :func:`ragged_bwd`.  The offsets must not change between the two.  No tangents: forward-mode
    differentiation is refused."""
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or forward_ad._current_level >= 0:
        cu_q = int32_on(cu_q, q.device)
        return _RaggedFn.apply(q, k, v, cu_q, cu_q if cu_k is None else int32_on(cu_k, q.device), causal, softmax_scale, window, sinks)
    return ragged_fwd(q, k, v, cu_q, cu_k, causal=causal, sm_scale=softmax_scale, need_lse=False, window=window, sinks=sinks)[0]

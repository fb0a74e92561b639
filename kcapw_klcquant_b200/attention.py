"""Attention of the layer loop: whole prompts, single tokens over the paged cache, rotary append.

The reference's :class:`StreamedAttention` (streamed_attention.py:100-152) runs
one token at a time against a Python list of keys and values.  Here a batch of
sequences is one call:

* :func:`attn_prompt` -- causal attention over packed prompts of any lengths;
* :func:`attn_decode` -- one new token per sequence over the paged cache
  (:class:`~kcapw_klcquant_b200.kv_cache.PagedKvCache`), a prefix that a group
  of sequences shares read once;
* :func:`rope_append` -- rotary embedding of new tokens and their write into the
  cache,

with grouped heads, attention sinks and a sliding window as the reference has
them.  Elements are bf16 or f16, head width 64 or 128; softmax statistics are
fp32.  All math runs in the CUDA kernels of libklcmoe.so.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib
from .moe import workspace

_STATUS: dict[int, torch.Tensor] = {}
_STATUS_LOCK = threading.Lock()


def device_status(device: torch.device) -> torch.Tensor | None:
    """The device's fault word (klc_status_bytes, zeroed once).  None while a graph is being
    captured before the first eager call made it: that graph then records no faults."""
    idx = device.index
    st = _STATUS.get(idx)
    if st is None and not torch.cuda.is_current_stream_capturing():
        with _STATUS_LOCK:
            st = _STATUS.get(idx)
            if st is None:
                n = ctypes.c_size_t(0)
                _lib.check(_lib.lib().klc_status_bytes(ctypes.byref(n)))
                st = torch.zeros(n.value, dtype=torch.uint8, device=device)
                torch.cuda.current_stream(device).synchronize()  # zeroed before a call on any other stream
                _STATUS[idx] = st
    return st


def check_device_status(device: torch.device | str | int = "cuda") -> None:
    """Raise if an attention or cache kernel on ``device`` recorded a fault (offsets that leave the
    tensors, a page id that is no page, a cache out of pages) since the last check.

    Synchronises the device's current stream; faults of calls still running on
    other streams are seen by a later check.
    """
    dev = torch.device(device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    st = _STATUS.get(dev.index)
    if st is None:
        return
    with torch.cuda.device(dev):
        try:
            _lib.check(_lib.lib().klc_workspace_status(st.data_ptr(), None, None, None, _lib.stream_ptr(dev)))
        except _lib.KlcError:
            st.zero_()
            raise


def check_tensor(name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device, ndim: int) -> None:
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {tuple(t.shape)}")


def _rows(name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A [tokens, heads, D] operand the kernels can address: contiguous rows, 16-byte aligned strides."""
    check_tensor(name, t, dtype, device, 3)
    if t.numel() == 0:
        return t
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0
    for dim in (0, 1):
        if t.shape[dim] > 1:
            ok = ok and t.stride(dim) % 8 == 0 and t.stride(dim) >= t.shape[2]
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """Token and head strides in elements; a dimension of one row gets the contiguous stride."""
    d = t.shape[2]
    hs = t.stride(1) if t.shape[1] > 1 else d
    ts = t.stride(0) if t.shape[0] > 1 else t.shape[1] * max(hs, d)
    return ts, hs


def _offsets(name: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    check_tensor(name, t, torch.int32, device, 1)
    return t.contiguous()


def _sinks(sinks: torch.Tensor | None, heads: int, device: torch.device) -> torch.Tensor | None:
    if sinks is None:
        return None
    check_tensor("sinks", sinks, torch.float32, device, 1)
    if sinks.numel() != heads:
        raise ValueError(f"sinks must have {heads} elements")
    return sinks.contiguous()


def _dims(q: torch.Tensor, kv_heads: int, window: int, scale: float | None) -> _lib.KlcAttnDims:
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"attention expects bf16 or f16, got {q.dtype}")
    heads, d = int(q.shape[1]), int(q.shape[2])
    if not 0 <= int(window) < 1 << 31:
        raise ValueError("window must be >= 0 and fit 32 bits")
    return _lib.KlcAttnDims(_lib.DTYPE_CODE[q.dtype], heads, kv_heads, d, int(window), float(d ** -0.5 if scale is None else scale))


def _out(out: torch.Tensor | None, q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    check_tensor("out", out, q.dtype, q.device, 3)
    if out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    if out.numel() and _rows("out", out, q.dtype, q.device) is not out:
        raise ValueError("out must have contiguous, 16-byte aligned rows and strides of multiples of 8 elements")
    return out


def _require_cuda(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise ValueError("kcapw_klcquant_b200 runs on CUDA devices only (no CPU fallback); got a CPU tensor")
    return t.device


def attn_prompt(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    cu_seqlens_k: torch.Tensor | None = None,
    scale: float | None = None,
    window: int = 0,
    sinks: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Causal attention over whole prompts, packed: q [T, heads, D], k and v [Tk, kv_heads, D].

    Sequence ``b`` has the rows ``cu_seqlens[b]:cu_seqlens[b + 1]`` (int32 on
    the device) of q, and of k and v unless ``cu_seqlens_k`` gives them their
    own; its last query sees its last key, so with more keys than queries the
    first keys are an earlier part of the sequence.  ``window`` w > 0 limits a
    row to its last w keys; ``sinks`` fp32 [heads] adds one logit per head to
    the denominator.  q, k and v may be slices of one projection.  Rows of
    ``out`` past the last sequence are not written.  Returns out [T, heads, D]
    (and the log-sum-exp fp32 [T, heads] with ``return_lse``).
    """
    dev = _require_cuda(q)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, D]")
    dims = _dims(q, int(k.shape[1]), window, scale)
    if k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"k and v must both be [tokens, kv_heads, {q.shape[2]}], got {tuple(k.shape)} and {tuple(v.shape)}")
    cu_q = _offsets("cu_seqlens", cu_seqlens, dev)
    cu_k = cu_q if cu_seqlens_k is None else _offsets("cu_seqlens_k", cu_seqlens_k, dev)
    if cu_q.numel() < 1 or cu_q.numel() != cu_k.numel():
        raise ValueError("cu_seqlens (and cu_seqlens_k) must have batch + 1 elements")
    if cu_seqlens_k is None and k.shape[0] != q.shape[0]:
        raise ValueError("q and k have different numbers of rows: give cu_seqlens_k")
    q, k, v = _rows("q", q, q.dtype, dev), _rows("k", k, q.dtype, dev), _rows("v", v, q.dtype, dev)
    sk = _sinks(sinks, dims.heads, dev)
    o = _out(out, q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if return_lse else None
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().klc_attn_prompt(
            ctypes.byref(dims), q.data_ptr(), q.shape[0], *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v),
            k.shape[0], cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, _lib.ptr(sk), o.data_ptr(), *_strides(o),
            _lib.ptr(lse), _lib.ptr(device_status(dev)), _lib.stream_ptr(dev)))
    return (o, lse) if return_lse else o


def _workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch for one call: the stream's own, or, under capture, memory of the graph (two captured
    graphs never share it, on whichever streams they are replayed)."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return workspace(device, nbytes, _lib.stream_ptr(device))


def _pools(k_pages: torch.Tensor, v_pages: torch.Tensor, dtype: torch.dtype, device: torch.device, d: int) -> int:
    """Checks a pair of page pools [pages, kv_heads, page_size, D] and returns their common page stride."""
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        check_tensor(name, t, dtype, device, 4)
        if t.shape[3] != d:
            raise ValueError(f"{name} must be [pages, kv_heads, page_size, {d}], got {tuple(t.shape)}")
        if t.shape[1:].numel() and not t[:1].is_contiguous():
            raise ValueError(f"{name}: a page must be contiguous")
    if k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    if k_pages.shape[0] < 1:
        raise ValueError("the pools have no pages")
    if k_pages.shape[0] == 1:
        return k_pages.shape[1:].numel()
    if k_pages.stride(0) != v_pages.stride(0):
        raise ValueError("k_pages and v_pages must have the same page stride")
    return k_pages.stride(0)


def _table(block_table: torch.Tensor, device: torch.device) -> tuple[torch.Tensor, int]:
    check_tensor("block_table", block_table, torch.int32, device, 2)
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table rows must be contiguous")
    if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table rows overlap")
    return block_table, (block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1])


def attn_decode(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lens: torch.Tensor,
    *,
    scale: float | None = None,
    window: int = 0,
    sinks: torch.Tensor | None = None,
    group_starts: torch.Tensor | None = None,
    prefix_lens: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Attention of one token per sequence over its pages: q [B, heads, D].

    ``k_pages`` and ``v_pages`` are pools [pages, kv_heads, page_size, D]
    (page_size 16, 32, 64 or 128); row b sees the ``lens[b]`` keys of the pages
    ``block_table[b]`` (int32 [B, width]), the own one among them, or the last
    ``window`` of them.  ``sinks`` as for :func:`attn_prompt`.  With
    ``group_starts`` (int32 [G + 1]) and ``prefix_lens`` (int32 [G], multiples of
    page_size) the rows ``group_starts[g]:group_starts[g + 1]`` share the pages of
    their first ``prefix_lens[g]`` keys, which are then read once for all of them,
    through the first row's table.  At most 4096 rows.  Lengths stay on the device: a captured
    call serves other lengths on replay.  Returns out [B, heads, D] (and the
    log-sum-exp fp32 [B, heads] with ``return_lse``).
    """
    dev = _require_cuda(q)
    if q.dim() != 3 or k_pages.dim() != 4:
        raise ValueError("q must be [batch, heads, D] and the pools [pages, kv_heads, page_size, D]")
    dims = _dims(q, int(k_pages.shape[1]), window, scale)
    page_stride = _pools(k_pages, v_pages, q.dtype, dev, int(q.shape[2]))
    B = int(q.shape[0])
    table, table_stride = _table(block_table, dev)
    ln = _offsets("lens", lens, dev)
    if table.shape[0] != B or ln.numel() != B:
        raise ValueError(f"block_table and lens must have {B} rows")
    if (group_starts is None) != (prefix_lens is None):
        raise ValueError("group_starts and prefix_lens go together")
    gs = None if group_starts is None else _offsets("group_starts", group_starts, dev)
    pl = None if prefix_lens is None else _offsets("prefix_lens", prefix_lens, dev)
    groups = 0 if pl is None else pl.numel()
    if gs is not None and gs.numel() != groups + 1:
        raise ValueError("group_starts must have one element more than prefix_lens")
    q = _rows("q", q, q.dtype, dev)
    sk = _sinks(sinks, dims.heads, dev)
    o = _out(out, q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if return_lse else None
    with torch.cuda.device(dev):
        n = ctypes.c_size_t(0)
        _lib.check(_lib.lib().klc_attn_decode_workspace_size(ctypes.byref(dims), B, groups, ctypes.byref(n)))
        ws = _workspace(dev, n.value)
        _lib.check(_lib.lib().klc_attn_decode(
            ctypes.byref(dims), q.data_ptr(), *_strides(q), k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0],
            int(k_pages.shape[2]), page_stride, table.data_ptr(), table.shape[1], table_stride, ln.data_ptr(), B, _lib.ptr(gs),
            _lib.ptr(pl), groups, _lib.ptr(sk), o.data_ptr(), *_strides(o), _lib.ptr(lse), ws.data_ptr(), ws.numel(),
            _lib.ptr(device_status(dev)), _lib.stream_ptr(dev)))
    return (o, lse) if return_lse else o


def rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    rows: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    *,
    out: torch.Tensor | None = None,
    return_k: bool = False,
):
    """Rotary embedding of q [T, heads, D] and k [T, kv_heads, D], and the write of k and v into the cache.

    Token t is key ``positions[t]`` of sequence ``rows[t]`` (int32 on the device;
    row -1: padding, nothing is written); its page must be reserved.  ``cos`` and
    ``sin`` are fp32 [max_pos, D / 2]; the halves of a head's row are rotated
    against each other, in fp32, rounded once.  Returns the rotated queries
    (``out``, which may be q), and with ``return_k`` the rotated keys [T, kv_heads, D] too.
    """
    dev = _require_cuda(q)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, D]")
    T, d = int(q.shape[0]), int(q.shape[2])
    dims = _dims(q, int(k.shape[1]), 0, 1.0)
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != d:
        raise ValueError(f"k and v must both be [{T}, kv_heads, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    page_stride = _pools(k_pages, v_pages, q.dtype, dev, d)
    if k_pages.shape[1] != k.shape[1]:
        raise ValueError(f"the pools have {k_pages.shape[1]} key heads, k has {k.shape[1]}")
    for name, t in (("cos", cos), ("sin", sin)):
        check_tensor(name, t, torch.float32, dev, 2)
        if t.shape[1] != d // 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [max_pos, {d // 2}]")
    if cos.shape != sin.shape:
        raise ValueError("cos and sin must have the same shape")
    table, table_stride = _table(block_table, dev)
    pos, rw = _offsets("positions", positions, dev), _offsets("rows", rows, dev)
    if pos.numel() != T or rw.numel() != T:
        raise ValueError(f"positions and rows must have {T} elements")
    q, k, v = _rows("q", q, q.dtype, dev), _rows("k", k, q.dtype, dev), _rows("v", v, q.dtype, dev)
    o = _out(out, q)
    ko = torch.empty(k.shape, dtype=k.dtype, device=dev) if return_k else None
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().klc_rope_append(
            ctypes.byref(dims), q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), cos.data_ptr(),
            sin.data_ptr(), cos.shape[0], pos.data_ptr(), rw.data_ptr(), T, o.data_ptr(), *_strides(o), _lib.ptr(ko),
            *(_strides(ko) if ko is not None else (0, 0)), k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0],
            int(k_pages.shape[2]), page_stride, table.data_ptr(), table.shape[0], table.shape[1], table_stride,
            _lib.ptr(device_status(dev)), _lib.stream_ptr(dev)))
    return (o, ko) if return_k else o

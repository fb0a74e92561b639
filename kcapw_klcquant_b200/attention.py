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
import functools
import math
import threading

import torch

from . import _lib
from .moe import as_bf16

# the current stream of a device as an integer, without making a Stream object for it where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _lib.stream_ptr)

_STATUS: dict[int, torch.Tensor] = {}
_STATUS_LOCK = threading.Lock()


def device_status(index: int) -> torch.Tensor | None:
    """The fault word of CUDA device ``index`` (klc_status_bytes, zeroed once).  None while a graph is being
    captured before the first eager call made it: that graph then records no faults."""
    st = _STATUS.get(index)
    if st is None and not torch.cuda.is_current_stream_capturing():
        with _STATUS_LOCK:
            st = _STATUS.get(index)
            if st is None:
                n = ctypes.c_size_t(0)
                _lib.check(_lib.lib().klc_status_bytes(ctypes.byref(n)))
                st = torch.zeros(n.value, dtype=torch.uint8, device=torch.device("cuda", index))
                torch.cuda.current_stream(index).synchronize()  # zeroed before a call on any other stream
                _STATUS[index] = st
    return st


def check_device_status(device: torch.device | str | int = "cuda") -> None:
    """Raise if an attention or cache kernel on ``device`` recorded a fault (offsets that leave the
    tensors, a page id that is no page, a cache out of pages) since the last check.

    Synchronises the device's current stream; faults of calls still running on
    other streams are seen by a later check.
    """
    dev = torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    st = _STATUS.get(index)
    if st is None:
        return
    with on_device(index) as stream:
        try:
            _lib.check(_lib.lib().klc_workspace_status(st.data_ptr(), None, None, None, stream))
        except _lib.KlcError:
            st.zero_()
            raise


def check_tensor(name: str, t: torch.Tensor, dtype: torch.dtype, index: int, ndim: int) -> None:
    """``t`` has the dtype and number of dimensions and is on CUDA device ``index``."""
    if t.get_device() != index or t.dtype is not dtype or t.dim() != ndim:
        raise ValueError(f"{name} must be {dtype} with {ndim} dimensions on cuda:{index}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _rows(name: str, t: torch.Tensor, dtype: torch.dtype, index: int) -> tuple[torch.Tensor, int, int, int]:
    """A [tokens, heads, D] operand as the kernels address it: (tensor, address, token stride, head stride).

    Rows are contiguous and 16-byte aligned, strides multiples of 8 elements; anything else is copied.  A
    dimension of one row gets a contiguous stride.
    """
    check_tensor(name, t, dtype, index, 3)
    n, h, d = t.shape
    ts, hs, one = t.stride()
    if h == 1:
        hs = d
    if n == 1:
        ts = h * max(hs, d)
    ptr = t.data_ptr()
    if (one != 1 or ptr & 15 or ts & 7 or hs & 7 or ts < d or hs < d) and t.numel():
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.data_ptr(), h * d, d
    return t, ptr, ts, hs


def _ints(name: str, t: torch.Tensor, index: int) -> torch.Tensor:
    check_tensor(name, t, torch.int32, index, 1)
    return t if t.is_contiguous() else t.contiguous()


def _sinks(sinks: torch.Tensor | None, heads: int, index: int) -> torch.Tensor | None:
    if sinks is None:
        return None
    check_tensor("sinks", sinks, torch.float32, index, 1)
    if sinks.shape[0] != heads:
        raise ValueError(f"sinks must have {heads} elements")
    return sinks if sinks.is_contiguous() else sinks.contiguous()


@functools.lru_cache(maxsize=256)
def _dims_of(code: int, heads: int, kv_heads: int, d: int, window: int, scale: float) -> _lib.KlcAttnDims:
    return _lib.KlcAttnDims(code, heads, kv_heads, d, window, scale)


def _dims(q: torch.Tensor, kv_heads: int, window: int, scale: float | None) -> _lib.KlcAttnDims:
    code = _lib.DTYPE_CODE.get(q.dtype)
    if code is None or q.dtype is torch.float32:
        raise ValueError(f"attention expects bf16 or f16, got {q.dtype}")
    if not 0 <= window < 1 << 31:
        raise ValueError("window must be >= 0 and fit 32 bits")
    _, heads, d = q.shape
    return _dims_of(code, heads, kv_heads, d, window, d ** -0.5 if scale is None else float(scale))


def _out(out: torch.Tensor | None, q: torch.Tensor, index: int) -> tuple[torch.Tensor, int, int, int]:
    if out is None:
        out = torch.empty_like(q)  # (half the time of empty; contiguous unless q's heads lie outside its tokens)
        if not out.is_contiguous():
            out = q.new_empty(q.shape)
        _, h, d = q.shape
        return out, out.data_ptr(), h * d, d
    if out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    got = _rows("out", out, q.dtype, index)
    if got[0] is not out:
        raise ValueError("out must have contiguous, 16-byte aligned rows and strides of multiples of 8 elements")
    return got


def _device_of(q: torch.Tensor) -> int:
    if not q.is_cuda:
        raise ValueError("kcapw_klcquant_b200 runs on CUDA devices only (no CPU fallback); got a CPU tensor")
    return q.get_device()


class on_device:
    """``torch.cuda.device`` that costs nothing when the device is current already; gives the device's current stream."""

    __slots__ = ("index", "guard")

    def __init__(self, index: int):
        self.index = index
        self.guard = None

    def __enter__(self) -> int:
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return _raw_stream(self.index)

    def __exit__(self, *exc) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


@functools.lru_cache(maxsize=256)
def _decode_bytes(dtype: int, heads: int, kv_heads: int, d: int, batch: int, groups: int, device: int) -> int:
    """Workspace of a decode call of these sizes (asked of the library once per set of sizes)."""
    n = ctypes.c_size_t(0)
    dims = _lib.KlcAttnDims(dtype, heads, kv_heads, d, 0, 1.0)
    _lib.check(_lib.lib().klc_attn_decode_workspace_size(ctypes.byref(dims), batch, groups, ctypes.byref(n)))
    return n.value


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
    ``out`` (which may be q) past the last sequence are not written.  Returns out [T, heads, D]
    (and the log-sum-exp fp32 [T, heads] with ``return_lse``).
    """
    dev = _device_of(q)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, D]")
    T, _, d = q.shape
    Tk, kv_heads, dk = k.shape
    dims = _dims(q, kv_heads, window, scale)
    if k.shape != v.shape or dk != d:
        raise ValueError(f"k and v must both be [tokens, kv_heads, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    cu_q = _ints("cu_seqlens", cu_seqlens, dev)
    cu_k = cu_q if cu_seqlens_k is None else _ints("cu_seqlens_k", cu_seqlens_k, dev)
    batch = cu_q.shape[0] - 1
    if batch < 0 or cu_k.shape[0] != batch + 1:
        raise ValueError("cu_seqlens (and cu_seqlens_k) must have batch + 1 elements")
    if cu_seqlens_k is None and Tk != T:
        raise ValueError("q and k have different numbers of rows: give cu_seqlens_k")
    q, *qa = _rows("q", q, q.dtype, dev)
    k, *ka = _rows("k", k, q.dtype, dev)
    v, *va = _rows("v", v, q.dtype, dev)
    sk = _sinks(sinks, dims.heads, dev)
    o, *oa = _out(out, q, dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    with on_device(dev) as stream:
        _lib.check(_lib.lib().klc_attn_prompt(
            ctypes.byref(dims), qa[0], T, qa[1], qa[2], *ka, *va, Tk, cu_q.data_ptr(), cu_k.data_ptr(), batch, _lib.ptr(sk), *oa,
            _lib.ptr(lse), _lib.ptr(device_status(dev)), stream))
    return (o, lse) if return_lse else o


class _Scratch:
    """Scratch of the calls on one stream.  ``lock`` is held while a call is launched: its kernels follow each other in the
    stream without another thread's call, on the same scratch, between them."""

    __slots__ = ("lock", "buf")

    def __init__(self):
        self.lock = threading.Lock()
        self.buf = None

    def get(self, nbytes: int, device: torch.device) -> torch.Tensor:
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        return self.buf


# by (device, stream), apart from the MoE workspaces: those begin with a fault word that is still to be read
_SCRATCH: dict[tuple[int, int], _Scratch] = {}


def _scratch(index: int, stream: int) -> _Scratch:
    """The stream's scratch, or, under capture, one of the call's own in the graph's memory (two captured
    graphs never share it, on whichever streams they are replayed)."""
    if torch.cuda.is_current_stream_capturing():
        return _Scratch()
    key = (index, stream)
    return _SCRATCH.get(key) or _SCRATCH.setdefault(key, _Scratch())


def _pools(k_pages: torch.Tensor, v_pages: torch.Tensor, dtype: torch.dtype, index: int, d: int) -> tuple[int, int]:
    """Checks a pair of page pools [pages, kv_heads, page_size, D]; (page size, common page stride)."""
    check_tensor("k_pages", k_pages, dtype, index, 4)
    check_tensor("v_pages", v_pages, dtype, index, 4)
    shape, stride = k_pages.shape, k_pages.stride()
    pages, heads, ps, width = shape
    if v_pages.shape != shape or width != d or pages < 1:
        raise ValueError(f"k_pages and v_pages must both be [pages, kv_heads, page_size, {d}], got {tuple(shape)} and {tuple(v_pages.shape)}")
    want = (ps * d, d, 1)
    if (stride[1:] != want or v_pages.stride()[1:] != want) and not (k_pages[0].is_contiguous() and v_pages[0].is_contiguous()):
        raise ValueError("k_pages and v_pages: a page must be contiguous")
    if pages == 1:
        return ps, heads * ps * d
    if stride[0] != v_pages.stride(0):
        raise ValueError("k_pages and v_pages must have the same page stride")
    return ps, stride[0]


def _table(block_table: torch.Tensor, index: int) -> tuple[int, int, int]:
    """Checks a page table; (rows, width, row stride)."""
    check_tensor("block_table", block_table, torch.int32, index, 2)
    (rows, width), (stride, one) = block_table.shape, block_table.stride()
    if one != 1 and width > 1:
        raise ValueError("block_table rows must be contiguous")
    if rows <= 1:
        stride = width
    if stride < width:
        raise ValueError("block_table rows overlap")
    return rows, width, stride


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
    dev = _device_of(q)
    if q.dim() != 3 or k_pages.dim() != 4:
        raise ValueError("q must be [batch, heads, D] and the pools [pages, kv_heads, page_size, D]")
    B, _, d = q.shape
    pages, kv_heads = k_pages.shape[:2]
    dims = _dims(q, kv_heads, window, scale)
    ps, page_stride = _pools(k_pages, v_pages, q.dtype, dev, d)
    rows, width, table_stride = _table(block_table, dev)
    ln = _ints("lens", lens, dev)
    if rows != B or ln.shape[0] != B:
        raise ValueError(f"block_table and lens must have {B} rows")
    gs = pl = None
    groups = 0
    if group_starts is not None or prefix_lens is not None:
        if group_starts is None or prefix_lens is None:
            raise ValueError("group_starts and prefix_lens go together")
        gs, pl = _ints("group_starts", group_starts, dev), _ints("prefix_lens", prefix_lens, dev)
        groups = pl.shape[0]
        if gs.shape[0] != groups + 1:
            raise ValueError("group_starts must have one element more than prefix_lens")
    q, *qa = _rows("q", q, q.dtype, dev)
    sk = _sinks(sinks, dims.heads, dev)
    o, *oa = _out(out, q, dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    L = _lib.lib()
    with on_device(dev) as stream:
        nbytes = _decode_bytes(dims.dtype, dims.heads, kv_heads, d, B, groups, dev)
        status = device_status(dev)
        scratch = _scratch(dev, stream)
        with scratch.lock:
            ws = scratch.get(nbytes, q.device)
            _lib.check(L.klc_attn_decode(
                ctypes.byref(dims), *qa, k_pages.data_ptr(), v_pages.data_ptr(), pages, ps, page_stride, block_table.data_ptr(), width,
                table_stride, ln.data_ptr(), B, _lib.ptr(gs), _lib.ptr(pl), groups, _lib.ptr(sk), *oa, _lib.ptr(lse), ws.data_ptr(),
                ws.numel(), _lib.ptr(status), stream))
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
    row -1: padding, nothing is written, ``out`` included); its page must be reserved,
    and no other token of the call may have the same row and position.  ``cos`` and
    ``sin`` are fp32 [max_pos, D / 2]; the halves of a head's row are rotated
    against each other, in fp32, rounded once.  Returns the rotated queries
    (``out``, which may be q), and with ``return_k`` the rotated keys [T, kv_heads, D] too.
    """
    dev = _device_of(q)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, D]")
    T, _, d = q.shape
    kv_heads = k.shape[1]
    dims = _dims(q, kv_heads, 0, 1.0)
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != d:
        raise ValueError(f"k and v must both be [{T}, kv_heads, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    ps, page_stride = _pools(k_pages, v_pages, q.dtype, dev, d)
    if k_pages.shape[1] != kv_heads:
        raise ValueError(f"the pools have {k_pages.shape[1]} key heads, k has {kv_heads}")
    check_tensor("cos", cos, torch.float32, dev, 2)
    check_tensor("sin", sin, torch.float32, dev, 2)
    max_pos, half = cos.shape
    if cos.shape != sin.shape or 2 * half != d or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"cos and sin must both be contiguous [max_pos, {d // 2}], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    rows_n, width, table_stride = _table(block_table, dev)
    pos, rw = _ints("positions", positions, dev), _ints("rows", rows, dev)
    if pos.shape[0] != T or rw.shape[0] != T:
        raise ValueError(f"positions and rows must have {T} elements")
    q, *qa = _rows("q", q, q.dtype, dev)
    k, *ka = _rows("k", k, q.dtype, dev)
    v, *va = _rows("v", v, q.dtype, dev)
    o, *oa = _out(out, q, dev)
    ko, koa = None, (None, 0, 0)
    if return_k:
        ko = k.new_empty(k.shape)
        koa = _rows("k_out", ko, q.dtype, dev)[1:]
    with on_device(dev) as stream:
        _lib.check(_lib.lib().klc_rope_append(
            ctypes.byref(dims), *qa, *ka, *va, cos.data_ptr(), sin.data_ptr(), max_pos, pos.data_ptr(), rw.data_ptr(), T, *oa, *koa,
            k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0], ps, page_stride, block_table.data_ptr(), rows_n, width,
            table_stride, _lib.ptr(device_status(dev)), stream))
    return (o, ko) if return_k else o


class AttentionLayer:
    """The attention half of a decoder layer: q, k and v projections, rotary embedding, attention, output projection.

    ``qkv_weight`` bf16 [(heads + 2 kv_heads) * D, H] holds the q, k and v rows one after the other, ``o_weight`` [H, heads * D];
    biases and ``sinks`` [heads] may be None.  ``window`` as for :func:`attn_prompt`.  The projections are plain library
    products (torch.nn.functional.linear).
    """

    def __init__(self, qkv_weight: torch.Tensor, o_weight: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                 qkv_bias: torch.Tensor | None = None, o_bias: torch.Tensor | None = None, sinks: torch.Tensor | None = None,
                 window: int = 0, scale: float | None = None):
        rows = (heads + 2 * kv_heads) * head_dim
        if qkv_weight.dim() != 2 or qkv_weight.shape[0] != rows:
            raise ValueError(f"qkv_weight must be [{rows}, hidden], got {tuple(qkv_weight.shape)}")
        if o_weight.shape != (qkv_weight.shape[1], heads * head_dim):
            raise ValueError(f"o_weight must be [{qkv_weight.shape[1]}, {heads * head_dim}], got {tuple(o_weight.shape)}")
        if kv_heads < 1 or heads < kv_heads or heads % kv_heads != 0 or heads // kv_heads > 64 or head_dim not in (64, 128):
            raise ValueError("heads must be a multiple of kv_heads (at most 64 times), head_dim 64 or 128")
        if not 0 <= window < 1 << 31 or not (scale is None or 0 < scale < math.inf):
            raise ValueError("window must be >= 0 and fit 32 bits, scale finite and > 0")
        for name, b, n in (("qkv_bias", qkv_bias, rows), ("o_bias", o_bias, qkv_weight.shape[1]), ("sinks", sinks, heads)):
            if b is not None and b.shape != (n,):
                raise ValueError(f"{name} must be [{n}], got {tuple(b.shape)}")
        dev = qkv_weight.device
        self.heads, self.kv_heads, self.head_dim, self.window, self.scale = int(heads), int(kv_heads), int(head_dim), int(window), scale
        self.qkv_weight, self.o_weight = as_bf16(qkv_weight, dev), as_bf16(o_weight, dev)
        self.qkv_bias = None if qkv_bias is None else as_bf16(qkv_bias, dev)
        self.o_bias = None if o_bias is None else as_bf16(o_bias, dev)
        self.sinks = None if sinks is None else sinks.to(device=dev, dtype=torch.float32).contiguous()

    @classmethod
    def from_tensors(cls, layer_idx: int, tensors: dict[str, torch.Tensor], device, heads: int, kv_heads: int, head_dim: int,
                     window: int = 0) -> "AttentionLayer":
        """Build from checkpoint-named tensors (``model.layers.{L}.self_attn.*``; biases and sinks optional)."""
        p = f"model.layers.{layer_idx}.self_attn"
        dev = torch.device(device)

        def get(name):
            t = tensors.get(f"{p}.{name}")
            return None if t is None else t.to(dev)

        parts = [get(f"{n}_proj.bias") for n in "qkv"]
        if any(b is None for b in parts) and not all(b is None for b in parts):
            raise ValueError("q, k and v must all have a bias or none")
        weights = [tensors[f"{p}.{n}_proj.weight"].to(dev) for n in "qkvo"]
        return cls(torch.cat(weights[:3]), weights[3], heads, kv_heads, head_dim,
                   qkv_bias=None if parts[0] is None else torch.cat(parts), o_bias=get("o_proj.bias"), sinks=get("sinks"), window=window)

    def check_cache(self, cache, rope: tuple[torch.Tensor, torch.Tensor]) -> None:
        """Raise unless the pages of ``cache`` and the rotary tables fit this layer."""
        dev, pool = self.qkv_weight.device, cache.pool
        want = (self.kv_heads, self.head_dim)
        if pool.dtype is not torch.bfloat16 or (pool.shape[3], pool.shape[5]) != want or pool.device != dev:
            raise ValueError(f"the layer writes bf16 keys of {want[0]} heads of {want[1]} on {dev}, the cache holds {pool.dtype} "
                             f"of {pool.shape[3]} heads of {pool.shape[5]} on {pool.device}")
        if len(rope) != 2 or rope[0].shape != rope[1].shape or rope[0].dim() != 2 or 2 * rope[0].shape[1] != self.head_dim:
            raise ValueError(f"the rotary tables must both be [max_pos, {self.head_dim // 2}]")

    def project(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q [T, heads, D], k and v [T, kv_heads, D] of x bf16 [T, H]: slices of one product."""
        h, g = self.heads, self.kv_heads
        qkv = torch.nn.functional.linear(x, self.qkv_weight, self.qkv_bias).view(x.shape[0], h + 2 * g, self.head_dim)
        return qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]

    def output(self, o: torch.Tensor) -> torch.Tensor:
        return torch.nn.functional.linear(o.reshape(o.shape[0], -1), self.o_weight, self.o_bias)

    def prompt(self, x: torch.Tensor, cache, layer: int, rope: tuple[torch.Tensor, torch.Tensor], cu_seqlens: torch.Tensor,
               positions: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        """Whole prompts (packed tokens x [T, H], reserved in ``cache``): writes their keys and values, returns [T, H]."""
        q, k, v = self.project(x)
        q, k = rope_append(q, k, v, *rope, positions, rows, cache.k(layer), cache.v(layer), cache.block_table, return_k=True)
        return self.output(attn_prompt(q, k, v, cu_seqlens, window=self.window, sinks=self.sinks, scale=self.scale))

    def decode(self, x: torch.Tensor, cache, layer: int, rope: tuple[torch.Tensor, torch.Tensor], positions: torch.Tensor,
               rows: torch.Tensor, group_starts: torch.Tensor | None = None, prefix_lens: torch.Tensor | None = None) -> torch.Tensor:
        """One token for every row of ``cache`` (x [rows, H], token r that of row r, reserved): writes its key and value, returns
        [rows, H].  ``rows[r]`` is r, or -1 for a row that sits out (nothing is written, its output means nothing)."""
        q, k, v = self.project(x)
        q = rope_append(q, k, v, *rope, positions, rows, cache.k(layer), cache.v(layer), cache.block_table)
        o = attn_decode(q, cache.k(layer), cache.v(layer), cache.block_table, cache.lens, window=self.window, sinks=self.sinks,
                        scale=self.scale, group_starts=group_starts, prefix_lens=prefix_lens)
        return self.output(o)

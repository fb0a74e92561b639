"""The paged key/value cache of the attention layers.

The reference keeps a Python list of tensors per layer (KVCacheManager,
kv_cache_manager.py:23-113).  Here the keys and values of all layers live in one
pool of fixed-size pages, and which page belongs to which sequence is device
state (page tables, lengths, reference counts) that only kernels change: no
call waits for the host, and a captured decode step can grow its sequences.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib
from .attention import check_device_status, check_tensor, device_status, on_device


class PagedKvCache:
    """Pages of keys and values for ``rows`` sequences over ``layers`` layers.

    ``pool`` [layers, 2, pages, kv_heads, page_size, D] holds keys (0) and values
    (1); ``block_table`` int32 [rows, row_pages] the page ids of each sequence
    (-1: none), ``lens`` int32 [rows] its number of keys, ``refs`` int32 [pages]
    how many sequences hold a page.  New pages are the free ones with the lowest
    ids, in the order of the requests.  Requests that cannot be met leave their
    row as it was and are reported by :meth:`check`; when the free pages do not
    suffice for one, the later ones of the call that need pages are refused with
    it (small requests do not overtake a large one).  The methods take int32
    tensors on the device; calls on one cache are ordered on one stream, from
    whichever threads they come.
    """

    def __init__(self, *, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, rows: int, row_pages: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the cache holds bf16 or f16, got {dtype}")
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size must be 16, 32, 64 or 128")
        if min(layers, pages, kv_heads, rows, row_pages) < 1 or head_dim not in (64, 128):
            raise ValueError("layers, pages, kv_heads, rows and row_pages must be positive, head_dim 64 or 128")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("kcapw_klcquant_b200 runs on CUDA devices only (no CPU fallback)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device, self.page_size = dev, int(page_size)
        self.pool = torch.zeros((layers, 2, pages, kv_heads, page_size, head_dim), dtype=dtype, device=dev)
        self.block_table = torch.full((rows, row_pages), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.live = torch.zeros(1, dtype=torch.int32, device=dev)
        self._c = _lib.KlcKvCache(
            self.pool.data_ptr(), 2 * layers, self.pool.stride(1) * self.pool.element_size(),
            self.pool.stride(2) * self.pool.element_size(), pages, self.refs.data_ptr(), self.block_table.data_ptr(), row_pages,
            row_pages, self.lens.data_ptr(), rows, page_size, _lib.ptr(device_status(dev.index)))
        n = ctypes.c_size_t(0)
        _lib.check(_lib.lib().klc_kv_workspace_size(ctypes.byref(self._c), ctypes.byref(n)))
        self._ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
        self._lock = threading.Lock()  # a call's kernels follow each other in the stream: they share _ws with other calls'

    @property
    def rows(self) -> int:
        return int(self.lens.numel())

    def k(self, layer: int) -> torch.Tensor:
        """The key pages [pages, kv_heads, page_size, D] of a layer."""
        return self.pool[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 1]

    def _list(self, name: str, t: torch.Tensor) -> torch.Tensor:
        check_tensor(name, t, torch.int32, self.device.index, 1)
        return t if t.is_contiguous() else t.contiguous()

    def _call(self, fn, *args) -> None:
        with on_device(self.device.index) as stream, self._lock:
            _lib.check(fn(ctypes.byref(self._c), *args, stream))

    def reserve(self, add: torch.Tensor) -> None:
        """Every row grows by ``add[row]`` keys: takes the pages it needs and advances ``lens``."""
        add = self._list("add", add)
        if add.numel() != self.rows:
            raise ValueError(f"add must have {self.rows} elements")
        self._call(_lib.lib().klc_kv_reserve, add.data_ptr(), self._ws.data_ptr(), self._ws.numel())

    def fork(self, parents: torch.Tensor, children: torch.Tensor, copy: bool = False) -> None:
        """Row ``children[i]`` (empty, listed once) becomes row ``parents[i]``: its full pages are shared and a
        partial last page copied, or all pages copied with ``copy``."""
        parents, children = self._list("parents", parents), self._list("children", children)
        if parents.numel() != children.numel():
            raise ValueError("parents and children must have the same length")
        self._call(_lib.lib().klc_kv_fork, parents.data_ptr(), children.data_ptr(), parents.numel(), int(bool(copy)),
                   self._ws.data_ptr(), self._ws.numel())

    def free(self, rows: torch.Tensor) -> None:
        """The listed rows become empty; pages nobody else holds become free."""
        rows = self._list("rows", rows)
        self._call(_lib.lib().klc_kv_free, rows.data_ptr(), rows.numel())

    def compact(self) -> torch.Tensor:
        """Moves live pages to the front of the pool; returns their number (int32 [1] on the device)."""
        self._call(_lib.lib().klc_kv_compact, self.live.data_ptr(), self._ws.data_ptr(), self._ws.numel())
        return self.live

    def snapshot(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The page tables, lengths and reference counts (copies; not the pages' contents): with :meth:`restore`,
        sequences go back to an earlier length (KVCacheManager.snapshot, kv_cache_manager.py:80-91)."""
        return self.block_table.clone(), self.lens.clone(), self.refs.clone()

    def restore(self, state: tuple[torch.Tensor, torch.Tensor, torch.Tensor]) -> None:
        """Back to a :meth:`snapshot`.  Keys up to the restored lengths must still be in their pages: nothing was freed and
        handed out again, or compacted, since."""
        for mine, theirs in zip((self.block_table, self.lens, self.refs), state):
            mine.copy_(theirs)

    def check(self) -> None:
        """Raise if a call could not serve a request (synchronises)."""
        check_device_status(self.device)

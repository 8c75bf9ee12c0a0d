"""A K/V cache of many sequences in pages of one pool, and the attention over it.

    cache = PagedCache.create(layers=6, pages=4096, page_size=16, kv_heads=4, head_dim=256, slots=64,
                              max_length=8192)
    cache.reserve(counts)                          # the sequences grow by counts[i] positions
    for layer in range(6):
        cache.append(k, v, starts, layer=layer)    # their K/V rows
        out = cache.prefill(q, starts, layer=layer)    # many new tokens per sequence, or
        out = cache.decode(q, layer=layer)             # one
    cache.fork(src, dst); cache.free(slots); cache.compact()
    cache.check()                                  # what the device-side checks found

Calls forward device pointers to librta_cuda.so (include/rta.h, section 1c), are
asynchronous on torch's current stream and never wait for the device, so a
serving step can be captured as a CUDA graph; only check() synchronises.  A
cache's calls share one workspace: order them on one stream.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import BF16, F16, F32, RtaError, check

_FORMAT = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}


def _ints(t: torch.Tensor, name: str, device: torch.device, n: int | None = None) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or t.dim() != 1:
        raise ValueError(f"{name} must be a contiguous 1-d int32 tensor on {device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} has {t.shape[0]} entries, {n} expected")
    return t


class PageMap:
    """Which page holds which positions: refs [pages], table [slots, width] (-1: unused) and lengths [slots], int32."""

    def __init__(self, refs: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor):
        for t, dims, name in ((refs, 1, "refs"), (table, 2, "table"), (lengths, 1, "lengths")):
            if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.dim() != dims:
                raise ValueError(f"{name} must be a contiguous {dims}-d int32 CUDA tensor")
            if t.device != refs.device:
                raise ValueError("refs, table and lengths must be on one device")
        if table.shape[0] != lengths.shape[0]:
            raise ValueError("table and lengths differ in slots")
        self.refs, self.table, self.lengths = refs, table, lengths
        self._c = _lib.PageMapC(refs.data_ptr(), table.data_ptr(), lengths.data_ptr(), table.shape[0], table.shape[1])
        self._at = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, pages: int, slots: int, width: int, device="cuda") -> "PageMap":
        """No sequence holds anything: every page free, every table entry -1."""
        return cls(torch.zeros(pages, dtype=torch.int32, device=device),
                   torch.full((slots, width), -1, dtype=torch.int32, device=device),
                   torch.zeros(slots, dtype=torch.int32, device=device))

    def clone(self) -> "PageMap":
        return PageMap(self.refs.clone(), self.table.clone(), self.lengths.clone())


class PagedCache:
    """K and V pools [layers, pages, kv_heads, page_size, head_dim] (fp16 or bf16, any strides that keep head_dim
    contiguous, the same for both), a PageMap and the workspace of their calls."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, map: PageMap):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("k and v must be fp16 or bf16 [layers, pages, kv_heads, page_size, head_dim] of one shape")
        if not k.is_cuda or k.device != v.device or k.device != map.refs.device:
            raise ValueError("k, v and the map must be on one CUDA device")
        strides = [0 if n == 1 else s for n, s in zip(k.shape, k.stride())]  # a stride nothing steps by
        if strides != [0 if n == 1 else s for n, s in zip(v.shape, v.stride())] or k.stride(4) != 1 or v.stride(4) != 1:
            raise ValueError("k and v must have the same strides, head_dim contiguous")
        if map.refs.shape[0] != k.shape[1]:
            raise ValueError("refs has an entry per page of the pool")
        self.k, self.v, self.map = k, v, map
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.device, self.dtype = k.device, k.dtype
        self._lib = _lib.load()
        self._c = _lib.PagePoolC(k.data_ptr(), v.data_ptr(), _FORMAT[k.dtype], self.layers, self.pages, self.page_size,
                                 self.kv_heads, self.head_dim, *strides[:4])
        self._at = ctypes.addressof(self._c)
        n = self._lib.rta_paged_workspace_bytes(self._at, map._at)
        if n == 0:
            raise ValueError("head_dim must be 64, 128 or 256, page_size 1 .. 65536, the pool's strides multiples of 8 "
                             "elements and its rows 16-byte aligned")
        self.workspace = torch.zeros(n, dtype=torch.uint8, device=self.device)
        self._ws, self._ws_bytes = self.workspace.data_ptr(), n

    @classmethod
    def create(cls, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int,
               max_length: int, dtype=torch.float16, device="cuda", order: str = "heads") -> "PagedCache":
        """An empty cache.  order: how a page lies in memory, "heads" [head][position] or "positions"
        [position][head]."""
        if order not in ("heads", "positions"):
            raise ValueError('order is "heads" or "positions"')
        inner = (kv_heads, page_size) if order == "heads" else (page_size, kv_heads)
        k, v = (torch.zeros(layers, pages, *inner, head_dim, dtype=dtype, device=device) for _ in range(2))
        if order == "positions":
            k, v = k.transpose(2, 3), v.transpose(2, 3)
        return cls(k, v, PageMap.empty(pages, slots, -(-max_length // page_size), device))

    # ------------------------------------------------------------ attention
    def _q(self, q: torch.Tensor):
        if q.dim() != 3 or q.device != self.device or q.shape[2] != self.head_dim or q.stride(2) != 1:
            raise ValueError(f"q must be [rows, heads, {self.head_dim}] on {self.device}, head_dim contiguous")
        fmt = _FORMAT.get(q.dtype)
        if fmt is None:
            raise ValueError("q must be fp16, bf16 or fp32")
        rows, heads, _ = q.shape
        return rows, heads, fmt, q.stride(0) if rows > 1 else 0, q.stride(1) if heads > 1 else 0

    @staticmethod
    def _reach(window: int, sinks: int):
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks are not negative")
        return min(window, 0xffffffff), min(sinks, 0xffffffff)

    def _out(self, q: torch.Tensor, out: torch.Tensor | None, lse: bool):
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous():
            raise ValueError("out must be contiguous and have q's shape, type and device")
        return out, torch.empty(q.shape[:2], dtype=torch.float32, device=self.device) if lse else None

    def decode(self, q: torch.Tensor, layer: int = 0, slots: torch.Tensor | None = None, window: int = 0,
               sinks: int = 0, scale: float | None = None, out: torch.Tensor | None = None, lse: bool = False,
               map: PageMap | None = None):
        """Attention of the newest token of each sequence (rta_paged_decode): q [sequences, heads, head_dim] of slots
        0, 1, ... or of `slots`.  window: how many positions back it sees (0: all), sinks: first tokens that stay
        visible, scale: 1 / sqrt(head_dim) unless given.  Returns out, or (out, lse) with lse=True."""
        rows, heads, fmt, row, head = self._q(q)
        out, l = self._out(q, out, lse)
        window, sinks = self._reach(window, sinks)
        m = self._map(map)
        if rows:
            check(self._lib.rta_paged_decode(
                self._at, m._at, layer, None if slots is None else _ints(slots, "slots", self.device, rows).data_ptr(),
                rows, q.data_ptr(), fmt, heads, row, head, self.head_dim ** -0.5 if scale is None else scale, window,
                sinks, out.data_ptr(), l.data_ptr() if lse else None, self._ws, self._ws_bytes, self._stream()))
        return (out, l) if lse else out

    def prefill(self, q: torch.Tensor, starts: torch.Tensor, layer: int = 0, slots: torch.Tensor | None = None,
                window: int = 0, sinks: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                lse: bool = False, map: PageMap | None = None):
        """Attention of the newest tokens of each sequence (rta_paged_prefill): rows starts[b] .. starts[b + 1] - 1 of
        q [rows, heads, head_dim] are sequence b's, its last ones.  The rest as in decode; q in the cache's type, out
        not over q.  Rows that `starts` gives to no sequence are flagged and not written."""
        rows, heads, fmt, row, head = self._q(q)
        out, l = self._out(q, out, lse)
        window, sinks = self._reach(window, sinks)
        m = self._map(map)
        batch = _ints(starts, "starts", self.device).shape[0] - 1
        if rows:
            check(self._lib.rta_paged_prefill(
                self._at, m._at, layer, None if slots is None else _ints(slots, "slots", self.device, batch).data_ptr(),
                max(batch, 0), starts.data_ptr(), rows, q.data_ptr(), fmt, heads, row, head,
                self.head_dim ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
                l.data_ptr() if lse else None, self._ws, self._ws_bytes, self._stream()))
        return (out, l) if lse else out

    # ------------------------------------------------------------ writes and bookkeeping
    def append(self, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, layer: int = 0,
               slots: torch.Tensor | None = None, map: PageMap | None = None) -> None:
        """Write the K/V rows [rows, kv_heads, head_dim] (the cache's type, or fp32) of the sequences' newest tokens
        (rta_paged_append), after reserve."""
        for t in (k, v):
            if (t.dim() != 3 or tuple(t.shape[1:]) != (self.kv_heads, self.head_dim) or t.device != self.device
                    or t.stride(2) != 1):
                raise ValueError(f"k and v must be [rows, {self.kv_heads}, {self.head_dim}] on {self.device}, head_dim "
                                 "contiguous")
        if k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _FORMAT:
            raise ValueError("k and v must have one shape and type: the cache's, or fp32")
        rows = k.shape[0]
        row, head = (k.stride(0) if rows > 1 else 0), (k.stride(1) if self.kv_heads > 1 else 0)
        if (row, head) != ((v.stride(0) if rows > 1 else 0), (v.stride(1) if self.kv_heads > 1 else 0)):
            raise ValueError("k and v must have the same strides")
        m = self._map(map)
        batch = _ints(starts, "starts", self.device).shape[0] - 1
        if rows:
            check(self._lib.rta_paged_append(
                self._at, m._at, layer, None if slots is None else _ints(slots, "slots", self.device, batch).data_ptr(),
                max(batch, 0), starts.data_ptr(), rows, k.data_ptr(), v.data_ptr(), _FORMAT[k.dtype], row, head,
                self._ws, self._ws_bytes, self._stream()))

    def reserve(self, counts: torch.Tensor, slots: torch.Tensor | None = None, out: PageMap | None = None,
                map: PageMap | None = None) -> PageMap:
        """Grow the sequences by counts[i] positions (rta_pages_reserve).  Like every bookkeeping call it updates the
        cache's map (or `map`), or leaves it and writes the result to `out`; returns the map it wrote."""
        m, out = self._maps(map, out)
        n = _ints(counts, "counts", self.device).shape[0]
        check(self._lib.rta_pages_reserve(
            self._at, m._at, out._at, None if slots is None else _ints(slots, "slots", self.device, n).data_ptr(),
            counts.data_ptr(), n, self._ws, self._ws_bytes, self._stream()))
        return out

    def fork(self, src: torch.Tensor, dst: torch.Tensor, out: PageMap | None = None,
             map: PageMap | None = None) -> PageMap:
        """The empty slots dst[i] become copies of src[i] that share its full pages (rta_pages_fork)."""
        m, out = self._maps(map, out)
        n = _ints(src, "src", self.device).shape[0]
        check(self._lib.rta_pages_fork(self._at, m._at, out._at, src.data_ptr(),
                                       _ints(dst, "dst", self.device, n).data_ptr(), n, self._ws, self._ws_bytes,
                                       self._stream()))
        return out

    def free(self, slots: torch.Tensor, out: PageMap | None = None, map: PageMap | None = None) -> PageMap:
        """Drop the sequences in `slots` (rta_pages_free)."""
        m, out = self._maps(map, out)
        n = _ints(slots, "slots", self.device).shape[0]
        check(self._lib.rta_pages_free(self._at, m._at, out._at, slots.data_ptr(), n, self._ws, self._ws_bytes,
                                       self._stream()))
        return out

    def compact(self, out: PageMap | None = None, map: PageMap | None = None,
                live: torch.Tensor | None = None) -> PageMap:
        """Move the pages in use to the pool's front (rta_pages_compact); live [1] int32 receives how many there are."""
        m, out = self._maps(map, out)
        check(self._lib.rta_pages_compact(
            self._at, m._at, out._at, None if live is None else _ints(live, "live", self.device, 1).data_ptr(),
            self._ws, self._ws_bytes, self._stream()))
        return out

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page dst[i] takes the data of page src[i] in every layer (rta_pages_copy)."""
        n = _ints(src, "src", self.device).shape[0]
        check(self._lib.rta_pages_copy(self._at, src.data_ptr(), _ints(dst, "dst", self.device, n).data_ptr(), n,
                                       self._ws, self._ws_bytes, self._stream()))

    def check(self) -> None:
        """Waits for the stream, raises RtaError with what the device-side checks have found since the last check
        (include/rta.h, section 1c), and clears it."""
        word = ctypes.c_uint32(0)
        status = self._lib.rta_workspace_error(self._ws, self._ws_bytes, self._stream(), ctypes.byref(word))
        if status == _lib.RTA_OK:
            return
        message = self._lib.rta_last_error().decode(errors="replace")
        if word.value:
            self.workspace[:4].zero_()
        raise RtaError(status, message)

    def _map(self, map: PageMap | None) -> PageMap:
        if map is None:
            return self.map
        if (map.refs.shape[0] != self.pages or map.refs.device != self.device
                or map.table.shape != self.map.table.shape):
            raise ValueError("the map must have the cache's pages, slots, width and device")
        return map

    def _maps(self, map: PageMap | None, out: PageMap | None):
        m = self._map(map)
        return m, m if out is None else self._map(out)

    def _stream(self) -> int:
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the cache lives on {self.device}, another device is current")
        return torch._C._cuda_getCurrentRawStream(self.device.index)  # current_stream() builds an object: 3 us


__all__ = ["PageMap", "PagedCache"]

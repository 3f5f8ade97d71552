"""The 4-bit key/value cache and the attention that reads it, over the C ABI
(madi_kv4_* in include/madi_q8.h, which states the format, the layout and what
each argument may be).

    cache = kv4.alloc(n_pages, page=64, heads=8, dim=128)
    batch = kv4.Batch(table, lens, rows=1)       # one new token per sequence
    batch.reserve(cache, nh=32)
    kv4.kvStore(cache, batch, k, v)              # rows into the cache
    kv4.kvAttn(out, q, cache, batch, nh=32)      # their attention
    kv4.kvLoad(cache, batch, k_back, v_back)     # and back out of it

Rows are torch tensors of float16 or float32, [m][heads * dim] or [m][heads][dim]
with the elements of a row contiguous (a slice of a stacked projection's output is fine).
Work is enqueued on the library's stream (madi_amd.q8.init).  As in madi_amd.q8,
a refused call raises MadiError; tensors in host memory or on another GPU than the
library's are refused.
"""
from __future__ import annotations

import ctypes
import math

from ._lib import F16, F32, MadiError, calls, lib
from .q8 import ptr


class _Cache(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("n_pages", ctypes.c_uint32), ("page", ctypes.c_uint32),
                ("nkv", ctypes.c_uint32), ("d", ctypes.c_uint32)]


class _Batch(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("row_off", ctypes.c_void_p),
                ("b", ctypes.c_uint32), ("max_pages", ctypes.c_uint32), ("rows", ctypes.c_uint32),
                ("m", ctypes.c_uint32), ("len_max", ctypes.c_uint32), ("work", ctypes.c_void_p),
                ("work_bytes", ctypes.c_size_t)]


def _bytes(n_pages: int, page: int, heads: int, dim: int) -> int:
    for v in (n_pages, page, heads, dim):
        if not 0 <= v < 1 << 32:
            raise MadiError(-5, "kv4", f"{v} is not a 32-bit size")
    n = lib().madi_kv4_bytes(n_pages, page, heads, dim)
    if n == 0:
        raise MadiError(-5, "kv4", f"a cache of {n_pages} pages of {page} tokens, {heads} heads of {dim}")
    return n


DEVICE = 0  # the library's (madi_init)


def _on(what, *tensors) -> int:
    """0 where all are on the library's device, else another number."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise MadiError(-9, what, f"tensors on {' and '.join(sorted(map(str, devices)))}")
    device = devices.pop()
    return 0 if device.type == "cuda" and device.index == DEVICE else -1


def _device(cache, batch, what: str) -> int:
    """The device that a call's rows have to be on.  (Without one the library refuses
    every call by itself: -1, any will do.)"""
    if cache.on | batch.on:
        if lib().madi_device_cu_count():
            raise MadiError(-9, what, f"cache and batch must be in the memory of GPU {DEVICE}, "
                                      f"are on {cache.data.device} and {batch.table.device}")
        return -1
    return DEVICE


class KV4:
    """A pool of pages over `data`, a contiguous device tensor of at least
    madi_kv4_bytes bytes (one pool per layer)."""

    def __init__(self, data, page: int, heads: int, dim: int, n_pages: int | None = None):
        held = data.numel() * data.element_size()
        if n_pages is None:
            n_pages = held // _bytes(1, page, heads, dim)
        if not data.is_contiguous() or _bytes(n_pages, page, heads, dim) > held:
            raise MadiError(-5, "kv4.KV4", f"data must be contiguous and hold {n_pages} pages, has {held} bytes")
        self.data, self.page, self.heads, self.dim, self.n_pages = data, page, heads, dim, n_pages
        self.width, self.scale = heads * dim, 1.0 / math.sqrt(dim)
        self.on = _on("kv4.KV4", data)
        self._c = _Cache(data.data_ptr(), n_pages, page, heads, dim)
        self.addr = ctypes.addressof(self._c)


def alloc(n_pages: int, page: int, heads: int, dim: int, device="cuda") -> KV4:
    import torch
    data = torch.empty(_bytes(n_pages, page, heads, dim), dtype=torch.uint8, device=device)
    return KV4(data, page, heads, dim, n_pages)


def _index(t, shape, what):
    """A device tensor of 32-bit integers of this shape."""
    if t.element_size() != 4 or t.is_floating_point() or not t.is_contiguous() or tuple(t.shape) != shape:
        raise MadiError(-5, "kv4.Batch", f"{what} must be 32-bit integers, contiguous, {shape}; "
                                         f"is {t.dtype} {tuple(t.shape)}")
    return t


class Batch:
    """The sequences and rows of a call (madi_kv4_batch): table [b][max_pages] and lens
    [b] on the device; `rows` new rows per sequence, or at most `rows` with their
    starts in row_off [b + 1] and m rows in all.  The tensors are read when the kernels run, so a
    decode loop (or a captured graph) adds to lens and fills in table in
    place and keeps the Batch.  Calls that may overlap take a Batch each: its
    workspace holds their partial results."""

    def __init__(self, table, lens, rows: int = 1, row_off=None, m: int | None = None, len_max: int = 0):
        if table.dim() != 2:
            raise MadiError(-5, "kv4.Batch", f"table must be [b][max_pages], is {tuple(table.shape)}")
        b, max_pages = table.shape
        _index(table, (b, max_pages), "table")
        _index(lens, (b,), "lens")
        if row_off is not None:
            _index(row_off, (b + 1,), "row_off")
            if m is None:
                raise MadiError(-9, "kv4.Batch", "row_off needs m, the number of rows in all")
        m = b * rows if m is None else m
        for what, v in (("rows", rows), ("m", m), ("len_max", len_max)):
            if not 0 <= v < 1 << 31:
                raise MadiError(-5, "kv4.Batch", f"{what} = {v}")
        self.table, self.lens, self.row_off, self.work = table, lens, row_off, None
        self._outgrown: list = []
        self.b, self.rows, self.m = b, rows, m
        self.on = _on("kv4.Batch", table, lens, row_off)
        self._c = _Batch(ptr(table), ptr(lens), ptr(row_off), b, max_pages, rows, m, len_max, None, 0)
        self.addr = ctypes.addressof(self._c)

    def reserve(self, cache: KV4, nh: int) -> int:
        """Allocate the workspace with which kvAttn splits long caches over
        workgroups as it sees fit; returns its bytes.  (The largest of several
        caches' or heads' needs is kept.  A smaller one that was there before lives as
        long as the Batch: calls still running and captured graphs point to it.)"""
        import torch
        if not 1 <= nh < 1 << 32 or nh % cache.heads:  # (the library would ask for no bytes)
            raise MadiError(-5, "kv4.Batch.reserve", f"{nh} query heads over {cache.heads} kv heads")
        need = int(lib().madi_kv4_attn_bytes(cache.addr, self.addr, nh))
        if need > self._c.work_bytes:
            if self.work is not None:
                self._outgrown.append(self.work)
            self.work = torch.empty(need, dtype=torch.uint8, device=self.table.device)
            self._c.work, self._c.work_bytes = self.work.data_ptr(), need
        return need


_check: tuple = ()


def _rows(t, m: int, width: int, device: int, what: str) -> int:
    """2 * row distance + dtype code of rows [m][width].  (Rows that are not apart, a
    broadcast's, are left to the library to refuse.)"""
    global _check
    if not _check:
        import torch
        from ._pycall import rows
        _check = rows, torch.float16, torch.float32
    rows, f16, f32 = _check
    r = rows(t, m, width, f16, f32, device)
    if r == -2:
        raise MadiError(-9, what, f"rows must be in the memory of GPU {device}, are on {t.device}")
    if r < 0:
        raise MadiError(-5, what, f"rows must be float16 or float32 [{m}][{width}] with contiguous rows; "
                                  f"got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")
    return r


def _pair(a, b, cache: KV4, batch: Batch, width: int, what: str):
    device = _device(cache, batch, what)
    a, b = _rows(a, batch.m, width, device, what), _rows(b, batch.m, width, device, what)
    if (a ^ b) & 1:
        raise MadiError(-9, what, "the two tensors are of two types")
    return a >> 1, b >> 1, a & 1


def kvStore(cache: KV4, batch: Batch, k, v) -> None:
    """Quantise rows k, v into the cache, at each sequence's last positions."""
    ldk, ldv, dt = _pair(k, v, cache, batch, cache.width, "kvStore")
    calls.madi_kv4_store(cache.addr, batch.addr, k, v, ldk, ldv, dt)


def kvLoad(cache: KV4, batch: Batch, k, v) -> None:
    """Read each sequence's last rows back into k, v."""
    ldk, ldv, dt = _pair(k, v, cache, batch, cache.width, "kvLoad")
    calls.madi_kv4_load(k, v, ldk, ldv, dt, cache.addr, batch.addr)


def kvAttn(out, q, cache: KV4, batch: Batch, nh: int, causal: bool = True, window: int = 0,
           scale: float | None = None) -> None:
    """out = softmax(scale q K^T) V over the cache, scale 1 / sqrt(dim) by
    default.  causal: a row sees the positions up to its own, the last `window`
    of them where window is not 0; else all of its sequence (cross-attention)."""
    if not 0 <= window < 1 << 32:  # (an argument of 32 bits: others would wrap)
        raise MadiError(-5, "kvAttn", f"window {window}")
    ldo, ldq, dt = _pair(out, q, cache, batch, nh * cache.dim, "kvAttn")
    calls.madi_kv4_attn(out, q, cache.addr, batch.addr, nh, ldo, ldq, window, 1 if causal else 0, dt,
                        cache.scale if scale is None else scale)


__all__ = ["KV4", "Batch", "alloc", "kvStore", "kvLoad", "kvAttn", "F16", "F32"]

"""Projections with low-rank adapters of many requests, over the C ABI (madi_lora in
include/madi_q8.h, which states what is computed and what each argument may be).

    ad = lora.Adapters(a, b, scale)                     # of every request that is served
    ad.reserve(m)
    lora.pprojLora(x, w, out, m, n, k, ad, adapter)     # out = W x + scale B (A x), row by row

Work is enqueued on the library's stream (madi_amd.q8.init); a refused call raises
MadiError; tensors in host memory or on another GPU than the library's are refused.
"""
from __future__ import annotations

import ctypes

from ._lib import MadiError, calls, lib
from .kv4 import DEVICE, _here, _on, _torch
from .q8 import Q8, ptr


class _Lora(ctypes.Structure):
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("scale", ctypes.c_void_p),
                ("adapter", ctypes.c_void_p), ("row_seq", ctypes.c_void_p), ("adapters", ctypes.c_uint32),
                ("rank", ctypes.c_uint32), ("seqs", ctypes.c_uint32), ("work", ctypes.c_void_p),
                ("work_bytes", ctypes.c_size_t)]


class Adapters:
    """The adapters of one projection: a [adapters][rank][k] and b [adapters][n][rank]
    float16, scale [adapters] float32; ranks smaller than `rank` filled up with zeros.
    Calls that may overlap take an Adapters each (over the same tensors): its workspace holds A x."""

    def __init__(self, a, b, scale):
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise MadiError(-5, "lora.Adapters", f"a must be [adapters][rank][k] and b [adapters][n][rank], are "
                                                 f"{tuple(a.shape)} and {tuple(b.shape)}")
        self.n, self.rank, self.k = a.shape
        self.width = b.shape[1]
        if not lib().madi_lora_bytes(1, self.k, self.rank):
            raise MadiError(-5, "lora.Adapters", f"rank {self.rank} (a multiple of 8, 8 to 128)")
        t = _torch()
        at = (_here("lora.Adapters", "a", a, a.shape, t.f16, t.f16), _here("lora.Adapters", "b", b, b.shape, t.f16, t.f16),
              _here("lora.Adapters", "scale", scale, (self.n,), t.f32, t.f32))
        self.a, self.b, self.scale, self.work = a, b, scale, None
        self.on = _on("lora.Adapters", a, b, scale)
        self._outgrown: list = []
        self.rows = 0  # that the workspace is enough for
        self._c = _Lora(*at, None, None, self.n, self.rank, 0, None, 0)
        self.addr = ctypes.addressof(self._c)

    def reserve(self, m: int) -> int:
        """Allocate the workspace for calls of up to m rows; returns its bytes.  (A smaller
        one that was there before lives as long as the Adapters: calls still running and captured
        graphs point to it.)"""
        import torch
        if not 0 <= m < 1 << 32:
            raise MadiError(-5, "lora.Adapters.reserve", f"{m} rows")
        need = int(lib().madi_lora_bytes(m, self.k, self.rank))
        if need > self._c.work_bytes:
            if self.work is not None:
                self._outgrown.append(self.work)
            self.work = torch.empty(need, dtype=torch.uint8, device=self.a.device)
            self._c.work, self._c.work_bytes = self.work.data_ptr(), need
        self.rows = max(self.rows, m)
        return need


def pprojLora(in_f32, w: Q8, out_f32, M: int, N: int, Kk: int, ad: Adapters, adapter, row_seq=None) -> None:
    """pproj with the adapter of each row: in_f32 [M][Kk] -> out_f32 [M][N].  adapter: int32,
    [M], or [sequences] with row_seq [M], the rows' sequences (kv4.Pages.row_seq); a number that
    is no adapter (-1), or a row without a sequence: none."""
    what, t = "pprojLora", _torch()
    if Kk != ad.k or N != ad.width:
        raise MadiError(-5, what, f"adapters of {ad.k} -> {ad.width} for a projection of {Kk} -> {N}")
    if ad.on and lib().madi_device_cu_count():
        raise MadiError(-9, what, f"the Adapters must be in the memory of GPU {DEVICE}, are on {ad.a.device}")
    x, y = _here(what, "in_f32", in_f32, (M, Kk), t.f32, t.f32), _here(what, "out_f32", out_f32, (M, N), t.f32, t.f32)
    c = ad._c
    if row_seq is None:
        c.adapter, c.row_seq = _here(what, "adapter", adapter, (M,), t.i32, t.u32), 0
    else:
        c.adapter = _here(what, "adapter", adapter, (adapter.shape[0],), t.i32, t.u32)
        c.row_seq = _here(what, "row_seq", row_seq, (M,), t.i32, t.u32)
        c.seqs = adapter.shape[0]
    if M > ad.rows:
        ad.reserve(M)
    calls.madi_q8_pproj_lora(y, x, w.qs, w.scales, M, N, Kk, ad.addr)


__all__ = ["Adapters", "pprojLora"]

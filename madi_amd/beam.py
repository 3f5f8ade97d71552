"""Beam search over the C ABI (madi_beam_* in include/madi_q8.h, which states what is
computed and what each argument may be).

    s = beam.Search(groups=8, beams=5, vocab=51866, eos=50257)
    beam.beamSelect(s, logits, score)                   # s.score, s.parent, s.token
    beam.beamGather(caches, caches, s.parent, beams=5)  # dense states, in place
    kv4.kvFork(pages, s.parent, beams=5)                # or page tables

Work is enqueued on the library's stream (madi_amd.q8.init); a refused call raises
MadiError; tensors in host memory or on another GPU than the library's are refused.
"""
from __future__ import annotations

import ctypes
import struct
import threading

from ._lib import F16, F32, MadiError, calls, lib
from .kv4 import DEVICE, _here, _on, _torch
from .q8 import ptr


class _Beam(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("score", ctypes.c_void_p), ("done", ctypes.c_void_p),
                ("ban", ctypes.c_void_p), ("ban_ld", ctypes.c_uint32), ("ld", ctypes.c_uint32),
                ("groups", ctypes.c_uint32), ("beams", ctypes.c_uint32), ("vocab", ctypes.c_uint32),
                ("n", ctypes.c_uint32), ("eos", ctypes.c_uint32), ("dtype", ctypes.c_int),
                ("out_score", ctypes.c_void_p), ("out_parent", ctypes.c_void_p), ("out_token", ctypes.c_void_p),
                ("work", ctypes.c_void_p), ("work_bytes", ctypes.c_size_t)]


class _States(ctypes.Structure):
    _fields_ = [("dst", ctypes.c_void_p), ("src", ctypes.c_void_p), ("n_states", ctypes.c_uint32),
                ("stride", ctypes.c_size_t), ("row_bytes", ctypes.c_size_t), ("rows", ctypes.c_uint32),
                ("lens", ctypes.c_void_p), ("parent", ctypes.c_void_p), ("ldp", ctypes.c_uint32),
                ("groups", ctypes.c_uint32), ("beams", ctypes.c_uint32)]


class Search:
    """The sizes of a selection, its workspace and its results: score (float32), parent and
    token (int32), [groups][n], overwritten by each beamSelect.  n (default beams) best
    are kept.  Selections that may overlap take a Search each."""

    def __init__(self, groups: int, beams: int, vocab: int, n: int | None = None, eos: int = 0, device="cuda"):
        import torch
        n = beams if n is None else n
        for v in (groups, beams, vocab, n, eos):
            if not 0 <= v < 1 << 32:
                raise MadiError(-5, "beam.Search", f"{v} is not a 32-bit size")
        need = lib().madi_beam_bytes(groups, beams, vocab, n)
        if need == 0:
            raise MadiError(-5, "beam.Search", f"{groups} groups of {beams} beams, vocab {vocab}, n {n}")
        self.groups, self.beams, self.vocab, self.n, self.eos = groups, beams, vocab, n, eos
        self.score = torch.empty(groups, n, dtype=torch.float32, device=device)
        self.parent = torch.empty(groups, n, dtype=torch.int32, device=device)
        self.token = torch.empty(groups, n, dtype=torch.int32, device=device)
        self.work = torch.empty(need, dtype=torch.uint8, device=device)
        self.on = _on("beam.Search", self.work)
        self._c = _Beam(None, None, None, None, 0, 0, groups, beams, vocab, n, eos, F32, ptr(self.score),
                        ptr(self.parent), ptr(self.token), ptr(self.work), need)
        self.addr = ctypes.addressof(self._c)
        self._shapes = (groups, beams), ((vocab + 31) // 32,), (groups * beams, (vocab + 31) // 32)


def beamSelect(s: Search, logits, score, done=None, ban=None) -> None:
    """The n best continuations of each group into s.score, s.parent, s.token.
    logits: [groups * beams][vocab] float16 or float32, contiguous within a row; score
    [groups][beams] float32 (s.score itself where n is beams); done [groups][beams], bool or
    uint8: beams that have ended; ban: int32 bitmaps [words] or [groups * beams][words],
    words = (vocab + 31) // 32, bit v % 32 of word v // 32 for each token v left out."""
    what, m, t = "beamSelect", s.groups * s.beams, _torch()
    device = DEVICE
    if s.on and lib().madi_device_cu_count():
        raise MadiError(-9, what, f"the Search must be in the memory of GPU {DEVICE}, is on {s.work.device}")
    r = t.rows(logits, m, s.vocab, t.f16, t.f32, device) if logits.dim() == 2 and logits.shape[0] == m else -1
    if r == -2 and not lib().madi_device_cu_count():  # (the library refuses the call by itself)
        device, r = -1, t.rows(logits, m, s.vocab, t.f16, t.f32, -1)
    if r == -2:
        raise MadiError(-9, what, f"tensors must be in the memory of GPU {DEVICE}, are on {logits.device}")
    if r < 0 or r >> 1 < s.vocab:
        raise MadiError(-5, what, f"logits must be float16 or float32 [{m}][{s.vocab}] with contiguous rows; got "
                                  f"{logits.dtype} {tuple(logits.shape)} with strides {logits.stride()}")
    scores, flat, rows = s._shapes
    c = s._c
    c.score = _here(what, "score", score, scores, t.f32, t.f32)
    c.done = 0 if done is None else _here(what, "done", done, scores, t.bool, t.u8)
    if ban is None:
        c.ban = 0
    else:
        one = ban.dim() == 1
        c.ban = _here(what, "ban", ban, flat if one else rows, t.i32, t.u32)
        c.ban_ld = 0 if one else flat[0]
    c.logits, c.ld, c.dtype = logits.data_ptr(), r >> 1, F32 if r & 1 else F16
    calls.madi_beam_select(s.addr)


class _Call(threading.local):
    """What a call reads in host memory, for each thread its own."""

    def __init__(self):
        self.addresses, self.states = (ctypes.c_void_p * 64)(), _States()
        self.at = ctypes.addressof(self.addresses), ctypes.addressof(self.states)


_call = _Call()
_fill = struct.Struct("PPIxxxxNNIxxxxPPIII").pack_into  # (its fields in order, one call for all)


def beamGather(dst, src, parent, beams: int, lens=None) -> None:
    """Slot (g, i) of every state in dst becomes slot (g, parent[g][i]) of the state in
    src at the same place (src None, or the same tensors: in place); a parent that is no beam (-1) leaves it.
    dst, src: lists of tensors [groups * beams][rows][...], alike, each slot contiguous
    (32 go in one launch; more take several, each checked by itself before it).  lens [groups * beams], int32: rows that the slot read
    holds; the rows behind them are left as they were."""
    what, t = "beamGather", _torch()
    src = dst if src is None else src
    if not dst or len(dst) != len(src):
        raise MadiError(-5, what, f"{len(dst)} and {len(src)} states")
    base, states = _call.at
    for at in range(0, len(dst), 32):
        d, f = list(dst[at:at + 32]), list(src[at:at + 32])
        r = t.states(d, f, DEVICE, base)
        if r == -2 and not lib().madi_device_cu_count():
            r = t.states(d, f, -1, base)
        if r == -2:
            raise MadiError(-9, what, f"states must be in the memory of GPU {DEVICE}")
        if r == -1 or not 1 <= beams <= 32 or r[0] % beams or parent.dim() != 2 or parent.shape[1] < beams or \
                d[0].shape != dst[0].shape:
            raise MadiError(-5, what, f"{beams} beams (1 to 32), parent {tuple(parent.shape)}, states [slots][rows][...], alike "
                                      f"and contiguous within a slot: {[(tuple(x.shape), x.stride(), x.dtype) for x in d + f]}")
        slots, rows, row_bytes, apart = r
        groups = slots // beams
        _fill(_call.states, 0, base, base + 8 * len(d), len(d), apart, row_bytes, rows,
              0 if lens is None else _here(what, "lens", lens, (slots,), t.i32, t.u32),
              _here(what, "parent", parent, (groups, parent.shape[1]), t.i32, t.u32), parent.shape[1], groups, beams)
        calls.madi_beam_gather(states)


__all__ = ["Search", "beamSelect", "beamGather"]

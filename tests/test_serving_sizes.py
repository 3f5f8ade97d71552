"""Sizes of beam search whose products pass 64 bits: refused, without a GPU."""
import ctypes

import pytest

import madi_amd
from madi_amd import _lib, beam

torch = pytest.importorskip("torch")

AT = [0x10000000 * (i + 1) for i in range(16)]  # never dereferenced


@pytest.mark.parametrize("rows,row_bytes,stride", [
    (1 << 24, 1 << 40, 1 << 40),                # 2^64: 0 bytes
    ((1 << 24) + 1, 1 << 40, 1 << 40),          # 2^64 + 2^40
    ((1 << 32) - 1, 1 << 40, 0), ((1 << 31), 1 << 33, 64), (3 << 30, 0x155555558, 1 << 36), (2, 1 << 40, 1 << 40)])
def test_states_whose_size_passes_64_bits(rows, row_bytes, stride):
    d = (ctypes.c_void_p * 1)(AT[0])
    s = beam._States(ctypes.addressof(d), None, 1, stride, row_bytes, rows, None, AT[1], 1, 1, 1)
    assert madi_amd.lib().madi_beam_gather(ctypes.addressof(s)) == -5, _lib.last_error()

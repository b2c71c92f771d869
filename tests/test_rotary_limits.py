"""Sizes and positions beyond 32 bits are refused by rotate, on the CPU (nothing is launched)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from diffusorrt_amd import _lib
from diffusorrt_amd.rotary import RotaryPositions


@pytest.mark.parametrize("shape", [(2**32 + 5, 1, 8), (1, 2**32 + 5, 8), (2**31, 1, 8), (1, 2**31, 8)])
def test_sizes_beyond_32_bits_are_refused(shape):
    # (2^32 + 5 rows would be 5 of them in the library's 32 bits)
    x = torch.zeros(1, 1, 8).expand(shape)
    with pytest.raises(ValueError, match="2\\^31"):
        RotaryPositions(8, device="cpu").rotate(x, 0)


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")
@pytest.mark.parametrize("rows, pos0", [(2, 2**31 - 1), (2**31 - 1, 2)])
def test_positions_beyond_32_bits_are_refused_at_the_c_entry(rows, pos0):
    turns = _lib.Rotary(4096, 8, 0, 1.0)
    status = _lib.load().drt_op_rotate(4096, 8, 8, _lib.F32, rows, 1, 8, C.addressof(turns), None, pos0, 0,
                                       4096, 8, 8, None)
    assert status == _lib.INVALID_ARGUMENT and "positions" in _lib.last_error()

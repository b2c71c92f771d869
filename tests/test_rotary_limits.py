"""Sizes beyond 32 bits are refused by rotate, on the CPU (nothing is launched)."""
from __future__ import annotations

import pytest
import torch

from diffusorrt_amd.rotary import RotaryPositions


@pytest.mark.parametrize("shape", [(2**32 + 5, 1, 8), (1, 2**32 + 5, 8), (2**31, 1, 8), (1, 2**31, 8)])
def test_sizes_beyond_32_bits_are_refused(shape):
    # (2^32 + 5 rows would be 5 of them in the library's 32 bits)
    x = torch.zeros(1, 1, 8).expand(shape)
    with pytest.raises(ValueError, match="2\\^31"):
        RotaryPositions(8, device="cpu").rotate(x, 0)

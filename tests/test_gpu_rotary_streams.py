"""RotaryPositions.rotate: positions as numpy gives them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diffusorrt_amd.rotary import RotaryPositions

pytestmark = pytest.mark.gpu


def test_numpy_positions():
    rotary = RotaryPositions(64)
    x = torch.from_numpy(np.random.default_rng(0).standard_normal((5, 3, 64), np.float32)).cuda()
    want = rotary.rotate(x, 70000)
    for first in (np.int32(70000), np.int64(70000), np.arange(70000, 70003)[0]):
        assert torch.equal(rotary.rotate(x, first), want)
    for bad in (np.float64(3), np.True_, np.arange(5), "3", None, np.int64(2**31 - 2)):
        with pytest.raises(ValueError):
            rotary.rotate(x, bad)

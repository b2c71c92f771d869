"""RotaryPositions used on other streams than its own, and positions as numpy gives them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diffusorrt_amd.paged import PagedKVCache
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


BUSY = 20_000_000  # cycles, about 10 ms


@pytest.mark.parametrize("call", ["rotate", "append"])
def test_dropped_after_a_call_on_another_stream(call):
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((40, 3, 128), np.float32)).cuda()
    rotary = RotaryPositions(128)
    cache = PagedKVCache(1, 3, 2)
    batch = cache.batch([[1]], [40], [40], heads=3)

    def run():
        if call == "rotate":
            return rotary.rotate(x, 0)
        cache.append(0, x, x, batch, rotary=rotary)
        return cache.load(0, batch)[0]

    want = run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    cache.data.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
        got = run()
    n = rotary.turns.numel()
    del rotary, run
    taken = [torch.full((n,), 2**62, dtype=torch.int64, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(taken) == 64


def test_no_rotation_is_made_in_a_capture():
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured"):
            RotaryPositions(8)
        x += 1
    graph.replay()
    assert torch.equal(x.cpu(), torch.ones(4))


def test_streams_are_told_once_and_captures_never():
    rotary = RotaryPositions(8)
    x = torch.zeros(2, 1, 8, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(2):
        with torch.cuda.stream(side):
            rotary.rotate(x, 1)
        assert rotary._streams == {torch.cuda.current_stream().cuda_stream, side.cuda_stream}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary.rotate(x, 1)
    assert len(rotary._streams) == 2
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, x)

"""Copies of the paged cache's objects: a cache's has pages of its own, a plan and frequencies, which do not
change, are shared."""
from __future__ import annotations

import copy

import pytest
import torch

from diffusorrt_amd import _lib
from diffusorrt_amd.paged import PagedKVCache
from diffusorrt_amd.rotary import RotaryPositions


def test_a_copied_cache_has_its_own_pages():
    cache = PagedKVCache(2, 3, 4, device="cpu")
    other = copy.deepcopy(cache)
    assert other._geometry == cache._geometry and torch.equal(other.data, cache.data)
    other.data.fill_(1.0)
    assert not cache.data.any()
    assert cache.data.data_ptr() not in [v for v in vars(other).values() if isinstance(v, int)]


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")
def test_a_copied_plan_is_the_plan():
    batch = PagedKVCache(1, 1, 4, device="cpu").batch([[2]], [5], [1], heads=1)
    assert copy.deepcopy(batch) is batch and copy.copy(batch)._address == batch._address
    assert copy.deepcopy({"plans": [batch]})["plans"][0] is batch


def test_copied_frequencies_are_the_frequencies():
    rotary = RotaryPositions(8, device="cpu")
    assert copy.deepcopy(rotary) is rotary


@pytest.mark.gpu
def test_rows_of_a_copy_are_not_the_caches():
    k = torch.ones(5, 1, 128, dtype=torch.float16, device="cuda")
    cache = PagedKVCache(1, 1, 2)
    batch = cache.batch([[1]], [5], [5], heads=1)
    cache.append(0, k, k, batch)
    other = copy.deepcopy(cache)
    other.append(0, 2 * k, 3 * k, batch)
    assert all(torch.equal(x, k) for x in cache.load(0, batch))
    k2, v2 = other.load(0, batch)
    assert torch.equal(k2, 2 * k) and torch.equal(v2, 3 * k)
    del cache
    q = torch.zeros(5, 1, 128, dtype=torch.float16, device="cuda")
    assert torch.equal(other.attention(0, q, batch), torch.full((5, 128), 3.0, device="cuda"))


@pytest.mark.gpu
def test_no_cache_is_copied_in_a_capture():
    x, cache = torch.zeros(4, device="cuda"), PagedKVCache(1, 1, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured"):
            copy.deepcopy(cache)
        x += 1
    graph.replay()
    assert torch.equal(x.cpu(), torch.ones(4))

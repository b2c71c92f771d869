"""The paged cache on other streams than its own."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diffusorrt_amd.paged import PagedKVCache

pytestmark = pytest.mark.gpu
BUSY = 20_000_000  # cycles, about 10 ms


def _randn(seed, *shape, dtype=torch.float16):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape, np.float32)).cuda().to(dtype)


def test_the_zeros_do_not_overtake_another_streams_rows():
    k, v = _randn(1, 40, 3, 128), _randn(2, 40, 3, 128)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(BUSY)
    cache = PagedKVCache(1, 3, 4)
    with torch.cuda.stream(side):
        batch = cache.batch([[2]], [40], [40], heads=3)
        cache.append(0, k, v, batch)
    torch.cuda.synchronize()
    k2, v2 = cache.load(0, batch)
    assert torch.equal(k2, k) and torch.equal(v2, v)


def test_a_cache_dropped_after_a_call_on_another_stream():
    k, v = _randn(3, 40, 3, 128), _randn(4, 40, 3, 128)
    cache = PagedKVCache(1, 3, 2)
    batch = cache.batch([[1]], [40], [40], heads=3)
    cache.append(0, k, v, batch)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
        k2, v2 = cache.load(0, batch)
    n = cache.data.numel()
    del cache
    taken = [torch.ones(n, dtype=torch.float16, device="cuda") for _ in range(16)]
    torch.cuda.synchronize()
    assert torch.equal(k2, k) and torch.equal(v2, v) and len(taken) == 16


def test_no_cache_is_made_in_a_capture():
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured"):
            PagedKVCache(1, 1, 1)
        x += 1
    graph.replay()
    assert torch.equal(x.cpu(), torch.ones(4))


@pytest.mark.parametrize("bare", [False, True])
def test_a_batch_is_on_the_device_before_a_captured_graph_is_replayed(bare):
    k, v, q = _randn(5, 300, 2, 128), _randn(6, 300, 2, 128), _randn(7, 3, 4, 128)
    cache = PagedKVCache(1, 2, 8)
    pages, rows = [[7, 2, 5, 0, 3]], [300]
    cache.append(0, k, v, cache.batch(pages, rows, rows, heads=4))
    want = cache.attention(0, q, cache.batch(pages, rows, [3], heads=4))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    if bare:  # no wait begins it
        torch.cuda._sleep(BUSY)
        batch = cache.batch(pages, rows, [3], heads=4)
        with torch.cuda.stream(side):
            graph.capture_begin()
            out = cache.attention(0, q, batch)
            graph.capture_end()
            graph.replay()
    else:
        batch = cache.batch(pages, rows, [3], heads=4)
        with torch.cuda.graph(graph, stream=side):
            out = cache.attention(0, q, batch)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for _ in range(3):
        out.zero_()
        eager = cache.attention(0, q, batch)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager, want)


@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_appends_of_other_rows_of_the_same_tiles_overlap_in_time(src):
    # even rows' batches on one stream, odd ones on another: every tile is written by both at once, and
    # both again and again, as neither waits for the other
    size, hkv, n, times = 64, 4, 8, 6
    cache = PagedKVCache(1, hkv, n, page_size=size)
    pages = [[i] for i in range(n)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    halves = [(0, 7), (7, 20), (20, 33), (33, 45), (45, 50), (50, 64)]  # they part inside groups of eight
    work = [[], []]
    want = torch.zeros(2, n, size, hkv, 128, dtype=torch.float16, device="cuda")
    for i, (lo, hi) in enumerate(halves):
        k, v = (_randn(10 * i + j, n * (hi - lo), hkv, 128, dtype=src) for j in (0, 1))
        batch = cache.batch(pages, [size] * n, [hi - lo] * n, heads=hkv, positions=[lo] * n)
        want[0][:, lo:hi] = k.half().view(n, hi - lo, hkv, 128)
        want[1][:, lo:hi] = v.half().view(n, hi - lo, hkv, 128)
        work[i % 2].append((k, v, batch))
    whole = cache.batch(pages, [size] * n, [size] * n, heads=hkv)
    for _ in range(5):
        cache.data.fill_(float("nan"))
        torch.cuda.synchronize()
        for side in sides:
            with torch.cuda.stream(side):
                torch.cuda._sleep(BUSY // 10)  # both streams' appends are queued before either begins
        for _ in range(times):
            for side, calls in zip(sides, work):
                with torch.cuda.stream(side):
                    for k, v, batch in calls:
                        cache.append(0, k, v, batch)
        torch.cuda.synchronize()
        k2, v2 = cache.load(0, whole)
        assert torch.equal(k2.view_as(want[0]), want[0]) and torch.equal(v2.view_as(want[1]), want[1])

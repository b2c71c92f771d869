"""Stores of one cache on two streams: of different tiles at once, of one tile's rows in the order of
an event, as one stream's after the other. Each test prints its case first."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["i8", "f16"])
def test_stores_on_two_streams(dtype):
    from diffusorrt_amd.kernels import PrefixKVCache

    print("[case] stores on two streams", dtype, flush=True)
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn((4096, 2, 128), generator=gen).cuda() for _ in range(2))
    one, two = (PrefixKVCache(1, 2, 4096, dtype=dtype, block_sums=True) for _ in range(2))

    def store(cache, lo, hi):
        cache.store(0, k[lo:hi], v[lo:hi], lo)

    a, b = (torch.cuda.Stream() for _ in range(2))
    done = torch.cuda.Event()
    torch.cuda.synchronize()
    for i in range(0, 4096, 1024):
        with torch.cuda.stream(a):  # whole tiles, then half of one
            store(two, i, i + 512)
            store(two, i + 992, i + 1009)
            done.record()
        with torch.cuda.stream(b):  # whole tiles beside them, then that tile's other rows
            store(two, i + 512, i + 992)
            b.wait_event(done)
            store(two, i + 1009, i + 1024)
    torch.cuda.synchronize()
    for i in range(0, 4096, 1024):
        for lo, hi in ((0, 512), (512, 992), (992, 1009), (1009, 1024)):
            store(one, i + lo, i + hi)
    assert torch.equal(one.data, two.data) and torch.equal(one.sums, two.sums)
    assert one.scales is None or torch.equal(one.scales, two.scales)

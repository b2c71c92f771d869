"""Attention over a paged cache in units of 64 query vectors against 64 bits on the GPU: masks, head groups,
ragged batches beside units of 32, cut and whole, places that are not seen, many small weights."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_paged_large import TYPES, Batch

pytestmark = pytest.mark.gpu


class Medium(Batch):
    def wide(self):
        info = self.batch.info
        words = self.batch._list.cpu().numpy()
        return int(words[info.small:info.small + 16 * info.n_small].reshape(-1, 16)[:, 11].sum())

    def check(self, out="f32", cut=None):
        assert self.wide() > 0 and self.batch.info.n_large == 0
        assert cut is None or (self.batch.info.slots > 0) == cut
        got = self.cache.attention(0, self.q, self.batch, out_dtype=TYPES[out]).double()
        want, bound = self.want(out)
        off = (got.view_as(want) - want).abs()
        assert (off <= bound).all(), (float((off - bound).max()), int(off.isnan().sum()))
        return got


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("mask, geometry", [("causal", None), ("full", None), ("d2f_hybrid", (5900, 32)),
                                            ("d2f_hybrid", (0, 1000))])
def test_masks(kind, mask, geometry):
    Medium([6001], [150], g=7, hkv=4, kind=kind, mask=mask, geometry=geometry).check(cut=True)


@pytest.mark.parametrize("g, hkv, rows, keys, size", [(3, 5, 333, 9000, 32), (2, 16, 400, 5000, 256),
                                                      (7, 4, 150, 20000, 64)])
def test_head_groups(g, hkv, rows, keys, size):
    Medium([keys], [rows], g=g, hkv=hkv, size=size, seed=g).check("bf16")


def test_whole_units_of_many_sequences():
    b = Medium([3000] * 16, [20] * 16, g=7, hkv=4, kind="f16")
    got = b.check(cut=False)
    for _ in range(3):  # the same from call to call
        assert torch.equal(b.cache.attention(0, b.q, b.batch).double(), got)


def test_rows_without_keys_beside_others():
    b = Medium([9000, 0, 300, 4000], [100, 30, 1, 100], g=7, hkv=4, mask="full",
               positions=[8900, 0, 299, 3900])
    got = b.check()
    assert (got[100:130] == 0).all()


def test_large_scores():
    Medium([6001], [150], g=7, hkv=4, scale=1e4, seed=4).check()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_where_a_row_does_not_see_them(kind, what):
    b = Medium([6001], [150], g=7, hkv=4, kind=kind)
    assert b.wide() > 0
    want, bound = b.want()
    at = 6001 - 150 + 70
    b.k[at + 1, 0, 5] = what
    b.v[at, 3, 9] = what
    b.fill()
    got = b.cache.attention(0, b.q, b.batch).double().view_as(want)
    ok = (got - want).abs() <= bound
    assert ok[:70].all()        # rows that see neither
    assert ok[70, :21].all()    # K at + 1 is seen from row 71 on, by the heads of the first K/V head
    assert ok[70:, 7:21].all()
    if not np.isinf(what):
        assert not torch.isfinite(got[71:, :7]).any()
    other = np.delete(np.arange(128), 9)
    assert ok[70:, 21:][..., other].all()
    seen = got[70:, 21:, 9]
    assert (seen.isnan() if np.isnan(what) else seen == what).all()


def test_many_small_weights_add_up():
    # one key of each of the first four tiles scores 15.125, the others 0 and weigh 2^-21.8 of it each; their
    # values are 1 and the four's 0. fp16 weights of 2^7 times as much are off by 2^-10.2 of themselves at most,
    # the largest by 2^-11, both by their scores' sums of 130 fp32 roundings of 15.125 (2^-12.9) and the
    # power (2^-18)
    a = 1.15625
    b = Medium([5000], [400], g=2, hkv=16, kind="f16", mask="full")
    assert b.wide() > 0 and not b.batch.info.slots
    b.q.fill_(a)
    b.k.zero_()
    b.v.fill_(1.0)
    b.k[:128:32] = a
    b.v[:128:32] = 0.0
    b.fill()
    got = b.cache.attention(0, b.q, b.batch).double()
    w = 4996 * np.exp(-a * a * 128**0.5)
    assert (got / (w / (4 + w)) - 1).abs().max() < 2**-10.2 + 2**-11 + 2 * 2**-12.9 + 2**-17


def test_graph_and_other_streams():
    b = Medium([6001, 50], [150, 1], g=7, hkv=4)
    assert b.wide() > 0
    want = b.cache.attention(0, b.q, b.batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = b.cache.attention(0, b.q, b.batch)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.cache.attention(0, b.q, b.batch)
    for _ in range(3):
        b.q.mul_(-0.5)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, b.cache.attention(0, b.q, b.batch))
        torch.cuda.synchronize()

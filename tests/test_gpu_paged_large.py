"""Attention of many rows over a paged cache (the kernel of 256 query vectors, whole units and equal
shares) against 64 bits on the GPU: masks, head groups, ragged batches, other sequences beside, places
that are not seen."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diffusorrt_amd.paged import PagedKVCache
from oracle import paged as P

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _randn(seed, *shape, dtype, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _want(q, k, v, ends, kind, out, rows_at_once=512):
    """oracle.paged.attention of one sequence in float64 on the GPU. Its bound with |v - o| as |v| + |o|."""
    q, k, v = q.double(), k.double(), v.double()
    g = q.shape[1] // k.shape[1]
    ends = torch.tensor(ends, device="cuda")
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    if not k.shape[0]:
        return o, bound
    at = torch.arange(k.shape[0], device="cuda")
    for h in range(q.shape[1]):
        kk, vv = k[:, h // g], v[:, h // g]
        for r in range(0, q.shape[0], rows_at_once):
            part = slice(r, r + rows_at_once)
            unseen = at >= ends[part, None]
            none = (ends[part] == 0)[:, None]
            s = (q[part, h] @ kk.t() / 128**0.5).masked_fill(unseen, -torch.inf)
            w = (s - s.amax(-1, keepdim=True)).exp()
            w = torch.where(none, 0.0, w)
            total = w.sum(-1, keepdim=True).clamp_min(1e-300)
            w = w / total
            size = q[part, h].abs() @ kk.abs().t() / 128**0.5
            per = w * (P.HALF_STEP[kind] + 130 * 2.0**-24 * size + 2.0**-18)
            y = w @ vv
            b = per @ vv.abs() + y.abs() * per.sum(-1, keepdim=True) + \
                2.0**-18 * (w @ vv.abs() + y.abs())
            if kind == "f16":
                seen = (~unseen).double()
                b += 2.0**-25 / total * (seen @ vv.abs() + y.abs() * seen.sum(-1, keepdim=True))
            o[part, h], bound[part, h] = y, b + P.HALF_STEP[out] * (y.abs() + b)
    return o, bound


class Batch:
    def __init__(self, keys, rows, *, g, hkv, kind="bf16", mask="causal", geometry=None, size=64,
                 positions=None, stale=float("nan"), seed=0, scale=1.0):
        need = [-(-n // size) for n in keys]
        order = np.random.default_rng(seed).permutation(sum(need) + 3).tolist()
        table = [[order.pop() for _ in range(n)] for n in need]
        dtype = TYPES[kind]
        self.cache = PagedKVCache(1, hkv, sum(need) + 3, page_size=size, dtype=kind)
        self.cache.data.fill_(stale)
        self.k = _randn(seed + 1, sum(keys), hkv, 128, dtype=dtype)
        self.v = _randn(seed + 2, sum(keys), hkv, 128, dtype=dtype)
        self.q = _randn(seed + 3, sum(rows), hkv * g, 128, dtype=dtype, scale=scale)
        self.whole = self.cache.batch(table, keys, keys, heads=hkv)
        self.fill()
        self.batch = self.cache.batch(table, keys, rows, heads=hkv * g, positions=positions, kind=mask,
                                      mask_geometry=geometry)
        self.keys, self.rows, self.kind = keys, rows, kind
        self.ends = []
        for s, (n, k) in enumerate(zip(rows, keys)):
            pos0 = k - n if positions is None else positions[s]
            prompt, block = geometry or (0, 1)
            self.ends.append(P.key_ends(mask, pos0, n, k, prompt if isinstance(prompt, int) else prompt[s],
                                        block))

    def fill(self):
        self.cache.append(0, self.k, self.v, self.whole)

    def want(self, out="f32"):
        o, bound, r0, k0 = [], [], 0, 0
        for n, keys, ends in zip(self.rows, self.keys, self.ends):
            y, b = _want(self.q[r0:r0 + n], self.k[k0:k0 + keys], self.v[k0:k0 + keys], ends, self.kind, out)
            o.append(y)
            bound.append(b)
            r0, k0 = r0 + n, k0 + keys
        return torch.cat(o), torch.cat(bound)

    def check(self, out="f32", cut=None):
        assert self.batch.info.n_large > 0
        assert cut is None or (self.batch.info.slots > 0) == cut
        got = self.cache.attention(0, self.q, self.batch, out_dtype=TYPES[out]).double()
        want, bound = self.want(out)
        off = (got.view_as(want) - want).abs()
        assert (off <= bound).all(), (float((off - bound).max()), int(off.isnan().sum()))
        return got


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("mask, geometry", [("causal", None), ("full", None), ("d2f_hybrid", (5000, 32)),
                                            ("d2f_hybrid", (0, 1000))])
def test_masks(kind, mask, geometry):
    Batch([8001], [1023], g=2, hkv=64, kind=kind, mask=mask, geometry=geometry).check()


@pytest.mark.parametrize("g, hkv, rows, keys", [(1, 32, 2000, 9100), (7, 4, 2300, 9500), (40, 4, 400, 9000),
                                                (3, 64, 257, 5000), (5, 9, 1111, 19999)])
def test_head_groups(g, hkv, rows, keys):
    Batch([keys], [rows], g=g, hkv=hkv, seed=g).check("bf16")


@pytest.mark.parametrize("cut, rows, keys", [(False, 2048, 8192), (True, 600, 40000)])
def test_whole_units_and_shares(cut, rows, keys):
    b = Batch([keys], [rows], g=2, hkv=16, size=256, seed=1, scale=2.0)
    got = b.check(cut=cut)
    for _ in range(3):  # the same from call to call
        assert torch.equal(b.cache.attention(0, b.q, b.batch).double(), got)


def test_ragged_sequences_beside_small_ones():
    b = Batch([6000, 33, 4100, 1, 5000, 64, 300], [700, 1, 400, 1, 650, 64, 0], g=2, hkv=16, kind="f16",
              size=32)
    assert b.batch.info.n_small > 0
    b.check()


def test_rows_without_keys_beside_others():
    b = Batch([9000, 0, 40], [1900, 300, 5], g=2, hkv=32, mask="full", positions=[7100, 0, 35])
    got = b.check()
    assert (got[1900:2200] == 0).all()


def test_from_the_first_key_on():
    Batch([6000, 100], [6000, 100], g=4, hkv=16).check()


def test_large_scores():
    Batch([9000], [2048], g=2, hkv=16, scale=1e4, seed=4).check()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_where_a_row_does_not_see_them(kind, what):
    b = Batch([9000], [2048], g=2, hkv=16, kind=kind)
    want, bound = b.want()
    at = 9000 - 2048 + 500
    b.k[at + 1, 0, 5] = what
    b.v[at, 3, 9] = what
    b.fill()
    assert b.batch.info.n_large
    got = b.cache.attention(0, b.q, b.batch).double().view_as(want)
    ok = (got - want).abs() <= bound
    assert ok[:500].all()
    assert ok[500, :2].all()
    other = torch.ones(128, dtype=torch.bool, device="cuda")
    other[9] = False
    assert ok[500:, 2:][..., other].all()
    heads = torch.ones(32, dtype=torch.bool, device="cuda")
    heads[:2] = heads[6:8] = False
    assert ok[:, heads].all()
    seen = got[500:, 6:8, 9]
    assert not torch.isfinite(seen).any()
    if not np.isinf(what):
        assert not torch.isfinite(got[501:, :2]).any()


def test_graph_and_other_streams():
    b = Batch([9000, 50], [2000, 1], g=2, hkv=16)
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


def test_many_small_weights_add_up():
    # one key of each of the first two tiles scores 15.125, the others 0 and weigh 2^-21.8 of it each: the
    # bound of a row's result, whose values are 1 there and 0 at the two, is that of fp16 weights of 2^7
    # times as much (off by 2^-10.2 of themselves at most, the largest by 2^-11, both by their scores' sums
    # of 130 fp32 roundings of 15.125, 2^-12.9, and the power, 2^-18)
    a = 1.15625
    b = Batch([4096], [2048], g=2, hkv=16, kind="f16", mask="full")
    assert b.batch.info.n_large > 0 and not b.batch.info.slots
    b.q.fill_(a)
    b.k.zero_()
    b.v.fill_(1.0)
    b.k[:64:32] = a
    b.v[:64:32] = 0.0
    b.fill()
    got = b.cache.attention(0, b.q, b.batch).double()
    w = 4094 * np.exp(-a * a * 128**0.5)
    assert (got / (w / (2 + w)) - 1).abs().max() < 2**-10.2 + 2**-11 + 2 * 2**-12.9 + 2**-17


def test_values_near_the_types_largest():
    b = Batch([4096], [2048], g=2, hkv=16, mask="full", kind="bf16")
    b.q.zero_()
    b.v[..., 9] = 3e38
    b.v[..., 10] = -3e38
    b.fill()
    b.check()

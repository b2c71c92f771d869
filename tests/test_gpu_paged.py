"""The paged cache against 64 bits: appends (rotated, of any type and strides, into any part of a page),
reading back, attention of ragged batches under every mask, what lies behind a sequence's keys, streams,
graphs and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diffusorrt_amd.paged import PagedKVCache
from diffusorrt_amd.rotary import RotaryPositions
from oracle import paged as P

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _np(t):
    return t.detach().double().cpu().numpy()


def _randn(seed, *shape, dtype=torch.float32, scale=1.0):
    x = torch.from_numpy(np.random.default_rng(seed).standard_normal(shape, np.float32))
    return (x * scale).to(dtype).cuda()


def _tables(seed, keys, size, spare=3):
    need = [-(-k // size) for k in keys]
    order = np.random.default_rng(seed).permutation(sum(need) + spare).tolist()
    return [[order.pop() for _ in range(n)] for n in need], sum(need) + spare


class Sequences:
    """Sequences in a cache whose every other place holds `stale`."""

    def __init__(self, keys, rows, *, g=2, hkv=2, size=64, kind="f16", mask="causal", geometry=None,
                 positions=None, stale=0.0, seed=0, layers=1, layer=0, scale=1.0):
        self.keys, self.rows, self.kind, self.mask = keys, rows, kind, mask
        self.positions, self.geometry = positions, geometry
        self.table, pages = _tables(seed, keys, size)
        self.cache = PagedKVCache(layers, hkv, pages, page_size=size, dtype=kind)
        self.cache.data.fill_(stale)
        self.layer = layer
        dtype = TYPES[kind]
        total = sum(keys)
        self.k = _randn(seed + 1, max(total, 1), hkv, 128, dtype=dtype)[:total]
        self.v = _randn(seed + 2, max(total, 1), hkv, 128, dtype=dtype)[:total]
        self.fill()
        self.q = _randn(seed + 3, sum(rows), hkv * g, 128, dtype=dtype, scale=scale)
        self.batch = self.cache.batch(self.table, keys, rows, heads=hkv * g, positions=positions,
                                      kind=mask, mask_geometry=geometry)

    def fill(self):
        if sum(self.keys):
            b = self.cache.batch(self.table, self.keys, self.keys, heads=self.cache.kv_heads)
            self.cache.append(self.layer, self.k, self.v, b)

    def want(self, out="f32"):
        o, bound, r0, k0 = [], [], 0, 0
        q, k, v = _np(self.q), _np(self.k), _np(self.v)
        for s, (n, keys) in enumerate(zip(self.rows, self.keys)):
            pos0 = keys - n if self.positions is None else self.positions[s]
            prompt, block = self.geometry or (0, 1)
            prompt = prompt if isinstance(prompt, int) else prompt[s]
            ends = P.key_ends(self.mask, pos0, n, keys, prompt, block)
            x = P.attention(q[r0:r0 + n], k[k0:k0 + keys], v[k0:k0 + keys], ends, self.kind, out)
            o.append(x[0])
            bound.append(x[1])
            r0, k0 = r0 + n, k0 + keys
        return np.concatenate(o), np.concatenate(bound)

    def check(self, out="f32"):
        got = self.cache.attention(self.layer, self.q, self.batch, out_dtype=TYPES[out])
        assert got.dtype == TYPES[out]
        want, bound = self.want(out)
        off = np.abs(_np(got).reshape(want.shape) - want)
        assert (off <= bound).all(), (float(np.nanmax(off - bound)), np.isnan(off).sum())
        return got


# ---------------------------------------------------------------- append, load

@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("layout, dim", [("half", 128), ("interleaved", 128), ("half", 96),
                                         ("interleaved", 16)])
def test_append_turns_keys_and_queries(src, kind, layout, dim):
    keys, rows = [40, 5, 200, 64, 1], [37, 1, 70, 0, 1]
    hq, hkv = 14, 2
    table, pages = _tables(1, keys, 64)
    cache = PagedKVCache(2, hkv, pages, page_size=64, dtype=kind)
    cache.data.fill_(7.0)
    n = sum(rows)
    fused = _randn(2, n, (hq + 2 * hkv) * 128 + 3, dtype=TYPES[src])[:, 3:].view(n, hq + 2 * hkv, 128)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    rotary = RotaryPositions(dim, layout=layout, scaling={"type": "yarn", "factor": 4.0,
                                                          "original_max_position_embeddings": 64})
    batch = cache.batch(table, keys, rows, heads=hq)
    out = cache.append(1, k, v, batch, rotary=rotary, q=q)
    k2, v2 = cache.load(1, batch)
    assert out.dtype == k2.dtype == v2.dtype == TYPES[kind]
    pos = np.concatenate([np.arange(a - b, a) for a, b in zip(keys, rows)])
    for x, y in ((q, out), (k, k2)):
        want = P.rotate(_np(x), pos, rotary.frequencies, rotary.magnitude, layout)
        bound = P.rotate_bound(_np(x), want, rotary.frequencies, rotary.magnitude, layout, kind)
        bound[..., dim:] = P.HALF_STEP[kind] * np.abs(want[..., dim:]) + 2.0**-25
        assert (np.abs(_np(y) - want) <= bound).all()
    assert torch.equal(v2, v.to(TYPES[kind]))
    # the other layer, and every place of this one that no row has, as they were
    assert (cache.data[0] == 7.0).all()
    assert int((cache.data[1] != 7.0).sum()) <= 2 * n * hkv * 128
    whole = cache.batch(table, keys, keys, heads=hq)
    k3, _ = cache.load(1, whole)
    new = np.concatenate([np.arange(a) >= a - b for a, b in zip(keys, rows)])
    assert torch.equal(k3[torch.from_numpy(new).cuda()], k2)
    assert (k3[torch.from_numpy(~new).cuda()] == 7.0).all()


@pytest.mark.parametrize("size", [32, 64, 512])
@pytest.mark.parametrize("pos0, n", [(0, 1), (31, 1), (31, 2), (5, 3), (0, 32), (0, 33), (17, 300),
                                     (500, 40)])
def test_rows_around_an_append_stay(size, pos0, n):
    keys = 600
    table, pages = _tables(3, [keys], size)
    cache = PagedKVCache(1, 3, pages, page_size=size, dtype="bf16")
    k, v = _randn(4, keys, 3, 128, dtype=torch.bfloat16), _randn(5, keys, 3, 128, dtype=torch.bfloat16)
    whole = cache.batch(table, [keys], [keys], heads=3)
    cache.append(0, k, v, whole)
    assert all(torch.equal(a, b) for a, b in zip(cache.load(0, whole), (k, v)))
    before = cache.data.clone()
    a, b = _randn(6, n, 3, 128, dtype=torch.bfloat16), _randn(7, n, 3, 128, dtype=torch.bfloat16)
    part = cache.batch(table, [keys], [n], heads=3, positions=[pos0])
    cache.append(0, a, b, part)
    k[pos0:pos0 + n], v[pos0:pos0 + n] = a, b
    assert all(torch.equal(x, y) for x, y in zip(cache.load(0, whole), (k, v)))
    assert all(torch.equal(x, y) for x, y in zip(cache.load(0, part), (a, b)))
    cache.append(0, k, v, whole)
    old = torch.full((n, 3, 128), 0.0, dtype=torch.bfloat16, device="cuda")
    cache.append(0, old, old, part)
    assert int((cache.data != before).sum()) <= 2 * n * 3 * 128


def test_append_many_heads_and_no_queries():
    hkv = 40
    cache = PagedKVCache(1, hkv, 9, page_size=32)
    k, v = _randn(8, 70, hkv, 128), _randn(9, 70, hkv, 128)
    batch = cache.batch([[8, 0, 5]], [70], [70], heads=hkv)
    assert cache.append(0, k, v, batch) is None
    k2, v2 = cache.load(0, batch)
    assert torch.equal(k2, k.half()) and torch.equal(v2, v.half())


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("mask, geometry", [("full", None), ("causal", None), ("d2f_hybrid", (0, 32)),
                                            ("d2f_hybrid", ([3, 50, 0, 0, 700, 9], 8))])
@pytest.mark.parametrize("g, hkv", [(2, 8), (7, 4)])
def test_ragged_batches(kind, mask, geometry, g, hkv):
    s = Sequences([700, 33, 1, 64, 301, 95], [1, 9, 1, 32, 80, 0], g=g, hkv=hkv, kind=kind, mask=mask,
                  geometry=geometry, stale=float("nan"))
    s.check("f32")
    s.check("bf16")


@pytest.mark.parametrize("keys", [0, 1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1000, 4100])
def test_one_token(keys):
    s = Sequences([keys], [1], hkv=2, mask="full", positions=[keys], stale=float("inf"), seed=keys)
    got = s.check()
    if not keys:
        assert (got == 0).all()


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 63, 65, 100, 127, 129, 200, 300])
@pytest.mark.parametrize("mask", ["full", "causal"])
def test_rows(rows, mask):
    Sequences([rows + 150, rows], [rows, rows], hkv=2, g=2, mask=mask, seed=rows, kind="bf16",
              size=32).check()


@pytest.mark.parametrize("g, hkv", [(1, 1), (1, 3), (3, 2), (5, 1), (8, 2), (33, 1), (64, 2)])
def test_head_groups(g, hkv):
    Sequences([90, 500], [3, 20], g=g, hkv=hkv, seed=g, stale=float("nan")).check()


@pytest.mark.parametrize("size", [32, 128, 4096])
def test_page_sizes(size):
    Sequences([5000, 31, 129], [40, 31, 1], size=size, seed=size, stale=float("nan")).check()


def test_no_keys_beside_others():
    s = Sequences([0, 40, 0], [3, 2, 200], mask="full", positions=[0, 38, 5], stale=float("nan"))
    got = s.check()
    assert (got[:3] == 0).all() and (got[5:] == 0).all()


def test_positions_beyond_the_keys_see_all():
    # rows that are not among the keys (a prefix alone is in the cache)
    Sequences([100, 64], [5, 9], positions=[100, 1000]).check()


@pytest.mark.parametrize("rows, keys", [(1, 70000), (4, 33000), (32, 20000), (300, 9000)])
def test_long_sequences(rows, keys):
    Sequences([keys, 77], [rows, 1], g=2, hkv=1, size=128, kind="bf16", seed=keys, scale=2.0).check()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_large_scores(kind):
    # bases far from zero, and one key that takes all
    s = Sequences([400, 90], [20, 1], kind=kind, scale=60.0 if kind == "f16" else 1e4, seed=3)
    s.check()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rows", [9, 130])
def test_values_that_are_not_finite_where_a_row_does_not_see_them(kind, what, rows):
    s = Sequences([200], [rows], kind=kind, hkv=2, g=2)
    want, bound = s.want()
    first = 200 - rows
    at = first + rows // 2        # rows below do not see key `at`
    s.k[at + 1, 0, 5] = what
    s.v[at, 1, 9] = what
    s.fill()
    got = _np(s.cache.attention(0, s.q, s.batch)).reshape(want.shape)
    off = np.abs(got - want)
    below = rows // 2
    assert (off[:below] <= bound[:below]).all()
    # K: the rows that see it, of its head's group; V: the one head dim
    assert (off[below:below + 1, :2] <= bound[below:below + 1, :2]).all()
    if not np.isinf(what):
        assert not np.isfinite(got[below + 1:, :2]).any()
    assert not np.isfinite(got[below:, 2:, 9]).any()
    other = np.delete(np.arange(128), 9)
    assert (off[below:, 2:][..., other] <= bound[below:, 2:][..., other]).all()
    if np.isinf(what):
        assert (got[below:, 2:, 9] == what).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_many_small_weights_add_up(rows):
    # One key of each of the first eight tiles scores a^2 128 / sqrt(128) = 15.125, the others 0, so each of
    # those weighs 2^-21.8 of it; their values are 1 and the others' 0. A weight of 2^7 2^-21.8 is off by
    # 2^-25 at most in fp16, 2^-10.2 of itself, the largest by 2^-11, both by their scores' sums (130
    # roundings of 15.125 in fp32, 2^-12.9) and the power (2^-18).
    a = 1.15625
    s = Sequences([1024], [rows], kind="f16", mask="full", hkv=2, g=1)
    s.q.fill_(a)
    s.k.zero_()
    s.v.fill_(1.0)
    s.k[:256:32] = a
    s.v[:256:32] = 0.0
    s.fill()
    got = _np(s.cache.attention(0, s.q, s.batch))
    w = 1016 * np.exp(-a * a * 128**0.5)
    assert np.abs(got / (w / (8 + w)) - 1).max() < 2**-10.2 + 2**-11 + 2 * 2**-12.9 + 2**-17


@pytest.mark.parametrize("rows", [1, 40])
def test_values_near_the_types_largest(rows):
    # bf16: sums ahead of the division stay finite; q of zeros, so every weight is the same
    s = Sequences([500, 3], [rows, 1], kind="bf16", mask="full")
    s.q.zero_()
    s.v[..., 9] = 3e38
    s.v[..., 10] = -3e38
    s.fill()
    s.check()


def test_places_beyond_4_gib():
    # the last pages of a layer of 5.4 GB, and of the second layer
    cache = PagedKVCache(2, 8, 20480, page_size=64, dtype="bf16")
    assert cache.data[0].numel() * 2 > 2**32
    keys = 3000
    table = [list(range(20479, 20479 - 47, -1))]
    k, v = (_randn(i, keys, 8, 128, dtype=torch.bfloat16) for i in (1, 2))
    q = _randn(3, 5, 16, 128, dtype=torch.bfloat16)
    whole, batch = cache.batch(table, [keys], [keys], heads=16), cache.batch(table, [keys], [5], heads=16)
    small = PagedKVCache(1, 8, 47, page_size=64, dtype="bf16")
    table2 = [list(range(47))]
    small.append(0, k, v, small.batch(table2, [keys], [keys], heads=16))
    want = small.attention(0, q, small.batch(table2, [keys], [5], heads=16))
    for layer in (0, 1):
        cache.append(layer, k, v, whole)
        assert all(torch.equal(a, b) for a, b in zip(cache.load(layer, whole), (k, v)))
        assert torch.equal(cache.attention(layer, q, batch), want)


def test_a_prefix_in_common():
    cache = PagedKVCache(1, 2, 8, page_size=64)
    k, v = _randn(1, 128, 2, 128), _randn(2, 128, 2, 128)
    cache.append(0, k, v, cache.batch([[5, 2]], [128], [128], heads=4))
    batch = cache.batch([[5, 2, 1], [5, 2, 7], [5]], [131, 129, 64], [3, 1, 0], heads=4)
    rotary = RotaryPositions(128)
    k2, v2, q2 = _randn(3, 4, 2, 128), _randn(4, 4, 2, 128), _randn(5, 4, 4, 128)
    q = cache.append(0, k2, v2, batch, rotary=rotary, q=q2)
    out = cache.attention(0, q, batch)
    held, _ = cache.load(0, batch)
    for rows, at, keys in ((slice(0, 3), 128, 131), (slice(3, 4), 128, 129)):
        ks = np.concatenate([_np(k.half()), _np(held[rows])])
        vs = np.concatenate([_np(v.half()), _np(v2[rows].half())])
        n = keys - at
        want, bound = P.attention(_np(q[rows]), ks, vs, P.key_ends("causal", at, n, keys))
        assert (np.abs(_np(out[rows]).reshape(want.shape) - want) <= bound).all()


def test_steps_of_a_prompt_and_its_tokens_equal_one_pass():
    """A run of them as they are used: chunks, then tokens, of two layers; every row's result as of the
    whole sequence's attention in 64 bits over the turned keys."""
    hq, hkv, n = 14, 2, 300
    rotary = RotaryPositions(128)
    cache = PagedKVCache(2, hkv, 12, page_size=32, dtype="bf16")
    q, k, v = (_randn(i, n, h, 128) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    table = [[7, 3, 0, 11, 5, 2, 9, 1, 10, 4]]
    outs, turned, at = [], [], 0
    for step in [130, 70, 33, 1, 1, 1, 9, 55]:
        batch = cache.batch(table, [at + step], [step], heads=hq)
        rows = slice(at, at + step)
        for layer in (0, 1):
            q2 = cache.append(layer, k[rows], v[rows] * (1 + layer), batch, rotary=rotary, q=q[rows])
            out = cache.attention(layer, q2, batch)
        outs.append(out)
        turned.append(q2)
        at += step
    whole = cache.batch(table, [n], [n], heads=hq)
    held = cache.load(1, whole)
    want, bound = P.attention(_np(torch.cat(turned)), _np(held[0]), _np(held[1]),
                              P.key_ends("causal", 0, n, n), "bf16")
    assert (np.abs(_np(torch.cat(outs)).reshape(want.shape) - want) <= bound).all()
    exact = P.rotate(_np(k), np.arange(n), rotary.frequencies)
    assert (np.abs(_np(held[0]) - exact) <= P.rotate_bound(_np(k), exact, rotary.frequencies, 1.0,
                                                          "half", "bf16")).all()
    assert torch.equal(held[1], (2 * v).bfloat16())


# ---------------------------------------------------------------- streams, graphs, refusals

def test_results_do_not_change_from_call_to_call():
    s = Sequences([5000, 300, 64], [1, 9, 64], hkv=4, g=7, kind="bf16", size=32)
    want = s.cache.attention(0, s.q, s.batch)
    for _ in range(5):
        assert torch.equal(s.cache.attention(0, s.q, s.batch), want)


def test_other_streams():
    s = Sequences([3000, 77], [1, 40], hkv=2, g=2)
    want = s.cache.attention(0, s.q, s.batch)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for side in sides * 3:
        with torch.cuda.stream(side):
            outs.append(s.cache.attention(0, s.q, s.batch))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    with torch.cuda.stream(sides[0]):  # a batch of another stream's, used here at once
        batch = s.cache.batch(s.table, s.keys, s.rows, heads=4)
    sides[1].wait_stream(sides[0])
    assert torch.equal(s.cache.attention(0, s.q, batch), want)


def test_two_captured_graphs_replayed_in_turn():
    s = Sequences([3000, 77], [1, 40], hkv=2, g=2, kind="bf16")
    rotary = RotaryPositions(128)
    k, v, x = (_randn(i, 41, h, 128) for i, h in ((11, 2), (12, 2), (13, 4)))

    def step():
        q = s.cache.append(0, k, v, s.batch, rotary=rotary, q=x)
        return s.cache.attention(0, q, s.batch)

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(3):
        x.add_(0.25 * i)
        k.mul_(-1)
        for g, out in graphs:
            g.replay()
            got = out.clone()
            assert torch.equal(got, step())
            torch.cuda.synchronize()
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], graphs[1][1])


def test_refusals():
    s = Sequences([100, 64], [5, 9])
    c, b, q = s.cache, s.batch, s.q
    other = PagedKVCache(1, 2, 99, page_size=64)
    k = torch.zeros(14, 2, 128, device="cuda")
    qf = torch.zeros(14, 4, 128, device="cuda")
    bad = [
        lambda: c.attention(1, q, b), lambda: c.attention(-1, q, b), lambda: other.attention(0, q, b),
        lambda: c.attention(0, q, s.table), lambda: c.attention(0, q[:13], b),
        lambda: c.attention(0, q.float(), b), lambda: c.attention(0, q.bfloat16(), b),
        lambda: c.attention(0, q.cpu(), b), lambda: c.attention(0, q[:, :2], b),
        lambda: c.attention(0, q.transpose(0, 1).contiguous().transpose(0, 1), b),
        lambda: c.attention(0, q, b, out_dtype=torch.float16),
        lambda: c.append(0, k[:3], k, b), lambda: c.append(0, k, k.half(), b),
        lambda: c.append(0, k.double(), k.double(), b), lambda: c.append(0, k, k, b, q=qf[:, :2]),
        lambda: c.append(0, k, k, b, q=qf.half()), lambda: c.append(0, k.cpu(), k, b),
        lambda: c.append(0, k, k, b, rotary=RotaryPositions(24)),
        lambda: c.append(0, k, k, b, rotary=RotaryPositions(130)),
        lambda: c.append(0, torch.zeros(14, 128, 2, device="cuda").transpose(1, 2), k, b),
        lambda: c.append(2, k, k, b), lambda: c.load(-1, b),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="captured"):
        with torch.cuda.graph(graph):
            c.batch(s.table, [100, 64], [5, 9], heads=4)
    behind = c.batch(s.table, [100, 64], [5, 9], heads=4, positions=[98, 0])
    twice = c.batch([s.table[0], s.table[0]], [100, 100], [5, 9], heads=4)
    for batch in (behind, twice):
        with pytest.raises(ValueError, match="tile"):
            c.append(0, k, k, batch)
        with pytest.raises(ValueError, match="tile"):
            c.load(0, batch)
        assert torch.isfinite(c.attention(0, q, batch)).all()


# ---------------------------------------------------------------- every key once

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("mask, geometry", [("full", None), ("causal", None), ("d2f_hybrid", (70, 32))])
@pytest.mark.parametrize("keys, rows, g, hkv", [
    ([1, 31, 33, 500, 4100], [1, 9, 1, 100, 1], 2, 2), ([70000], [1], 2, 2), ([20000, 64], [40, 64], 7, 1),
    ([3000], [300], 2, 16),
    ([8200, 77], [1024, 5], 2, 16),   # the kernel of many rows, whole units
    ([16384], [600], 2, 16)])         # ... and equal shares
def test_every_key_counts_once(keys, rows, g, hkv, kind, mask, geometry):
    """Queries of zero weigh all keys alike, exactly: with values that are small whole numbers the result is
    their sum, exact in 32 bits, over their number. A key left out, read twice or seen by a row that does
    not see it moves some of the 128 sums by a whole number."""
    table, pages = _tables(1, keys, 64)
    cache = PagedKVCache(1, hkv, pages, page_size=64, dtype=kind)
    cache.data.fill_(float("nan"))
    total, dtype = sum(keys), TYPES[kind]
    gen = torch.Generator(device="cuda").manual_seed(total)
    v = torch.randint(-3, 4, (total, hkv, 128), generator=gen, device="cuda")
    k = torch.randn((total, hkv, 128), generator=gen, device="cuda").to(dtype)
    cache.append(0, k, v.to(dtype), cache.batch(table, keys, keys, heads=hkv))
    batch = cache.batch(table, keys, rows, heads=g * hkv, kind=mask, mask_geometry=geometry)
    q = torch.zeros(sum(rows), g * hkv, 128, dtype=dtype, device="cuda")
    out = cache.attention(0, q, batch).view(-1, g * hkv, 128).double()
    r0 = k0 = 0
    for n, r in zip(keys, rows):
        ends = torch.tensor(P.key_ends(mask, n - r, r, n, *(geometry or (0, 1))), device="cuda")
        sums = v[k0:k0 + n].cumsum(0)[ends - 1].repeat_interleave(g, 1).double()
        want = sums / ends[:, None, None]
        # one division (and its reciprocal) and, in parts, a product with a power of two
        assert ((out[r0:r0 + r] - want).abs() <= 2.0**-22 * want.abs()).all()
        r0, k0 = r0 + r, k0 + n

"""RotaryPositions.rotate against its formula in 64 bits: types, layouts, sizes, strides, positions of 32
bits, in place, backwards, and its refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diffusorrt_amd.rotary import RotaryPositions
from oracle import paged as P

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _x(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape, np.float32)).cuda()


def _check(rotary, x, positions, got, kind, inverse=False):
    xs, pos = x.float().cpu().numpy(), np.asarray(positions, np.float64)
    want = P.rotate(xs, pos, rotary.frequencies, rotary.magnitude, rotary.layout, inverse)
    # (the oracle's own angle: p f rounds to 2^-53 of itself)
    angle = 2.0**-22 + np.abs(pos).max() * max(np.abs(rotary.frequencies)) * 2.0**-52
    bound = P.rotate_bound(xs, want, rotary.frequencies, rotary.magnitude, rotary.layout, kind, angle)
    off = np.abs(got.float().cpu().numpy() - want)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert (off <= bound).all(), (off - bound).max()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim, hd", [(128, 128), (64, 128), (96, 128), (32, 40), (8, 8), (2, 128),
                                     (72, 128), (6, 10), (64, 64), (250, 256)])
def test_sizes(kind, layout, dim, hd):
    rows, heads = 37, 5
    x = _x(dim, rows, heads, hd).to(TYPES[kind])
    positions = np.random.default_rng(1).integers(0, 200000, rows)
    rotary = RotaryPositions(dim, layout=layout)
    got = rotary.rotate(x, torch.tensor(positions, dtype=torch.int32, device="cuda"))
    _check(rotary, x, positions, got, kind)
    assert torch.equal(got[..., dim:], x[..., dim:])


@pytest.mark.parametrize("rows, heads", [(1, 1), (1, 28), (2, 16), (1000, 28), (4099, 16)])
def test_rows(rows, heads):
    x = _x(rows, rows, heads, 128).bfloat16()
    rotary = RotaryPositions(scaling={"type": "yarn", "factor": 4.0,
                                      "original_max_position_embeddings": 32768})
    _check(rotary, x, 131000 + np.arange(rows), rotary.rotate(x, 131000), "bf16")


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 3.0},
                                     {"type": "ntk", "factor": 3.0},
                                     {"type": "yarn", "factor": 8.0, "attention_factor": 0.7,
                                      "original_max_position_embeddings": 4096}])
def test_scalings(scaling):
    x = _x(7, 50, 3, 128)
    rotary = RotaryPositions(128, theta=1e4, scaling=scaling)
    pos = np.random.default_rng(2).integers(0, 40000, 50)
    _check(rotary, x, pos, rotary.rotate(x, torch.tensor(pos, dtype=torch.int32, device="cuda")),
           "f32")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_of_32_bits(layout):
    pos = [0, 1, -1, 2**24 + 1, -2**24 - 1, 2**31 - 1, -2**31, 12345678]
    # frequencies that a double holds with its product with any position: the oracle's angles are exact
    rotary = RotaryPositions(16, layout=layout, frequencies=[1.0, 0.5, 0.75, 2**-10, 3.0, 0.25, -1.0, 0.0])
    x = _x(3, len(pos), 2, 16)
    _check(rotary, x, pos, rotary.rotate(x, torch.tensor(pos, dtype=torch.int32, device="cuda")), "f32")
    got = rotary.rotate(x, torch.zeros(len(pos), dtype=torch.int32, device="cuda"))
    assert torch.equal(got, x)  # position zero turns nothing


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("layout, dim", [("half", 128), ("interleaved", 64), ("half", 6)])
def test_strides_in_place_and_out(kind, layout, dim):
    rotary = RotaryPositions(dim, layout=layout)
    fused = _x(4, 33, 9, 131).to(TYPES[kind])[:, :, 3:]  # neither rows nor heads side by side, unaligned
    x = fused[:, 2:7]
    want = rotary.rotate(x.contiguous(), 100)
    _check(rotary, x, 100 + np.arange(33), want, kind)
    assert torch.equal(rotary.rotate(x, 100), want)
    y = torch.full((33, 11, 128), 3.0, dtype=x.dtype, device="cuda")
    assert rotary.rotate(x, 100, out=y[:, 4:9]).data_ptr() == y[:, 4:9].data_ptr()
    assert torch.equal(y[:, 4:9], want) and (y[:, :4] == 3).all() and (y[:, 9:] == 3).all()
    one = x[:, :1].expand(33, 5, 128)  # a head that five share
    assert torch.equal(rotary.rotate(one, 100), rotary.rotate(one.contiguous(), 100))
    before = fused.clone()
    rotary.rotate(x, 100, out=x)
    assert torch.equal(x, want) and torch.equal(fused[:, :2], before[:, :2]) and \
        torch.equal(fused[:, 7:], before[:, 7:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_gradient(layout):
    rotary = RotaryPositions(64, layout=layout, scaling={"type": "yarn", "factor": 4.0,
                                                        "original_max_position_embeddings": 8192})
    x, g = _x(5, 20, 3, 128), _x(6, 20, 3, 128)
    pos = np.arange(20) * 1001
    at = torch.tensor(pos, dtype=torch.int32, device="cuda")
    back = rotary.rotate(g, at, inverse=True)
    _check(rotary, g, pos, back, "f32", inverse=True)
    # <rotate(x), g> = <x, rotate back(g)>, and differences of the formula along a direction
    y = P.rotate(x.cpu().numpy(), pos, rotary.frequencies, rotary.magnitude, layout)
    gd = g.double().cpu().numpy()
    assert np.isclose((y * gd).sum(), (x.double().cpu().numpy() * back.double().cpu().numpy()).sum(),
                      rtol=0, atol=2.0**-20 * np.abs(y * gd).sum())
    d = np.random.default_rng(9).standard_normal(x.shape)
    up, down = (P.rotate(x.cpu().numpy() + e * d, pos, rotary.frequencies, rotary.magnitude, layout)
                for e in (0.5, -0.5))
    assert np.isclose(((up - down) * gd).sum(), (d * back.double().cpu().numpy()).sum(), rtol=0,
                      atol=2.0**-20 * np.abs(d * gd).sum() * 2)


def test_values_that_are_not_finite_stay_in_their_pair():
    rotary = RotaryPositions(128)
    x = _x(8, 3, 2, 128)
    want = rotary.rotate(x, 5)
    x[1, 0, 3], x[2, 1, 70] = float("nan"), float("inf")
    got = rotary.rotate(x, 5)
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[1, 0, 3] = bad[1, 0, 67] = bad[2, 1, 70] = bad[2, 1, 6] = True
    assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], want[~bad])


def test_zero_rows_streams_and_graphs():
    rotary = RotaryPositions(128)
    assert rotary.rotate(torch.empty(0, 4, 128, device="cuda"), 3).shape == (0, 4, 128)
    x, at = _x(9, 64, 16, 128).bfloat16(), torch.arange(64, dtype=torch.int32, device="cuda")
    want = rotary.rotate(x, at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotary.rotate(x, at)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary.rotate(x, at)
    for step in range(3):
        at += 1000 * step
        x.mul_(-1)
        graph.replay()
        got = y.clone()
        assert torch.equal(got, rotary.rotate(x, at))


def test_refusals():
    rotary = RotaryPositions(64)
    x = torch.zeros(4, 2, 128, device="cuda")
    at = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [
        (x[0], 0), (x[..., :32], 0), (x.double(), 0), (x.cpu(), 0), (x, 1.5), (x, True),
        (x, 2**31 - 2), (x, -2**31 - 1), (x, at.long()), (x, at[:3]), (x, at.cpu()),
        (x.transpose(1, 2).contiguous().transpose(1, 2), 0), (x, torch.zeros(8, dtype=torch.int32,
                                                                             device="cuda")[::2]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            rotary.rotate(*call)
    big = torch.zeros(9, 2, 128, device="cuda")
    for out in (x.half(), x[:3], x.cpu(), big[1:5, :1].expand(4, 2, 128)):
        with pytest.raises(ValueError):
            rotary.rotate(x, 0, out=out)
    with pytest.raises(ValueError, match="apart"):  # half of it over x
        rotary.rotate(big[:4], 0, out=big[2:6])

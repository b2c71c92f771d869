"""Rotary positions: :class:`RotaryPositions`, of plain frequencies, linear, ntk and yarn scalings,
or frequencies of the caller's (other forms that configurations name are refused by their name).

:func:`.kernels.rope` takes fp32 rows and tables of the caller's (the reference's seam); here the
frequencies are kept and the angles made where they are used, for any 32-bit position.
"""
from __future__ import annotations

import ctypes as C
import math
import numbers
import operator
from fractions import Fraction

import numpy as np
import torch

from . import _lib
from .kernels import _launch

_I32_MIN, _I32_MAX = -2**31, 2**31 - 1
_TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
_LAYOUTS = ("half", "interleaved")
_SCALING_FIELDS = {
    "linear": {"factor"},
    "ntk": {"factor"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow",
             "attention_factor"},
}


def _number(scaling, key, default=None):
    value = scaling.get(key, default)
    if isinstance(value, bool) or not isinstance(value, numbers.Real) or \
            not math.isfinite(value) or value <= 0:
        raise ValueError(f"rope scaling needs a positive {key}")
    return float(value)


def _whole(value, what):
    try:
        if isinstance(value, (bool, np.bool_)):
            raise TypeError
        return operator.index(value)
    except TypeError:
        raise ValueError(f"{what} must be a whole number")


def rotary_frequencies(dim: int, theta: float = 1e6, scaling=None):
    """``(frequencies, magnitude)``: radians a position of each of ``dim / 2`` pairs, and what
    cosine and sine are multiplied by, as the scalings' papers define them
    (:func:`configured_frequencies` is what a configuration means; yarn differs).

    ``theta ** (-2 i / dim)``, or scaled for positions beyond those a model was trained on
    (``scaling``, a dictionary of ``rope_type`` or ``type``, and ``factor`` s):

    * ``linear``: divided by s;
    * ``ntk``: a base of ``theta * s ** (dim / (dim - 2))``, which leaves the first pair as it is
      and divides the last by s;
    * ``yarn``: pair i makes r = original_max_position_embeddings * f / 2 pi turns over the
      original positions; f stays where r >= beta_fast (32), is divided by s where r <= beta_slow
      (1), and lies between the two in proportion to r (arXiv 2309.00071, 3.2). The magnitude is
      ``attention_factor``, by default 0.1 ln s + 1, or 1 for a factor of no more than 1.
    """
    return _frequencies(dim, theta, scaling, _kept_by_turns)


def configured_frequencies(dim: int, theta: float = 1e6, scaling=None):
    """:func:`rotary_frequencies` of a configuration's ``rope_scaling``, as the models that carry
    one are run: between yarn's two ends the share that stays is linear in the pair's index, not in
    its turns. A pair at d ln(L / 2 pi r) / (2 ln theta) makes r turns over the L original
    positions; f stays up to the pair of beta_fast turns (rounded down) and is divided by s from
    that of beta_slow on (rounded up). For dim 128, theta 10^6, L 32768 and s 4 the two differ in
    16 of 64 frequencies, by up to 42 %."""
    return _frequencies(dim, theta, scaling, _kept_by_index)


def _kept_by_turns(dim, theta, plain, original, fast, slow):
    """The share of each pair's frequency that yarn leaves as it is."""
    turns = [original * f / (2 * math.pi) for f in plain]
    return [min(1.0, max(0.0, (r - slow) / (fast - slow))) for r in turns]


def _kept_by_index(dim, theta, plain, original, fast, slow):
    if theta <= 1:
        raise ValueError("yarn scaling needs a theta above 1")
    low, high = (dim * math.log(original / (2 * math.pi * r)) / (2 * math.log(theta))
                 for r in (fast, slow))
    low, high = max(0, math.floor(low)), min(dim - 1, math.ceil(high))
    if low > high:
        raise ValueError("yarn scaling: all pairs make more than beta_fast turns over the original "
                         "positions, or all fewer than beta_slow")
    return [1.0 - min(1.0, max(0.0, (i - low) / (high - low or 1e-3))) for i in range(dim // 2)]


def _frequencies(dim, theta, scaling, kept):
    try:
        frequencies, magnitude = _scaled(dim, theta, scaling, kept)
    except (OverflowError, ZeroDivisionError):
        frequencies = [math.inf]
    if not all(map(math.isfinite, frequencies)):
        raise ValueError("rotary frequencies of this theta and scaling are beyond a double")
    return frequencies, magnitude


def _scaled(dim, theta, scaling, kept):
    dim = _whole(dim, "rotary dim")
    if dim < 2 or dim % 2:
        raise ValueError("rotary dim must be an even number from 2 on")
    theta = float(theta)
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError("rotary theta must be positive")
    plain = [theta ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling is None:
        return plain, 1.0
    if not isinstance(scaling, dict):
        raise ValueError("rope scaling must be a dictionary")
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in _SCALING_FIELDS:
        raise ValueError(f"rope scaling type must be one of {sorted(_SCALING_FIELDS)}, not {kind!r}")
    if set(scaling) - {"rope_type", "type"} - _SCALING_FIELDS[kind]:
        raise ValueError("rope scaling contains unsupported fields")
    factor = _number(scaling, "factor")
    if kind == "linear":
        return [f / factor for f in plain], 1.0
    if kind == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs two pairs at least")
        base = theta * factor ** (dim / (dim - 2))
        return [base ** (-2.0 * i / dim) for i in range(dim // 2)], 1.0
    original = _number(scaling, "original_max_position_embeddings")
    fast, slow = _number(scaling, "beta_fast", 32.0), _number(scaling, "beta_slow", 1.0)
    if fast <= slow:
        raise ValueError("yarn scaling needs beta_fast > beta_slow")
    out = [f * (keep + (1.0 - keep) / factor)
           for f, keep in zip(plain, kept(dim, theta, plain, original, fast, slow))]
    return out, _number(scaling, "attention_factor", 0.1 * math.log(max(factor, 1.0)) + 1.0)


def _turns(f: float) -> int:
    """2^64 of a turn a position, whole turns taken off, as a signed 64-bit number."""
    u = round(Fraction(f) * 2**64 / _TWO_PI) % 2**64
    return u - 2**64 if u >= 2**63 else u


def _apart(t) -> bool:
    """Whether no two elements of a tensor share a place."""
    reach = 0
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (size - 1)
    return True


def _span(t):
    """The bytes [first, last) that a tensor lies in."""
    n = 1 + sum(s * (k - 1) for s, k in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _same_places(a, b) -> bool:
    return a.data_ptr() == b.data_ptr() and all(
        x == y or n == 1 for x, y, n in zip(a.stride(), b.stride(), a.shape))


_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _capturing(index):
    """Whether the current stream of device ``index`` is being captured."""
    if torch._C._cuda_getDevice() == index:
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _before_captures(device, what):
    """The device that ``what`` is made on, where no graph is being captured: what fills it would be
    the graph's."""
    device = torch.device(device or "cuda")
    if device.type == "cuda":
        with torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                raise ValueError(f"{what} is made before a graph is captured, not in it")
    return device


def _lend(tensor, index, streams):
    """The current stream, none of the tensor's ``streams`` yet, reads it: the allocator is told, so
    that dropping the tensor does not give its memory away under a launch. (In a capture there is
    nothing to tell: what a graph reads is the caller's to keep.)"""
    if not _capturing(index):
        tensor.record_stream(torch.cuda.current_stream(index))
        streams.add(torch._C._cuda_getCurrentRawStream(index))


class RotaryPositions:
    """The rotation of the first ``dim`` elements of heads by their rows' positions.

    ``layout``: ``"half"`` pairs elements ``(i, i + dim / 2)``, ``"interleaved"``
    ``(2 i, 2 i + 1)``. ``theta`` and ``scaling`` (a configuration's ``rope_scaling``) as in
    :func:`configured_frequencies`; or ``frequencies``, ``dim / 2`` radians a position of any other
    form, and ``magnitude`` (so :func:`rotary_frequencies` gives the paper's yarn). The frequencies
    are kept as 64-bit fractions of a turn on ``device`` (the current GPU): an angle is right to
    2^-31 of a turn at any position of 32 bits, cosine and sine to 2^-22. Any stream may use them;
    keep the object as long as a captured graph that used it is replayed."""

    def __init__(self, dim: int = 128, *, theta: float = 1e6, layout: str = "half", scaling=None,
                 frequencies=None, magnitude=None, device=None):
        if layout not in _LAYOUTS:
            raise ValueError(f"rotary layout is 'half' or 'interleaved', not {layout!r}")
        dim = _whole(dim, "rotary dim")
        if frequencies is None:
            if magnitude is not None:
                raise ValueError("magnitude comes with frequencies of the caller's own")
            self.frequencies, self.magnitude = configured_frequencies(dim, theta, scaling)
        else:
            if scaling is not None:
                raise ValueError("rotary takes either scaling or frequencies")
            self.frequencies = [float(f) for f in frequencies]
            if dim < 2 or 2 * len(self.frequencies) != dim or not all(
                    map(math.isfinite, self.frequencies)):
                raise ValueError("rotary frequencies must be dim / 2 finite numbers")
            self.magnitude = 1.0 if magnitude is None else float(magnitude)
        if not abs(self.magnitude) <= torch.finfo(torch.float32).max:
            raise ValueError("rotary magnitude must be a finite number of fp32")
        self.dim, self.layout = dim, layout
        self.turns = torch.tensor([_turns(f) for f in self.frequencies], dtype=torch.int64,
                                  device=_before_captures(device, "a rotation"))
        self._index = self.turns.get_device()
        # (they are on the device: the copy of pageable memory waits for itself)
        self._streams = {torch._C._cuda_getCurrentRawStream(self._index)} if self._index >= 0 else ()
        self._args = _lib.Rotary(self.turns.data_ptr(), dim, int(layout == "interleaved"),
                                 self.magnitude)
        self._address = C.addressof(self._args)
        self._rotate = None

    def __deepcopy__(self, memo):
        return self  # (frequencies do not change)

    def rotate(self, x, positions, *, inverse: bool = False, out=None):
        """``x [rows, heads, head_dim]`` (fp32, fp16 or bf16; any strides between rows and heads)
        with row r turned by ``positions[r]`` (int32 on the device, or a number: the first row's,
        the others one further each); elements from ``dim`` on as they are. ``inverse`` turns the
        other way, by the same magnitude, which is the rotation's gradient: that of ``x`` from that
        of the result (and takes a rotation of magnitude 1 back).

        ``out``: a tensor of x's shape and type, ``x`` itself or memory apart from it. Computed in
        fp32, rounded once."""
        # (a short call is mostly host time: each check once, in the order of what fails least)
        shape, index = x.shape, self._index
        if len(shape) != 3 or shape[2] < self.dim:
            raise ValueError(f"rotate takes x [rows, heads, head_dim >= {self.dim}]")
        rows, heads, hd = shape
        if rows > _I32_MAX or heads > _I32_MAX or hd > _I32_MAX:
            raise ValueError("rotate takes fewer than 2^31 rows, heads and elements of a head")
        code = _TYPES.get(x.dtype)
        if code is None:
            raise ValueError("rotate takes float32, float16 or bfloat16")
        if index < 0:
            raise ValueError("the rotary's frequencies must be on a GPU")
        if x.get_device() != index:
            raise ValueError("x must be on the frequencies' device")
        x0, x1, x2 = x.stride()
        if x2 != 1:
            raise ValueError("a head's elements must be side by side")
        if isinstance(positions, torch.Tensor):
            if positions.dtype is not torch.int32 or positions.shape != (rows,) or \
                    positions.get_device() != index or not positions.is_contiguous():
                raise ValueError("positions must be int32 [rows] on x's device, or a number")
            at, pos0 = positions.data_ptr(), 0
        else:
            at, pos0 = None, positions
            if type(positions) is not int:
                pos0 = _whole(positions, "positions, where no int32 tensor on x's device,")
            if not (_I32_MIN <= pos0 and pos0 + rows - 1 <= _I32_MAX):
                raise ValueError("positions must be of 32 bits")
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
            y0, y1 = heads * hd, hd
        else:
            if out.shape != shape or out.dtype != x.dtype or out.get_device() != index or \
                    out.stride(2) != 1 or not _apart(out):
                raise ValueError("out must be a tensor of x's shape, type and device, its elements "
                                 "apart and a head's side by side")
            y0, y1, _ = out.stride()
            if x.numel() and not _same_places(x, out):
                (a, b), (c, d) = _span(x), _span(out)
                if a < d and c < b:
                    raise ValueError("out must be x itself or memory apart from it")
        if rows and heads:
            if torch._C._cuda_getCurrentRawStream(index) not in self._streams:
                _lend(self.turns, index, self._streams)
            _launch(torch, self._rotate or self._bind(), index, x.data_ptr(), x0, x1, code, rows,
                    heads, hd, self._address, at, pos0, 1 if inverse else 0, out.data_ptr(), y0, y1)
        return out

    def _bind(self):
        self._rotate = _lib.load().drt_op_rotate
        return self._rotate

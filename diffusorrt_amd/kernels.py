"""Per-op kernel table on device tensors (the reference's ``KernelTable`` seam).

Signatures follow ``backends/kernel_table.py:118-126`` / ``backends/mlx_ops.py``
of the reference's ``python/src/edllm/``:

    rms_norm(x, weight, eps)
    linear(x, weight, bias=None)          # weight: DeviceQ4Weight | DeviceBF16Weight
    rope(x[rows, H, hd], cos[rows, 1, hd], sin[rows, 1, hd])
    swiglu(gate, up)
    attention(q[rq, Hq, hd], k[rk, Hkv, hd], v, *, head_dim, kind,
              mask_geometry=None, q_positions=None) -> [rq, Hq*hd]

Every op runs a HIP kernel of ``libdrt_rocm.so`` on the tensors' device and
current torch stream. Validation raises ``ValueError`` before any launch, like
the reference's fail-closed checks.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

from . import _lib

_I32_MAX = 2**31 - 1
KV_TILE_ELEMS = 8192  # one 32-key tile: K block + V block, 2-byte elements


def _torch():
    import torch

    return torch


def _stream(t):
    torch = _torch()
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _ptr(t) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise ValueError("kernel table ops take contiguous device tensors")


class DeviceQ4Weight:
    """A q4 g64 affine linear weight repacked into the device tile layout.

    Built once from an MLX-packed ``QuantizedWeight`` (``w_q`` uint32 ``[N, K/8]``
    as int32, ``scales``/``biases`` bf16 ``[N, K/64]``; ``mlx_ops.py:43-60``)."""

    def __init__(self, w_q, scales, biases):
        torch = _torch()
        _require_cuda(w_q, scales, biases)
        n, kw = w_q.shape
        k = kw * 8
        if scales.shape != (n, k // 64) or biases.shape != (n, k // 64):
            raise ValueError("scales/biases must be [N, K/64]")
        if w_q.dtype != torch.int32 or scales.dtype != torch.bfloat16 or biases.dtype != torch.bfloat16:
            raise ValueError("q4 weight needs int32 words and bf16 scales/biases")
        self.shape = (int(n), int(k))
        self.qw = torch.empty(n * k // 8, dtype=torch.int32, device=w_q.device)
        self.sb = torch.empty(n * (k // 64), dtype=torch.int32, device=w_q.device)
        _lib.check(_lib.load().drt_op_q4_repack(_ptr(w_q), _ptr(scales), _ptr(biases), n, k,
                                                _ptr(self.qw), _ptr(self.sb), _stream(w_q)))


class DeviceBF16Weight:
    """A bf16 ``[N, K]`` linear weight repacked into the device tile layout."""

    def __init__(self, w):
        torch = _torch()
        _require_cuda(w)
        if w.dtype != torch.bfloat16 or w.dim() != 2:
            raise ValueError("bf16 weight must be a 2-D bfloat16 tensor")
        n, k = w.shape
        self.shape = (int(n), int(k))
        self.wb = torch.empty_like(w)
        _lib.check(_lib.load().drt_op_bf16_repack(_ptr(w), n, k, _ptr(self.wb), _stream(w)))


def linear(x, weight, bias=None):
    """``x @ W.T (+ bias)`` with the reference's dtype rules (``mlx_ops.py:97-130``).

    q4: fp32 (or bf16) x -> fp32 y. bf16 weight: ``bf16(bf16(x) @ W.T)`` as fp32."""
    torch = _torch()
    _require_cuda(x, bias)
    lib = _lib.load()
    n, k = weight.shape
    if x.dim() != 2 or x.shape[1] != k:
        raise ValueError(f"linear x must be [M, {k}]")
    m = x.shape[0]
    y = torch.empty((m, n), dtype=torch.float32, device=x.device)
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (n,)):
        raise ValueError("linear bias must be bf16 [N]")
    bptr = _ptr(bias) if bias is not None else None
    if isinstance(weight, DeviceQ4Weight):
        if x.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("q4 linear x must be fp32 or bf16")
        ws_bytes = lib.drt_op_q4_linear_workspace_bytes(m, n, k)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
        _lib.check(lib.drt_op_q4_linear(_ptr(weight.qw), _ptr(weight.sb), _ptr(x),
                                        _lib.BF16 if x.dtype == torch.bfloat16 else _lib.F32,
                                        m, n, k, bptr, _ptr(y), _ptr(ws), ws_bytes, _stream(x)))
    elif isinstance(weight, DeviceBF16Weight):
        if x.dtype == torch.float32:  # rounded to bf16 on the way
            ws_bytes = lib.drt_op_bf16_linear_x_workspace_bytes(m, n, k)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
            _lib.check(lib.drt_op_bf16_linear_x(_ptr(weight.wb), _ptr(x), _lib.F32, m, n, k, bptr,
                                                _ptr(y), _ptr(ws), ws_bytes, _stream(x)))
        else:
            xb = x.to(torch.bfloat16).contiguous()
            ws_bytes = lib.drt_op_bf16_linear_workspace_bytes(m, n, k)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
            _lib.check(lib.drt_op_bf16_linear(_ptr(weight.wb), _ptr(xb), m, n, k, bptr, _ptr(y),
                                              _ptr(ws), ws_bytes, _stream(x)))
    else:
        raise ValueError("linear weight must be a DeviceQ4Weight or DeviceBF16Weight")
    return y


def rms_norm(x, weight, eps: float):
    """fp32 RMSNorm over the last axis with a bf16 weight (``mlx_ops.py:21-35``)."""
    torch = _torch()
    _require_cuda(x, weight)
    if x.dtype != torch.float32 or weight.dtype != torch.bfloat16:
        raise ValueError("rms_norm takes fp32 x and a bf16 weight")
    d = x.shape[-1]
    if weight.shape != (d,):
        raise ValueError("rms_norm weight must match the last axis")
    y = torch.empty_like(x)
    rows = x.numel() // d
    _lib.check(_lib.load().drt_op_rms_norm(_ptr(x), _ptr(weight), float(eps), _ptr(y), rows, d,
                                           _stream(x)))
    return y


def rope(x, cos, sin):
    """Split-half RoPE on fp32 ``x [rows, H, hd]`` with ``cos/sin [rows, 1, hd]``."""
    torch = _torch()
    _require_cuda(x)
    rows, h, hd = x.shape
    c = cos.reshape(rows, hd).to(device=x.device, dtype=torch.float32).contiguous()
    s = sin.reshape(rows, hd).to(device=x.device, dtype=torch.float32).contiguous()
    y = torch.empty_like(x)
    _lib.check(_lib.load().drt_op_rope(_ptr(x), _ptr(c), _ptr(s), _ptr(y), rows, h, hd,
                                       _stream(x)))
    return y


def swiglu(gate, up):
    """``silu(gate) * up`` in fp32 (``mlx_ops.py:147-154``)."""
    torch = _torch()
    _require_cuda(gate, up)
    if gate.shape != up.shape or gate.dtype != torch.float32 or up.dtype != torch.float32:
        raise ValueError("swiglu takes two fp32 tensors of one shape")
    y = torch.empty_like(gate)
    _lib.check(_lib.load().drt_op_swiglu(_ptr(gate), _ptr(up), _ptr(y), gate.numel(), _stream(gate)))
    return y


_Q_CODES = {}  # torch dtype -> code of what a query may be (filled on first use)


def _q_codes():
    if not _Q_CODES:
        torch = _torch()
        _Q_CODES.update({torch.float16: _lib.F16, torch.bfloat16: _lib.BF16})
    return _Q_CODES


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name, *shape) -> int:
    return getattr(_lib.load(), name)(*shape)


def _launch(torch, fn, index, *args):
    """``fn(*args, stream)`` on device ``index`` and its current stream. (A short call is mostly
    host time: addresses go as plain integers, and the device is only set where it differs.)"""
    back = torch._C._cuda_getDevice()
    if back == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        torch.cuda.set_device(index)
        try:
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        finally:
            torch.cuda.set_device(back)
    if status:
        _lib.check(status)


def _cache_dtype(dtype) -> int:
    """The code of a cache's type; what is no name of one is refused, never another type's cache."""
    code = {"f16": _lib.F16, "bf16": _lib.BF16, "i8": _lib.I8,
            # (other names that fp16 has always gone by here)
            None: _lib.F16, "fp16": _lib.F16, "float16": _lib.F16,
            _torch().float16: _lib.F16}.get(dtype)
    if code is None:
        raise ValueError(f"a cache's dtype is 'f16', 'bf16' or 'i8', not {dtype!r}")
    return code


class PrefixKVCache:
    """Tiled K/V cache for ``layers`` layers on one device.

    The build's prefix-cache object: rows are written once (``store``) at
    absolute positions and read by :meth:`attention`. Layout per (layer, kv
    head): 32-key tiles of 8192 elements (K block then V block) in the MFMA
    operand order of the attention kernel. Unwritten slots stay zero.

    ``dtype`` is ``"f16"``, ``"bf16"`` or ``"i8"``; another is a ValueError. ``"i8"``: whole numbers
    of [-127, 127] times one power of two for each tile's K and V (``scales [layers, kv_heads,
    tiles, 2]``), half the bytes of a 16-bit cache. A store into an ``"i8"`` cache quantizes each
    tile it touches as a whole, from the rows it keeps (as they read) and the new ones, to the least
    power of two >= 2^-40 that holds them: a value is off by at most half of it (max / 127 to
    2 max / 127), a row that later stores of its tile went past by less than one of the last scale.
    A tile with a value that is not finite, or beyond 127 * 2^40, reads as NaN until one store
    writes all 32 rows of it, or :meth:`clear`; so does a tile that keeps rows of an earlier
    sequence take their size into its scale. Clear an ``"i8"`` cache, or one with ``block_sums``,
    before another sequence. Stores into such a cache read and write whole tiles: two that touch
    one tile, be it other rows of it, must not overlap in time (order them by an event where they
    are on two streams); stores into a plain 16-bit cache may.

    ``block_sums=True`` keeps the sum of each tile's keys (``sums [layers, kv_heads, tiles,
    128]``) up to date, which :meth:`select_blocks` scores blocks by."""

    def __init__(self, layers: int, kv_heads: int, capacity: int, *, dtype="f16", device=None,
                 block_sums: bool = False):
        torch = _torch()
        self.layers, self.kv_heads = int(layers), int(kv_heads)
        self.tiles = (int(capacity) + 31) // 32
        self.capacity = self.tiles * 32
        self.head_stride = self.tiles * KV_TILE_ELEMS
        self.kv_dtype = _cache_dtype(dtype)
        shape = (self.layers, self.kv_heads, self.head_stride)
        device = device or "cuda"
        self.scales = self.sums = None
        if self.kv_dtype == _lib.I8:  # a byte is a code + 128
            self.data = torch.full(shape, 128, dtype=torch.uint8, device=device)
            self.scales = torch.ones((*shape[:2], self.tiles, 2), dtype=torch.float32,
                                     device=device)
        else:
            self.data = torch.zeros(shape, dtype=torch.bfloat16 if self.kv_dtype == _lib.BF16
                                    else torch.float16, device=device)
        if block_sums:
            self.sums = torch.zeros((*shape[:2], self.tiles, 128), dtype=torch.float32,
                                    device=device)
        self.length = 0
        self._index = self.data.get_device()  # (-1: on the host, where nothing runs)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.data, self.scales, self.sums)
                   if t is not None)

    def clear(self) -> None:
        """Forget every row: the cache as it was made."""
        self.data.fill_(128 if self.scales is not None else 0)
        if self.scales is not None:
            self.scales.fill_(1.0)
        if self.sums is not None:
            self.sums.fill_(0.0)
        self.length = 0

    def _check(self, layer, *tensors):
        """The layer, and where the tensors of a call are."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer must be in [0, {self.layers})")
        if self._index < 0:
            raise ValueError("the cache must be on a GPU")
        for t in tensors:
            if t.get_device() != self._index:
                raise ValueError("tensors must be on the cache's device")
            if not t.is_contiguous():
                raise ValueError("the cache's calls take contiguous tensors")

    def _data(self, layer):
        return self.data.data_ptr() + layer * self.kv_heads * self.head_stride * \
            (1 if self.scales is not None else 2)

    def _scales(self, layer):
        return None if self.scales is None else \
            self.scales.data_ptr() + layer * self.kv_heads * self.tiles * 8

    def _sums(self, layer):
        return None if self.sums is None else \
            self.sums.data_ptr() + layer * self.kv_heads * self.tiles * 512

    def _queries(self, q, n_keys, row_pos0):
        """(rows, query heads, dtype code) of a call's queries, checked against the cache."""
        if q.dim() != 3:
            raise ValueError("attention needs q [rows, Hq, 128]")
        rows, hq, hd = q.shape
        if hd != 128 or hq < 1 or hq % self.kv_heads:
            raise ValueError("attention needs q [rows, Hq, 128] and Hq % Hkv == 0")
        code = _q_codes().get(q.dtype)
        if code is None or (self.scales is None and code != self.kv_dtype):
            raise ValueError("q must be float16 or bfloat16 over an 8-bit cache, and of the "
                             "cache's own type over a 16-bit one")
        if n_keys < 1 or n_keys > self.capacity:
            raise ValueError("n_keys outside the cache")
        if rows < 1 or row_pos0 < 0 or row_pos0 + rows > _I32_MAX:
            raise ValueError("attention needs a query row, and row positions of 32 bits")
        return rows, hq, code

    def store(self, layer: int, k, v, pos0: int) -> None:
        """Write ``k/v [n, Hkv, 128]`` (fp32 or bf16) at positions ``pos0..pos0+n-1``."""
        torch = _torch()
        tiled = self.scales is not None or self.sums is not None
        if tiled:
            self._check(layer, k, v)
        else:
            _require_cuda(k, v)
        shape = k.shape
        n = shape[0]
        if shape != v.shape or shape[1:] != (self.kv_heads, 128):
            raise ValueError("store takes k, v of shape [n, kv_heads, 128]")
        if pos0 < 0 or pos0 + n > self.capacity:
            raise ValueError("store positions exceed the cache capacity")
        dtype = k.dtype
        if dtype not in (torch.float32, torch.bfloat16) or v.dtype != dtype:
            raise ValueError("store takes fp32 or bf16 k/v")
        src = _lib.BF16 if dtype is torch.bfloat16 else _lib.F32
        if tiled:
            lib, data, sums = _lib.load(), self._data(layer), self._sums(layer)
            if self.scales is not None:
                _launch(torch, lib.drt_op_kv8_store, self._index, k.data_ptr(), v.data_ptr(), src,
                        n, self.kv_heads, pos0, data, self.head_stride, self._scales(layer), sums)
            else:
                _launch(torch, lib.drt_op_kv16_store, self._index, k.data_ptr(), v.data_ptr(), src,
                        n, self.kv_heads, pos0, data, self.head_stride, self.kv_dtype, sums)
            self.length = max(self.length, pos0 + n)
            return
        layer_view = self.data[layer]
        _lib.check(_lib.load().drt_op_kv_pack(_ptr(k), _ptr(v), src, n, self.kv_heads, pos0,
                                              _ptr(layer_view), self.head_stride, self.kv_dtype,
                                              _stream(k)))
        self.length = max(self.length, pos0 + n)

    def load(self, layer: int, pos0: int, n: int, out_dtype=None):
        """``(k, v) [n, Hkv, 128]`` of positions ``pos0..pos0+n-1`` as the cache holds them, in
        fp32 (or bf16): what attention reads."""
        torch = _torch()
        out_dtype = out_dtype or torch.float32
        if out_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("load gives float32 or bfloat16")
        if n < 1 or pos0 < 0 or pos0 + n > self.capacity:
            raise ValueError("load positions outside the cache")
        self._check(layer)
        k = torch.empty((n, self.kv_heads, 128), dtype=out_dtype, device=self.data.device)
        v = torch.empty_like(k)
        _launch(torch, _lib.load().drt_op_kv_load, self._index, self._data(layer),
                self.head_stride, self.kv_dtype, self._scales(layer), n, self.kv_heads, pos0,
                k.data_ptr(), v.data_ptr(),
                _lib.F32 if out_dtype is torch.float32 else _lib.BF16)
        return k, v

    def attention(self, layer: int, q, *, n_keys: int, row_pos0: int, kind: str,
                  mask_geometry=None, out_dtype=None):
        """Attention of ``q [rows, Hq, 128]`` (cache dtype; fp16 or bf16 over an ``"i8"`` cache)
        over keys ``[0, n_keys)``."""
        torch = _torch()
        if self.kv_dtype == _lib.I8:
            return self._attention8(layer, q, n_keys, row_pos0, kind, mask_geometry, out_dtype)
        _require_cuda(q)
        rows, hq, hd = q.shape
        if hd != 128 or hq % self.kv_heads:
            raise ValueError("attention needs head_dim 128 and Hq % Hkv == 0")
        if n_keys < 1 or n_keys > self.capacity:
            raise ValueError("n_keys outside the cache")
        want = torch.bfloat16 if self.kv_dtype == _lib.BF16 else torch.float16
        if q.dtype != want:
            raise ValueError(f"q must be {want} to match the cache")
        mk, p, b = _mask_args(kind, mask_geometry)
        out_dtype = out_dtype or torch.float32
        odt = _lib.F32 if out_dtype == torch.float32 else _lib.BF16
        out = torch.empty((rows, hq * 128), dtype=out_dtype, device=q.device)
        lib = _lib.load()
        ws_bytes = lib.drt_op_attention_workspace_bytes(rows, hq, self.kv_heads, n_keys)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        _lib.check(lib.drt_op_attention(_ptr(q), _ptr(self.data[layer]), self.head_stride,
                                        self.kv_dtype, rows, hq, self.kv_heads, n_keys, row_pos0,
                                        mk, p, b, _ptr(out), odt, _ptr(ws), ws_bytes, _stream(q)))
        return out

    def _attention8(self, layer, q, n_keys, row_pos0, kind, mask_geometry, out_dtype):
        torch = _torch()
        self._check(layer, q)
        rows, hq, qdt = self._queries(q, n_keys, row_pos0)
        mk, p, b = _mask_args(kind, mask_geometry)
        out, odt = _attention_out(torch, q, rows, hq, out_dtype)
        need = _workspace_bytes("drt_op_attention_kv8_workspace_bytes", rows, hq, self.kv_heads,
                                n_keys)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _launch(torch, _lib.load().drt_op_attention_kv8, self._index, q.data_ptr(), qdt,
                self._data(layer), self.head_stride, self._scales(layer), rows, hq, self.kv_heads,
                n_keys, row_pos0, mk, p, b, out.data_ptr(), odt,
                None if ws is None else ws.data_ptr(), need)
        return out

    def select_blocks(self, layer: int, q, *, block_size: int, count: int, n_keys: int,
                      row_pos0: int, kind: str, mask_geometry=None, sinks: int = 0,
                      local: int = 1):
        """The blocks of ``block_size`` keys (a multiple of 32) that each row of ``q`` reads of
        keys ``[0, n_keys)``: int32 ``[rows, kv_heads, count]``, ascending.

        They are the first ``sinks`` and the last ``local`` blocks that the row sees and, of
        those between, the ones whose keys' sum has the largest product with the sum of the
        row's queries of the head's group (compared in 64 bits; equal ones: the lower block). A
        row that sees no more than ``count`` blocks lists them all, then ``-1``. Needs
        ``block_sums=True``."""
        torch = _torch()
        if self.sums is None:
            raise ValueError("select_blocks needs a cache with block_sums=True")
        self._check(layer, q)
        rows, hq, qdt = self._queries(q, n_keys, row_pos0)
        _sparse_args(block_size, count)
        if sinks < 0 or local < 1 or sinks + local > count:
            raise ValueError("select_blocks needs sinks >= 0, local >= 1, sinks + local <= count")
        mk, p, b = _mask_args(kind, mask_geometry)
        blocks = torch.empty((rows, self.kv_heads, count), dtype=torch.int32, device=q.device)
        need = _workspace_bytes("drt_op_select_blocks_workspace_bytes", rows, self.kv_heads,
                                n_keys, block_size)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _launch(torch, _lib.load().drt_op_select_blocks, self._index, q.data_ptr(), qdt,
                self._sums(layer), self.tiles, rows, hq, self.kv_heads, n_keys, row_pos0, mk, p, b,
                block_size, count, sinks, local, blocks.data_ptr(),
                None if ws is None else ws.data_ptr(), need)
        return blocks

    def sparse_attention(self, layer: int, q, blocks, *, block_size: int, n_keys: int,
                         row_pos0: int, kind: str, mask_geometry=None, out_dtype=None):
        """:meth:`attention` over the keys of ``blocks`` (int32 ``[rows, kv_heads, count]``, as
        :meth:`select_blocks` gives them or a caller's own) that the row sees.

        A list is a set: its order and repetitions do not matter, entries beyond the row's keys
        and negative ones are none; a row without any block gives zeros."""
        torch = _torch()
        self._check(layer, q, blocks)
        rows, hq, qdt = self._queries(q, n_keys, row_pos0)
        if blocks.dtype is not torch.int32 or blocks.dim() != 3:
            raise ValueError("blocks must be int32 [rows, kv_heads, count]")
        br, bh, count = blocks.shape
        if br != rows or bh != self.kv_heads:
            raise ValueError("blocks must be int32 [rows, kv_heads, count]")
        _sparse_args(block_size, count)
        mk, p, b = _mask_args(kind, mask_geometry)
        out, odt = _attention_out(torch, q, rows, hq, out_dtype)
        need = _workspace_bytes("drt_op_sparse_attention_workspace_bytes", rows, hq, self.kv_heads,
                                block_size, count)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _launch(torch, _lib.load().drt_op_sparse_attention, self._index, q.data_ptr(), qdt,
                self._data(layer), self.head_stride, self.kv_dtype, self._scales(layer), rows, hq,
                self.kv_heads, n_keys, row_pos0, mk, p, b, blocks.data_ptr(), block_size, count,
                out.data_ptr(), odt, None if ws is None else ws.data_ptr(), need)
        return out


def _attention_out(torch, q, rows, hq, out_dtype):
    out_dtype = out_dtype or torch.float32
    if out_dtype is not torch.float32 and out_dtype is not torch.bfloat16:
        raise ValueError("attention out must be float32 or bfloat16")
    out = torch.empty((rows, hq * 128), dtype=out_dtype, device=q.device)
    return out, _lib.F32 if out_dtype is torch.float32 else _lib.BF16


def _sparse_args(block_size, count):
    if block_size < 32 or block_size % 32 or block_size > _I32_MAX:
        raise ValueError("block_size must be a multiple of 32")
    if not 1 <= count <= 1024:
        raise ValueError("a row lists 1 to 1024 blocks")


def _mask_args(kind, mask_geometry):
    if kind in ("full", "bidirectional"):
        if mask_geometry is not None:
            raise ValueError("mask geometry is only consumed by the d2f_hybrid kind")
        return _lib.MASK_BIDIRECTIONAL, 0, 1
    if kind == "d2f_hybrid":
        if mask_geometry is None:
            raise ValueError("d2f_hybrid requires mask geometry")
        if isinstance(mask_geometry, dict):
            p, b = int(mask_geometry["prompt_len"]), int(mask_geometry["block_size"])
        else:
            p, b = (int(v) for v in mask_geometry)
        if not (0 <= p <= _I32_MAX and 1 <= b <= _I32_MAX):
            raise ValueError("bad d2f_hybrid mask geometry")
        return _lib.MASK_D2F_HYBRID, p, b
    raise ValueError(f"unsupported attention mask kind: {kind}")


def attention(q, k, v, *, head_dim: int, kind: str, mask_geometry=None, q_positions=None,
              kv_dtype: str = "bf16"):
    """Reference-signature attention (``mlx_ops.py:347-443``) via a temporary cache.

    ``q_positions`` (absolute positions of the q rows) must be contiguous; by
    default q rows are the last ``rq`` positions of the ``rk`` keys. The output
    dtype follows ``q`` like the reference's ``.astype(out_dtype)``.

    ``kv_dtype`` is the cache's: ``"bf16"``, ``"f16"`` or ``"i8"``. Queries are rounded to a
    16-bit cache's own type; over ``"i8"`` bf16 and fp16 ones stay as they are and others are
    rounded to fp16. Beyond 65504 a query in fp16 is an infinity and its row NaN: larger ones are
    for bf16."""
    torch = _torch()
    if head_dim != 128:
        raise ValueError("attention head_dim must be 128")
    rq, hq, _ = q.shape
    rk, hkv, _ = k.shape
    if k.shape != v.shape:
        raise ValueError(f"attention K/V shapes disagree: {tuple(k.shape)} != {tuple(v.shape)}")
    if hq % hkv:
        raise ValueError("attention query heads must be divisible by compact K/V heads")
    if q_positions is None:
        pos0 = rk - rq
        if pos0 < 0:
            raise ValueError("more query rows than keys needs explicit q_positions")
    else:
        qp = [int(p) for p in q_positions]
        if len(qp) != rq or any(b - a != 1 for a, b in zip(qp, qp[1:])):
            raise ValueError("q_positions must be one contiguous run per query row")
        pos0 = qp[0]
        if pos0 < 0 or qp[-1] >= rk:
            raise ValueError("q_positions outside the kv range")
    cache = PrefixKVCache(1, hkv, rk, dtype=kv_dtype, device=q.device)
    kd = k if k.dtype in (torch.float32, torch.bfloat16) else k.float()
    vd = v if v.dtype == kd.dtype else v.to(kd.dtype)
    cache.store(0, kd.contiguous(), vd.contiguous(), 0)
    if kv_dtype == "i8":  # queries keep a 16-bit type of their own
        qc = (q if q.dtype in (torch.float16, torch.bfloat16) else q.half()).contiguous()
    else:
        qc = q.to(torch.bfloat16 if kv_dtype == "bf16" else torch.float16).contiguous()
    out = cache.attention(0, qc, n_keys=rk, row_pos0=pos0, kind=kind, mask_geometry=mask_geometry,
                          out_dtype=torch.float32)
    return out.to(q.dtype)


KERNEL_OP_NAMES = ("rms_norm", "linear", "rope", "swiglu", "attention")


class KernelTable:
    """The op table a forward dispatches through (``kernel_table.py:118-126``)."""

    backend = "rocm"
    rms_norm = staticmethod(rms_norm)
    linear = staticmethod(linear)
    rope = staticmethod(rope)
    swiglu = staticmethod(swiglu)
    attention = staticmethod(attention)

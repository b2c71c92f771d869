"""A K/V cache in pages that many sequences share: :class:`PagedKVCache`.

:class:`.kernels.PrefixKVCache` holds one sequence, its keys one after the other; here a pool of
pages holds any number, each a list of pages that the caller keeps. Two sequences may list the
same page (a prefix in common).
"""
from __future__ import annotations

import copy
import ctypes as C
import operator

import numpy as np
import torch

from . import _lib
from .kernels import KV_TILE_ELEMS, _cache_dtype, _launch, _mask_args
from .rotary import _TYPES, _before_captures, _capturing, _lend, _whole

_I32_MAX = 2**31 - 1


def _whole_numbers(values, what):
    """int32 numpy of a list, an array or a host tensor of whole numbers."""
    if isinstance(values, torch.Tensor):
        if values.is_cuda:
            raise ValueError(f"{what} must be on the host")
        if values.is_floating_point() or values.is_complex() or values.dtype is torch.bool:
            raise ValueError(f"{what} must be whole numbers")
        values = values.numpy()
    a = np.asarray(values)
    if a.size == 0:
        a = a.astype(np.int32)
    if a.dtype.kind not in "iu":
        raise ValueError(f"{what} must be whole numbers")
    if a.size and (a.min() < -1 or a.max() > _I32_MAX):
        raise ValueError(f"{what} must be whole numbers of 32 bits")
    return np.asarray(a, dtype=np.int32, order="C")


def _table(pages):
    """int32 [seqs, width], -1 behind a list's end."""
    if isinstance(pages, (list, tuple)):
        lists = [_whole_numbers(p, "pages") for p in pages]
        if any(p.ndim != 1 for p in lists):
            raise ValueError("pages must be a list of page numbers for each sequence")
        out = np.full((len(lists), max([1] + [p.size for p in lists])), -1, dtype=np.int32)
        for row, p in zip(out, lists):
            row[:p.size] = p
        return out
    out = _whole_numbers(pages, "pages")
    if out.ndim != 2:
        raise ValueError("pages must be [sequences, width]")
    return out


class PagedBatch:
    """New rows of several sequences, as :meth:`PagedKVCache.batch` plans them: made once a step,
    it serves ``append``, ``attention`` and ``load`` of every layer, on any stream. Its lengths and
    pages are fixed, and none is planned inside a capture: a graph that used it is of its step
    alone. Keep it as long as that graph is replayed. How an attention is cut among the work-groups
    follows from all of the batch's lengths: a row's result is the same from call to call, and may
    differ in its last bits beside other sequences."""

    def __init__(self, cache, table, keys, rows, heads, positions, kind, mask_geometry):
        if cache._index >= 0 and _capturing(cache._index):
            raise ValueError("a batch is planned before a graph is captured, not in it")
        table = _table(table)
        heads = _whole(heads, "heads")
        if abs(heads) > _I32_MAX:
            raise ValueError("heads must be a whole number")
        keys, rows = _whole_numbers(keys, "keys"), _whole_numbers(rows, "rows")
        seqs = table.shape[0]
        if keys.shape != (seqs,) or rows.shape != (seqs,):
            raise ValueError("a batch takes pages, keys and rows of each sequence")
        pos0 = keys - rows if positions is None else _whole_numbers(positions, "positions")
        if pos0.shape != (seqs,):
            raise ValueError("positions are the first row's of each sequence")
        prompt = None
        if kind == "causal":
            if mask_geometry is not None:
                raise ValueError("mask geometry is only consumed by the d2f_hybrid kind")
            mask, block = _lib.MASK_D2F_HYBRID, 1
        else:
            if kind == "d2f_hybrid" and mask_geometry is not None and \
                    not isinstance(mask_geometry, dict):
                try:
                    first, block = mask_geometry
                except (TypeError, ValueError):
                    raise ValueError("d2f_hybrid mask geometry is (prompt length, block size)")
                try:
                    mask_geometry = (operator.index(first), block)
                except TypeError:  # a prompt's length for each sequence
                    prompt = _whole_numbers(first, "prompt lengths")
                    if prompt.shape != (seqs,):
                        raise ValueError("prompt lengths are one for each sequence")
                    mask_geometry = (0, block)
            mask, length, block = _mask_args(kind, mask_geometry)
            if prompt is None and length:
                prompt = np.full(seqs, length, dtype=np.int32)
        self.kind = kind
        self.info = _lib.PagedBatch()
        self._geometry = cache._geometry
        self._index = cache._index
        lib = _lib.load()

        def plan(out):
            _lib.check(lib.drt_paged_plan(
                table.ctypes.data, table.shape[1], seqs, rows.ctypes.data, keys.ctypes.data,
                pos0.ctypes.data, None if prompt is None else prompt.ctypes.data, cache.page_size,
                cache.pages, heads, cache.kv_heads, mask, block,
                None if out is None else out.data_ptr(), 0 if out is None else out.numel(),
                self.info))

        on_gpu = self._index >= 0
        host = torch.empty(1024 + 2 * table.size, dtype=torch.int32, pin_memory=on_gpu)
        plan(host)
        if self.info.words > host.numel():
            host = torch.empty(self.info.words, dtype=torch.int32, pin_memory=on_gpu)
            plan(host)
        host = host[:self.info.words]
        info = self.info
        self._address = C.addressof(info)
        self._q_shape, self._kv_shape = (info.rows, info.hq, 128), (info.rows, info.hkv, 128)
        self._out_shape = (info.rows, info.hq * 128)
        self._workspace = lib.drt_op_paged_attention_workspace_bytes(info)
        if not on_gpu:
            self._list = host
            return
        with torch.cuda.device(self._index):
            self._list = host.to(cache.data.device, non_blocking=True)
            self._at = self._list.data_ptr()
            self._ready = torch.cuda.Event()
            self._ready.record()
            self._stream = torch._C._cuda_getCurrentRawStream(self._index)

    @property
    def rows(self) -> int:
        """The rows of all sequences: what q, k and v have."""
        return self.info.rows

    @property
    def heads(self) -> int:
        return self.info.hq

    def __deepcopy__(self, memo):
        return self  # (a plan does not change)

    def _elsewhere(self):
        """The list is used on a stream that is not the one it was copied on."""
        if _capturing(self._index):
            # (a stream's wait would become the graph's, and the copy is no part of it)
            _lib.check(_lib.load().drt_event_wait(self._ready.cuda_event))
            return
        stream = torch.cuda.current_stream(self._index)
        stream.wait_event(self._ready)
        self._list.record_stream(stream)


class PagedKVCache:
    """Keys and values of ``layers`` layers in ``pages`` pages of ``page_size`` keys (a power of
    two from 32 on) and ``kv_heads`` heads of 128, on one device; ``dtype`` is ``"f16"`` or
    ``"bf16"``. Pages hold the 32-key tiles of :class:`.kernels.PrefixKVCache`.

    Which pages a sequence has, and in which order, is the caller's: :meth:`batch` takes the
    lists. A page may be given to another sequence without clearing it.

    Calls may be on any stream; that one which reads comes behind the one which wrote is the
    caller's to see to, as for any tensor. Keep the cache as long as a captured graph that used it
    is replayed. A deep copy has pages of its own, and takes the same batches."""

    def __init__(self, layers: int, kv_heads: int, pages: int, *, page_size: int = 64,
                 dtype="f16", device=None):
        self.layers, self.kv_heads, self.pages = int(layers), int(kv_heads), int(pages)
        self.page_size = int(page_size)
        if self.layers < 1 or self.kv_heads < 1 or self.pages < 1:
            raise ValueError("a paged cache has a layer, a K/V head and a page at least")
        if self.page_size < 32 or self.page_size & (self.page_size - 1):
            raise ValueError("page_size must be a power of two from 32 on")
        if self.pages * self.kv_heads * (self.page_size // 32) > _I32_MAX:
            raise ValueError("a layer has at most 2^31 - 1 tiles of 32 keys and one head")
        self.kv_dtype = _cache_dtype(dtype)
        if self.kv_dtype == _lib.I8:
            raise ValueError("a paged cache's dtype is 'f16' or 'bf16'")
        self.dtype = torch.bfloat16 if self.kv_dtype == _lib.BF16 else torch.float16
        self.data = torch.zeros((self.layers, self.pages, self.kv_heads,
                                 self.page_size // 32 * KV_TILE_ELEMS), dtype=self.dtype,
                                device=_before_captures(device, "a cache"))
        self._index = self.data.get_device()
        self._own_streams()
        self._geometry = (self.kv_heads, self.pages, self.page_size, self._index)
        self._layer_bytes = self.data.stride(0) * 2
        self._lib = None

    def __deepcopy__(self, memo):
        _before_captures(self.data.device, "a cache's copy")
        other = copy.copy(self)
        other.data = self.data.clone()
        other._own_streams()
        return other

    def _own_streams(self):
        """The tensor was made on the current stream: what fills it is done before any other uses it."""
        self._streams = ()
        if self._index >= 0:
            stream = torch.cuda.current_stream(self._index)
            stream.synchronize()
            self._streams = {stream.cuda_stream}

    @property
    def nbytes(self) -> int:
        return self.data.numel() * 2

    def batch(self, pages, keys, rows, *, heads: int, positions=None, kind: str = "causal",
              mask_geometry=None) -> PagedBatch:
        """The plan of a step of several sequences.

        For each sequence: ``pages``, its page numbers in order (a list each, or int32
        ``[sequences, width]`` on the host); ``keys``, how many keys it has, this step's with
        them; ``rows``, how many rows are new. The rows of all sequences come one sequence's
        behind the other's; they are a sequence's last positions, or ``positions`` says where the
        first is. ``heads`` is the number of query heads.

        ``kind``: ``"full"`` (every key of the sequence), ``"causal"`` (those up to the row's
        position) or ``"d2f_hybrid"`` with ``mask_geometry`` (prompt length, block size): the
        prompt, then whole blocks up to the row's own; the prompt length a number or one for each
        sequence."""
        return PagedBatch(self, pages, keys, rows, heads, positions, kind, mask_geometry)

    def _entry(self, layer, batch):
        """The library, the batch's list on the device and the layer's pages, once a call's layer and
        batch are checked and both are the current stream's to use."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer must be in [0, {self.layers})")
        if self._index < 0:
            raise ValueError("the cache must be on a GPU")
        if not isinstance(batch, PagedBatch) or (batch._geometry is not self._geometry and
                                                 batch._geometry != self._geometry):
            raise ValueError("the batch was planned for another cache")
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        if stream not in self._streams:
            _lend(self.data, self._index, self._streams)
        if stream != batch._stream:
            batch._elsewhere()
        if self._lib is None:
            self._lib = _lib.load()
        return self._lib, batch._at, self.data.data_ptr() + layer * self._layer_bytes

    def _bad_source(self, what, t, shape):
        if t.shape != shape or t.get_device() != self._index:
            raise ValueError(f"{what} must be {list(shape)} on the cache's device")
        raise ValueError(f"{what}: a head's elements must be side by side")

    def append(self, layer: int, k, v, batch: PagedBatch, *, rotary=None, q=None):
        """Write the batch's ``k, v [rows, kv_heads, 128]`` (fp32, fp16 or bf16, views of a fused
        projection as they are) into its sequences' pages.

        ``rotary`` (a :class:`.rotary.RotaryPositions` of a multiple of 16 elements): keys are
        turned by their positions on the way, and so is ``q [rows, heads, 128]`` where given,
        which comes back in the cache's type, ready for :meth:`attention`. Each value is rounded
        once. Raises ValueError where two sequences of the batch have rows in one tile of a page,
        or a row lies behind its sequence's keys."""
        lib, plan, pages = self._entry(layer, batch)
        index, shape = self._index, batch._kv_shape
        if k.shape != shape or k.get_device() != index or k.stride(2) != 1:
            self._bad_source("append's k", k, shape)
        if v.shape != shape or v.get_device() != index or v.stride(2) != 1:
            self._bad_source("append's v", v, shape)
        k0, k1, _ = k.stride()
        v0, v1, _ = v.stride()
        dtype = k.dtype
        code = _TYPES.get(dtype)
        if code is None or v.dtype is not dtype:
            raise ValueError("append takes k, v and q of one type: float32, float16 or bfloat16")
        turns = None
        if rotary is not None:
            if rotary.dim > 128 or rotary.dim % 16 or rotary._index != index:
                raise ValueError("append's rotary must turn a multiple of 16 elements, 128 at "
                                 "most, on the cache's device")
            turns = rotary._address
            if torch._C._cuda_getCurrentRawStream(index) not in rotary._streams:
                _lend(rotary.turns, index, rotary._streams)
        if q is None:
            out = q_at = out_at = None
            q0 = q1 = 0
        else:
            shape = batch._q_shape
            if q.shape != shape or q.get_device() != index or q.stride(2) != 1:
                self._bad_source("append's q", q, shape)
            q0, q1, _ = q.stride()
            if q.dtype is not dtype:
                raise ValueError("append takes k, v and q of one type: float32, float16 or "
                                 "bfloat16")
            out = q.new_empty(shape, dtype=self.dtype)
            q_at, out_at = q.data_ptr(), out.data_ptr()
        _launch(torch, lib.drt_op_paged_append, index, batch._address, plan,
                k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, q_at, q0, q1, code, turns,
                pages, self.kv_dtype, out_at)
        return out

    def load(self, layer: int, batch: PagedBatch):
        """``(k, v) [rows, kv_heads, 128]`` of the batch's rows as the cache holds them. Raises
        ValueError where :meth:`append` of the batch does."""
        lib, plan, pages = self._entry(layer, batch)
        k = self.data.new_empty(batch._kv_shape)
        v = self.data.new_empty(batch._kv_shape)
        _launch(torch, lib.drt_op_paged_load, self._index, batch._address, plan,
                pages, self.kv_dtype, k.data_ptr(), v.data_ptr())
        return k, v

    def attention(self, layer: int, q, batch: PagedBatch, *, out_dtype=None):
        """Attention of the batch's ``q [rows, heads, 128]`` (the cache's type) over the keys that
        each row sees: ``[rows, heads * 128]`` in fp32 or bf16. A row without any gives zeros.

        Scores, softmax sums and results are held in fp32; the weights are rounded to the cache's
        type for their product with the values (a row's result in fp32 is off by up to about 2.5
        parts in 10^4 of its size over an fp16 cache, 2 in 10^3 over a bf16 one)."""
        lib, plan, pages = self._entry(layer, batch)
        if q.shape != batch._q_shape or q.dtype is not self.dtype or \
                q.get_device() != self._index or not q.is_contiguous():
            raise ValueError(f"q must be contiguous {list(batch._q_shape)} of the cache's type and "
                             "device")
        if out_dtype is None:
            out_dtype = torch.float32
        if out_dtype is not torch.float32 and out_dtype is not torch.bfloat16:
            raise ValueError("attention out must be float32 or bfloat16")
        out = q.new_empty(batch._out_shape, dtype=out_dtype)
        need = batch._workspace
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        _launch(torch, lib.drt_op_paged_attention, self._index, batch._address, plan,
                q.data_ptr(), pages, self.kv_dtype,
                out.data_ptr(), _lib.BF16 if out_dtype is torch.bfloat16 else _lib.F32,
                None if ws is None else ws.data_ptr(), need)
        return out

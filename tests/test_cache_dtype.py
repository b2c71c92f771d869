"""A cache is of the type its caller names, or refused (no GPU)."""
from __future__ import annotations

import pytest

from diffusorrt_amd import _lib

torch = pytest.importorskip("torch")


def _cache(dtype):
    from diffusorrt_amd.kernels import PrefixKVCache

    return PrefixKVCache(1, 2, 64, dtype=dtype, device="cpu")


@pytest.mark.parametrize("dtype", ["int8", "I8", "fp8", "q8", "", "bfloat16", 8, torch.int8,
                                   torch.bfloat16, torch.uint8])
def test_a_type_that_no_cache_has_is_refused(dtype):
    from diffusorrt_amd import kernels

    with pytest.raises(ValueError, match="'f16', 'bf16' or 'i8'"):
        _cache(dtype)
    x = torch.zeros((4, 2, 128))
    with pytest.raises(ValueError, match="'f16', 'bf16' or 'i8'"):
        kernels.attention(x, x, x, head_dim=128, kind="full", kv_dtype=dtype)


@pytest.mark.parametrize("dtype,code,data", [
    ("f16", _lib.F16, torch.float16), ("bf16", _lib.BF16, torch.bfloat16),
    ("i8", _lib.I8, torch.uint8), ("fp16", _lib.F16, torch.float16),
    ("float16", _lib.F16, torch.float16), (torch.float16, _lib.F16, torch.float16),
    (None, _lib.F16, torch.float16)])
def test_a_cache_of_each_type(dtype, code, data):
    cache = _cache(dtype)
    assert cache.kv_dtype == code and cache.data.dtype is data
    assert (cache.scales is not None) == (code == _lib.I8)


def test_a_runtime_refuses_an_8_bit_cache():
    from diffusorrt_amd.runtime import Runtime

    with pytest.raises(ValueError, match="PrefixKVCache"):
        Runtime(None, kv_dtype="i8")

"""The key/value cache's Python arguments without a GPU: numbers past 32 bits are refused, not
taken modulo 2^32."""
import ctypes

import pytest

import jhq_gpu_amd as jg

GOOD = dict(num_pages=4, page_size=16, kv_heads=2, head_dim=64, bits=8)


@pytest.mark.parametrize("name", GOOD)
@pytest.mark.parametrize("more", [1 << 32, 1 << 64, -(1 << 32)])
def test_cache_parameters_past_32_bits(name, more):
    with pytest.raises(ValueError, match=name):
        jg.KVCache(**{**GOOD, name: GOOD[name] + more}, device="cpu")


def test_query_heads_past_32_bits():
    cache = object.__new__(jg.KVCache)  # the parameters alone: no device memory
    cache._c = jg._KvParams(8, 2, 64, 16, 4)
    cache._ref = ctypes.byref(cache._c)
    batch = type("Batch", (), {})()
    batch._c = jg._KvBatch(1, 4, 1 << 20, 1 << 20, 1 << 20, 1, 1, 64)
    batch._ref = ctypes.byref(batch._c)
    assert cache.work_bytes(batch, 4) >= 0
    for bad in ((1 << 32) + 4, 4 - (1 << 32)):
        with pytest.raises(ValueError, match="q_heads"):
            cache.work_bytes(batch, bad)

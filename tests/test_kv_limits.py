"""The key/value cache's entry points at the ends of their integers, without a GPU: sizes that no
call can have are refused or cut, and never divided by."""
import ctypes

import pytest

import jhq_gpu_amd as jg

FAKE = 1 << 20  # never dereferenced: nothing is launched


def _work(n_tokens, max_q, max_kv, kv_heads, q_heads, head_dim, n_seq=1):
    p = jg._KvParams(8, kv_heads, head_dim, 64, 10)
    b = jg._KvBatch(n_seq, 1 << 20, FAKE, FAKE, FAKE, n_tokens, max_q, max_kv)
    P, B = ctypes.byref(p), ctypes.byref(b)
    n = jg.lib().jhq_kv_work_bytes(P, B, q_heads, 0)
    if n < 0:  # the call itself refuses it too
        assert jg.lib().jhq_k_kv_attend(P, FAKE, B, FAKE, 512, 128, q_heads, 3, 0.1, 1, 0, FAKE, None,
                                        FAKE, 1 << 62, None) == jg.JHQ_EINVAL
    return n


@pytest.mark.parametrize("head_dim", [64, 256])
@pytest.mark.parametrize("q_heads", [2, 8, 16384])
@pytest.mark.parametrize("n_tokens", [1 << 31, 1 << 40, 1 << 50, (1 << 59) + 1, (1 << 63) - 1])
def test_more_rows_than_cu_q_can_name(n_tokens, q_heads, head_dim):
    for max_q in (1, 40, 1 << 16):
        for max_kv in (100, 1 << 26, 1 << 30):
            n = _work(n_tokens, max_q, max_kv, 2, q_heads, head_dim)
            assert n == _work((1 << 31) - 1, max_q, max_kv, 2, q_heads, head_dim)
            assert -1 <= n <= 1 << 50
            if n < 0:
                assert "workspace" in jg.lib().jhq_last_error().decode()


@pytest.mark.parametrize("max_q,G", [(1 << 30, 2), (1 << 30, 512), (1 << 25, 16384), (1 << 30, 16384)])
@pytest.mark.parametrize("n_seq", [1, 64])
def test_more_rows_of_a_key_head_than_an_int_holds(max_q, G, n_seq):
    assert _work(1 << 30, max_q, 1 << 26, 1, G, 128, n_seq) == -1
    assert "max_q" in jg.lib().jhq_last_error().decode()
    assert _work(1 << 30, (1 << 30) // G, 1 << 26, 1, G, 128, n_seq) >= -1

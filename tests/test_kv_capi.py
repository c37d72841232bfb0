"""The key/value cache's entry points without a GPU: sizes, and what they refuse
before anything is launched (jhq_kv_bytes, jhq_kv_work_bytes, jhq_k_kv_*)."""
import ctypes

import pytest

import jhq_gpu_amd as jg

FAKE = 1 << 20  # never dereferenced: the call is refused first


def _params(**kw):
    p = dict(bits=8, kv_heads=2, head_dim=128, page_size=64, num_pages=10)
    p.update(kw)
    return jg._KvParams(p["bits"], p["kv_heads"], p["head_dim"], p["page_size"], p["num_pages"])


def _batch(**kw):
    b = dict(n_seq=3, max_pages=4, pages=FAKE, kv_len=FAKE, cu_q=FAKE, n_tokens=9, max_q=4,
             max_kv=200)
    b.update(kw)
    return jg._KvBatch(b["n_seq"], b["max_pages"], b["pages"], b["kv_len"], b["cu_q"],
                       b["n_tokens"], b["max_q"], b["max_kv"])


def _err():
    return jg.lib().jhq_last_error().decode()


@pytest.mark.parametrize("bits,D,page,row", [(8, 128, 64, 128), (4, 128, 16, 64), (8, 64, 1024, 64),
                                              (4, 64, 32, 32), (8, 256, 16, 256)])
def test_bytes(bits, D, page, row):
    p = _params(bits=bits, head_dim=D, page_size=page)
    assert jg.lib().jhq_kv_bytes(ctypes.byref(p)) == 10 * 2 * page * (2 * row + 8)
    p = _params(bits=bits, head_dim=D, page_size=page, num_pages=0)
    assert jg.lib().jhq_kv_bytes(ctypes.byref(p)) == 0


BAD_PARAMS = [
    (dict(bits=2), "bits"), (dict(bits=16), "bits"), (dict(kv_heads=0), "kv_heads"),
    (dict(kv_heads=2000), "kv_heads"), (dict(head_dim=96), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(page_size=8), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"),
    (dict(num_pages=-1), "num_pages"), (dict(num_pages=1 << 31), "num_pages"),
]


@pytest.mark.parametrize("kw,msg", BAD_PARAMS)
def test_parameters_are_refused_everywhere(kw, msg):
    L, p, b = jg.lib(), _params(**kw), _batch()
    P, B = ctypes.byref(p), ctypes.byref(b)
    assert L.jhq_kv_bytes(P) == 0 and msg in _err()
    assert L.jhq_kv_work_bytes(P, B, 4, 0) == -1 and msg in _err()
    assert L.jhq_k_kv_write(P, FAKE, B, FAKE, 256, 128, FAKE, 256, 128, 3, None) == jg.JHQ_EINVAL
    assert msg in _err()
    assert L.jhq_k_kv_read(P, FAKE, B, FAKE, FAKE, 3, None) == jg.JHQ_EINVAL and msg in _err()
    assert L.jhq_k_kv_attend(P, FAKE, B, FAKE, 512, 128, 4, 3, 0.1, 1, 0, FAKE, None, FAKE,
                             1 << 40, None) == jg.JHQ_EINVAL and msg in _err()


BAD_BATCH = [
    (dict(n_seq=-1), "negative"), (dict(max_pages=-1), "negative"), (dict(n_tokens=-1), "negative"),
    (dict(max_q=-1), "negative"), (dict(max_kv=-1), "negative"), (dict(max_kv=(1 << 30) + 1), "2^30"),
    (dict(max_q=(1 << 30) + 1), "2^30"), (dict(kv_len=None), "null array"),
    (dict(cu_q=None), "null array"), (dict(pages=None), "null array"),
]


@pytest.mark.parametrize("kw,msg", BAD_BATCH)
def test_batches_are_refused_everywhere(kw, msg):
    L, p, b = jg.lib(), _params(), _batch(**kw)
    P, B = ctypes.byref(p), ctypes.byref(b)
    assert L.jhq_kv_work_bytes(P, B, 4, 0) == -1 and msg in _err()
    assert L.jhq_k_kv_write(P, FAKE, B, FAKE, 256, 128, FAKE, 256, 128, 3, None) == jg.JHQ_EINVAL
    assert msg in _err()
    assert L.jhq_k_kv_read(P, FAKE, B, FAKE, FAKE, 3, None) == jg.JHQ_EINVAL and msg in _err()
    assert L.jhq_k_kv_attend(P, FAKE, B, FAKE, 512, 128, 4, 3, 0.1, 1, 0, FAKE, None, FAKE,
                             1 << 40, None) == jg.JHQ_EINVAL and msg in _err()


def _attend(p=None, b=None, cache=FAKE, q=FAKE, heads=4, dtype=3, scale=0.1, causal=1, window=0,
            out=FAKE, work=FAKE, work_bytes=1 << 40):
    p, b = p or _params(), b or _batch()
    return jg.lib().jhq_k_kv_attend(ctypes.byref(p), cache, ctypes.byref(b), q, 512, 128, heads,
                                    dtype, scale, causal, window, out, None, work, work_bytes, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(cache=None), "null cache"), (dict(cache=FAKE + 8), "aligned"), (dict(heads=3), "multiple"),
    (dict(heads=0), "multiple"), (dict(heads=32768), "at most"), (dict(dtype=0), "queries"),
    (dict(dtype=7), "queries"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(causal=2), "causal"), (dict(window=-1), "window"),
    (dict(causal=0, window=5), "window"), (dict(q=None), "null queries"), (dict(out=None), "null"),
])
def test_attend_refuses(kw, msg):
    assert _attend(**kw) == jg.JHQ_EINVAL
    assert msg in _err()


def test_workspace_is_checked():
    p, b = _params(), _batch(n_seq=1, n_tokens=1, max_q=1, max_kv=256, max_pages=4)
    b2 = _batch(n_seq=1, n_tokens=1, max_q=1, max_kv=1 << 20, max_pages=1 << 14)
    n = jg.lib().jhq_kv_work_bytes(ctypes.byref(p), ctypes.byref(b2), 4, 0)
    assert n >= 0
    if n:  # a long sequence's partial results
        assert _attend(p, b2, work_bytes=n - 1) == jg.JHQ_EINVAL and "workspace" in _err()
        assert _attend(p, b2, work=None) == jg.JHQ_EINVAL and "workspace" in _err()
        assert _attend(p, b2, work=FAKE + 4) == jg.JHQ_EINVAL and "aligned" in _err()
    assert jg.lib().jhq_kv_work_bytes(ctypes.byref(p), ctypes.byref(b), 5, 0) == -1


@pytest.mark.parametrize("kw", [dict(n_seq=0), dict(n_tokens=0), dict(max_q=0)])
def test_nothing_to_do_is_no_error(kw):
    L, p, b = jg.lib(), _params(), _batch(**kw)
    P, B = ctypes.byref(p), ctypes.byref(b)
    assert L.jhq_kv_work_bytes(P, B, 4, 0) == 0
    assert L.jhq_k_kv_write(P, FAKE, B, None, 0, 0, None, 0, 0, 3, None) == jg.JHQ_OK
    assert L.jhq_k_kv_read(P, FAKE, B, None, None, 3, None) == jg.JHQ_OK
    assert _attend(p, b, q=None, out=None, work=None, work_bytes=0) == jg.JHQ_OK


def test_write_and_read_refuse():
    L, p, b = jg.lib(), _params(), _batch()
    P, B = ctypes.byref(p), ctypes.byref(b)
    for dt in (1, 2, 5, -1):  # bytes are no rows of a cache
        assert L.jhq_k_kv_write(P, FAKE, B, FAKE, 1, 1, FAKE, 1, 1, dt, None) == jg.JHQ_EINVAL
        assert L.jhq_k_kv_read(P, FAKE, B, FAKE, FAKE, dt, None) == jg.JHQ_EINVAL
    assert L.jhq_k_kv_write(P, FAKE, B, None, 1, 1, FAKE, 1, 1, 3, None) == jg.JHQ_EINVAL
    assert "null" in _err()
    assert L.jhq_k_kv_write(P, None, B, FAKE, 1, 1, FAKE, 1, 1, 3, None) == jg.JHQ_EINVAL
    assert L.jhq_k_kv_write(None, FAKE, B, FAKE, 1, 1, FAKE, 1, 1, 3, None) == jg.JHQ_EINVAL
    assert L.jhq_k_kv_write(P, FAKE, None, FAKE, 1, 1, FAKE, 1, 1, 3, None) == jg.JHQ_EINVAL


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_a_cache_is_on_a_gpu(device):
    with pytest.raises(ValueError, match="GPU"):
        jg.KVCache(4, 16, 2, 64, device=device)

"""Attention with a shared prefix without a GPU: what the entry points refuse before anything is
launched, and workspaces at the ends of their integers."""
import ctypes

import pytest

import jhq_gpu_amd as jg

FAKE = 1 << 20  # never dereferenced: the call is refused first


def _batch(**kw):
    b = dict(n_seq=3, max_pages=1 << 16, pages=FAKE, kv_len=FAKE, cu_q=FAKE, n_tokens=9, max_q=4, max_kv=200)
    b.update(kw)
    return jg._KvBatch(b["n_seq"], b["max_pages"], b["pages"], b["kv_len"], b["cu_q"], b["n_tokens"],
                       b["max_q"], b["max_kv"])


def _err():
    return jg.lib().jhq_last_error().decode()


def _calls(b, p, heads=4, once=0, work=FAKE, work_bytes=1 << 60, **kw):
    a = dict(cache=FAKE, q=FAKE, out=FAKE, dtype=3, causal=1)
    a.update(kw)
    L, P = jg.lib(), ctypes.byref(jg._KvParams(8, 2, 128, 64, 10))
    B, R = ctypes.byref(b), ctypes.byref(p) if p else None
    n = L.jhq_kv_shared_work_bytes(P, B, R, once, heads)
    rc = L.jhq_k_kv_attend_shared(P, a["cache"], B, R, once, a["q"], 512, 128, heads, a["dtype"], 0.1, a["causal"],
                                  a["out"], None, work, work_bytes, None)
    return n, rc


@pytest.mark.parametrize("b,p,msg", [
    (dict(), None, "null prefix"), (dict(), dict(n_tokens=8), "number of rows"),
    (dict(), dict(n_seq=-1), "negative"), (dict(), dict(max_kv=(1 << 30) + 1), "2^30"),
    (dict(), dict(max_q=(1 << 30) + 1), "2^30"), (dict(), dict(max_q=1 << 30), "max_q"),
    (dict(), dict(kv_len=None), "null array"), (dict(), dict(pages=None), "null array"),
    (dict(max_q=1 << 30), dict(), "max_q"), (dict(cu_q=None), dict(), "null array"),
])
def test_batches_are_refused(b, p, msg):
    n, rc = _calls(_batch(**b), None if p is None else _batch(**p))
    assert n == -1 and rc == jg.JHQ_EINVAL and msg in _err()


@pytest.mark.parametrize("kw,msg", [
    (dict(once=2), "once"), (dict(cache=None), "null cache"), (dict(q=None), "null queries"), (dict(out=None), "null"),
    (dict(dtype=0), "queries"), (dict(causal=2), "causal"), (dict(work=None), "null workspace"),
    (dict(work=FAKE + 4), "aligned"), (dict(work_bytes=0), "workspace"), (dict(heads=3), "multiple"),
])
def test_arguments_are_refused(kw, msg):
    kw = dict(dict(once=1), **kw)
    _, rc = _calls(_batch(), _batch(), **kw)
    assert rc == jg.JHQ_EINVAL and msg in _err()


def test_nothing_to_do_is_no_error():
    for kw in (dict(n_seq=0), dict(n_tokens=0), dict(max_q=0)):
        n, rc = _calls(_batch(**kw), _batch(n_tokens=kw.get("n_tokens", 9)), q=None, out=None, work=None,
                       work_bytes=0)
        assert n == 0 and rc == jg.JHQ_OK


@pytest.mark.parametrize("n_tokens", [1, 3, 1 << 20, 1 << 31, 1 << 45, (1 << 63) - 1])
@pytest.mark.parametrize("max_q,rows", [(1, 3), (4, 1000), (7, 1 << 20), (100, 1 << 25)])
def test_workspaces(n_tokens, max_q, rows):
    """Enough for the passes' parts, and refused past 2^50 bytes instead of overflowing."""
    for lead_kv in (0, 100, 5000, 1 << 30):
        for n_lead in (0, 1, 1 << 20):
            b = _batch(n_tokens=n_tokens, max_q=max_q, max_kv=1 << 22)
            p = _batch(n_tokens=n_tokens, max_q=rows, max_kv=lead_kv, n_seq=n_lead)
            for once in (0, 1):
                n, _ = _calls(b, p, once=once, cache=None)
                assert -1 <= n <= 1 << 50
                if n < 0:
                    assert "2^50" in _err() or n_tokens > 1 << 30

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


def _work(b, p, once, heads=4, D=128, bits=8, H=2):
    """Bytes with the prefix and without it, and what the former says."""
    L, P = jg.lib(), ctypes.byref(jg._KvParams(bits, H, D, 64, 10))
    n = L.jhq_kv_shared_work_bytes(P, ctypes.byref(b), ctypes.byref(p), once, heads)
    msg = _err()
    return n, L.jhq_kv_work_bytes(P, ctypes.byref(b), heads, 0), msg


@pytest.mark.parametrize("D", [64, 128, 256])
def test_once_ends_where_a_call_does(D):
    """Read once up to the documented rows and steps; past them it is attention of every sequence, whose
    workspace it then has."""
    def call(tokens, max_kv=5000, n_seq=3, heads=4):
        return _work(_batch(n_tokens=tokens, n_seq=n_seq), _batch(n_tokens=tokens, max_q=tokens, max_kv=max_kv, n_seq=1),
                     1, heads=heads, D=D)
    most = (1 << 31) // D // 4
    n, plain, _ = call(most - 1)
    # every row has a place of its own in both passes: sums of values, maximum and sum
    assert n >= 2 * (most - 1) * 4 * (D + 2) * 4 and n > plain
    n, plain, _ = call(most)
    assert n == plain
    # 1000 rows of 2 key heads, 2 query heads each, in tiles of 64 at least: 64 tokens a step
    n, plain, _ = call(1000, max_kv=1 << 24)
    assert n > plain
    n, plain, _ = call(100000, max_kv=1 << 30)
    assert n == plain
    n, plain, _ = call(1000, max_kv=0)
    assert n == plain


@pytest.mark.parametrize("n_tokens", [1, 9, 1000, 1 << 19])
@pytest.mark.parametrize("bits,D,H", [(8, 64, 8), (4, 128, 2), (8, 256, 1)])
@pytest.mark.parametrize("max_q,G", [(1, 1), (1, 8), (4, 4), (100, 2)])
def test_workspaces_have_room(n_tokens, bits, D, H, max_q, G):
    """For every row's place in both passes, for two parts of 16 rows of each workgroup, and for 8 bytes a
    key head of every tile that the rows can be cut into; no more than a hundred times that of the parts."""
    b = _batch(n_tokens=n_tokens, max_q=max_q, max_kv=9000, n_seq=5)
    p = _batch(n_tokens=n_tokens, max_q=min(n_tokens, 5 * max_q), max_kv=5000, n_seq=2)
    n, plain, _ = _work(b, p, 1, heads=H * G, D=D, bits=bits, H=H)
    rows = n_tokens * H * G
    if rows >= (1 << 31) // D:
        assert n == plain
        return
    each = (D + 2) * 4
    tiles = (n_tokens * G // 128 + 2 + n_tokens * G // 128 + 5) * H * 8
    parts = 2 * 2 * 256 * 16 * each
    assert n >= 2 * rows * each + parts + tiles
    most = (n_tokens * G // 16 + 2 + n_tokens * G // 16 + 5) * H * 8
    assert n <= 2 * rows * each + 100 * parts + most + 64


def test_workspaces_past_2_50_bytes_are_refused():
    """Attention of every sequence, which keeps every row of the call (2^31 x 64 of 130 floats, 2^50 bytes) for
    each of its parts: one sequence's few tiles over a context of 2^30 have many."""
    b = _batch(n_tokens=1 << 31, n_seq=1, max_q=16, max_kv=1 << 30, max_pages=1 << 24)
    p = _batch(n_tokens=1 << 31, n_seq=1, max_q=16, max_kv=5000)
    for once in (0, 1):
        n, plain, msg = _work(b, p, once, heads=64)
        assert n == plain == -1 and "2^50" in msg

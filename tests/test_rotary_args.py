"""Rotary positions without a GPU: frequencies as parts of a turn, scalings, refusals."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

import jhq_gpu_amd as jg
from jhq_gpu_amd import rotary
from rotary_ref import PER_TURN

FAKE = 1 << 20  # never dereferenced: the call is refused first


def _err():
    return jg.lib().jhq_last_error().decode()


def test_turns_are_exact():
    """The nearest 2^-64th of a turn, modulo one, for any float64."""
    for x in (1.0, 2 * math.pi, 1e-4, 123456.789, -0.3, 0.0, 2.0 ** -70, 1e12):
        n = rotary.turns([x])[0]
        assert -1 << 63 <= n < 1 << 63
        d = (Fraction(n, 1 << 64) - Fraction(x) * PER_TURN) % 1
        assert min(d, 1 - d) <= Fraction(1, 1 << 65) + Fraction(abs(x)) / (1 << 126)


def test_scalings():
    r, b = 64, 10000.0
    w = np.array([b ** (-2 * i / r) for i in range(r // 2)])

    def of(**kw):
        f, a = rotary._scaled(r, b, kw or None)
        return np.array(f), a
    assert np.allclose(of()[0], w, rtol=1e-14) and of()[1] == 1.0
    assert np.allclose(of(kind="linear", factor=4)[0], w / 4, rtol=1e-14)
    n = of(kind="ntk", factor=4)[0]
    # the fastest pair stays, the slowest turns `factor` times slower
    assert n[0] == 1.0 and math.isclose(n[-1], w[-1] / 4, rel_tol=1e-12)
    y, a = of(kind="yarn", factor=8, length=4096)
    assert math.isclose(a, 0.1 * math.log(8) + 1)
    turns = 4096 * w / (2 * math.pi)
    assert np.allclose(y[turns > 60], w[turns > 60]) and np.allclose(y[turns < 0.5], w[turns < 0.5] / 8)
    assert (np.diff(y) < 0).all() and (y <= w).all() and (y >= w / 8 * (1 - 1e-12)).all()
    s, a = of(kind="bands", factor=8, length=4096)
    assert a == 1.0
    assert np.allclose(s[turns > 4], w[turns > 4]) and np.allclose(s[turns < 1], w[turns < 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and (s[mid] < w[mid]).all() and (s[mid] > w[mid] / 8).all()


@pytest.mark.parametrize("kw,msg", [
    (dict(head_dim=0), "head_dim"), (dict(head_dim=63), "head_dim"), (dict(head_dim=1026), "head_dim"),
    (dict(head_dim=(1 << 32) + 64), "head_dim"), (dict(rot_dim=0), "rot_dim"),
    (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=7), "rot_dim"), (dict(base=0.0), "base"),
    (dict(base=float("nan")), "base"), (dict(scaling=dict(kind="other", factor=2)), "kind"),
    (dict(scaling=dict(factor=2)), "kind"), (dict(scaling=dict(kind="linear")), "needs factor"),
    (dict(scaling=dict(kind="linear", factor=0)), "positive"),
    (dict(scaling=dict(kind="linear", factor=2, length=4)), "no length"),
    (dict(scaling=dict(kind="yarn", factor=2)), "needs length"),
    (dict(scaling=dict(kind="bands", factor=2, length=9, low=4, high=4)), "low"),
    (dict(scaling=dict(kind="ntk", factor=2), rot_dim=2), "ntk"),
    (dict(scaling=dict(kind="yarn", factor=2, length=9), base=1.0), "base"),
    (dict(frequencies=[1.0]), "frequencies must be 32"),
    (dict(frequencies=[1.0] * 31 + [float("inf")]), "finite"),
    (dict(frequencies=[1.0] * 32, scaling=dict(kind="linear", factor=2)), "does not apply"),
    (dict(amplitude=float("nan")), "amplitude"), (dict(amplitude=1e39), "amplitude"),
    (dict(), "GPU"),
])
def test_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        jg.Rotary(**{**dict(head_dim=64, device="cpu"), **kw})


def _rot(head_dim=128, rot_dim=128, interleaved=0, amplitude=1.0, turns=FAKE):
    return jg._Rotary(head_dim, rot_dim, interleaved, amplitude, turns)


def _call(r=None, x=FAKE, n=5, heads=3, dtype=3, pos=FAKE, size=4, b=None, inverse=0, out=FAKE):
    r = r or _rot()
    return jg.lib().jhq_k_rotary(ctypes.byref(r), x, 384, 128, n, heads, dtype, pos, size,
                                 ctypes.byref(b) if b else None, inverse, out, 384, 128, None)


def _batch(n_seq=2, kv_len=FAKE, cu_q=FAKE, n_tokens=5):
    return jg._KvBatch(n_seq, 1, FAKE, kv_len, cu_q, n_tokens, 5, 16)


@pytest.mark.parametrize("kw,msg", [
    (dict(r=_rot(head_dim=127)), "head_dim"), (dict(r=_rot(head_dim=2048)), "head_dim"),
    (dict(r=_rot(rot_dim=0)), "rot_dim"), (dict(r=_rot(rot_dim=130)), "rot_dim"),
    (dict(r=_rot(rot_dim=3)), "rot_dim"), (dict(r=_rot(interleaved=2)), "interleaved"),
    (dict(r=_rot(amplitude=float("inf"))), "amplitude"), (dict(r=_rot(turns=None)), "turns"),
    (dict(r=_rot(turns=FAKE + 4)), "turns"), (dict(dtype=1), "rows must be"), (dict(n=-1), "n_tokens"),
    (dict(n=1 << 31), "n_tokens"), (dict(heads=-1), "heads"), (dict(heads=1 << 21), "heads"),
    (dict(inverse=2), "inverse"), (dict(pos=None), "positions"), (dict(b=_batch()), "positions"),
    (dict(size=2), "4 or 8"), (dict(pos=None, b=_batch(n_tokens=6)), "number of rows"),
    (dict(pos=None, b=_batch(n_seq=-1)), "negative"), (dict(pos=None, b=_batch(cu_q=None)), "null array"),
    (dict(x=None), "null rows"), (dict(out=None), "null rows"),
    (dict(n=(1 << 31) - 1, heads=1, r=_rot(head_dim=1024, rot_dim=1024), x=FAKE + 1), "more work"),
])
def test_the_entry_point_refuses(kw, msg):
    assert _call(**kw) == jg.JHQ_EINVAL
    assert msg in _err()


@pytest.mark.parametrize("kw", [dict(n=0, pos=None), dict(heads=0), dict(pos=None, b=_batch(n_seq=0))])
def test_nothing_to_do_is_no_error(kw):
    assert _call(x=None, out=None, **kw) == jg.JHQ_OK


def test_write_refuses_a_rotary_of_other_heads():
    L = jg.lib()
    p = jg._KvParams(8, 2, 128, 64, 10)
    b = _batch()
    P, B = ctypes.byref(p), ctypes.byref(b)

    def call(r):
        return L.jhq_k_kv_write_rotary(P, FAKE, B, FAKE, 256, 128, FAKE, 256, 128, 3,
                                       ctypes.byref(r) if r else None, None)
    assert call(None) == jg.JHQ_EINVAL and "null rotary" in _err()
    assert call(_rot(head_dim=64, rot_dim=64)) == jg.JHQ_EINVAL and "another" in _err()
    assert call(_rot(rot_dim=129)) == jg.JHQ_EINVAL and "rot_dim" in _err()


@pytest.mark.parametrize("kw,msg", [
    (dict(scaling=dict(kind="ntk", factor=1e308)), "range"), (dict(base=1e308, scaling=dict(kind="ntk", factor=100)), "range"),
    (dict(base=5e-324), "range"), (dict(scaling=dict(kind="yarn", factor=2, length=1e308, fast=1e-10, slow=1e-11)), "range"),
    (dict(scaling=dict(kind="linear", factor=5e-324)), "finite"), (dict(scaling=dict(kind="bands", factor=5e-324, length=9)), "finite"),
    (dict(scaling=dict(kind="yarn", factor=2, length=4096, fast=1, slow=32)), "fast must be above slow"),
    (dict(scaling=dict(kind="yarn", factor=2, length=4096, fast=0.5)), "fast must be above slow"),
])
def test_extreme_scalings_are_refused(kw, msg):
    """As any other argument that is not valid, instead of a frequency of 0 or a ramp the wrong way round."""
    with pytest.raises(ValueError, match=msg):
        jg.Rotary(**{**dict(head_dim=64, device="cpu"), **kw})

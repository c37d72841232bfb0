"""float64 restatement of the key/value cache's definition, for the tests:
what a row is held as, and attention over held rows with error bounds."""
import numpy as np

FLOOR = 2.0 ** -60
# unit roundoff of the types rows and outputs come in
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def held(x, bits):
    """float32 codes and scales [.., 1] of rows x (16-bit values, any array that
    holds them exactly): codes in exact arithmetic, the scale one float32
    division."""
    x = np.asarray(x, np.float64)
    top = 127.0 if bits == 8 else 7.0
    with np.errstate(invalid="ignore"):
        big = np.abs(x).max(-1, keepdims=True)
        live = np.isfinite(big) & (big >= FLOOR)
        safe = np.where(live, big, 1.0)
        # both sides of the quotient are exact in float64, so a tie is one
        code = np.rint(np.where(live, x, 0.0) * top / safe)
    scale = np.where(live, np.float32(safe) / np.float32(top), np.float32(0))
    return code.astype(np.float32), np.where(np.isfinite(big), scale, np.float32(np.nan))


def value32(x, bits):
    """What reads back, in float32."""
    code, scale = held(x, bits)
    return code * scale


def visible(q, n, causal, window):
    """[q, n] truth: what the new tokens see."""
    pos = np.arange(n - q, n)[:, None]
    j = np.arange(n)[None, :]
    m = np.ones((q, n), bool)
    if causal:
        m &= j <= pos
        if window:
            m &= j > pos - window
    return m


def attend(q, k, v, scale, causal=True, window=0, unit=0.0):
    """q [a, Hq, D], k, v [n, H, D] float64 -> out [a, Hq, D], lse [a, Hq] and the
    bounds of their errors.

    Bound of out: the weights are rounded to 11 bits before the second product
    (2^-11 relative, or 2^-25 of the row's largest weighted scale where they are
    that small), logits are float32 sums of D products (and a few operations
    more) whose relative error is (D + 8) 2^-24 of the sum of magnitudes, weights
    are exponentials and sums in float32 (n 2^-24 and a few units), and the
    result is rounded once to its type (unit)."""
    a, Hq, D = q.shape
    n, H, _ = k.shape
    G = Hq // H
    out = np.zeros((a, Hq, D))
    lse = np.full((a, Hq), -np.inf)
    tol = np.zeros_like(out)
    ltol = np.zeros_like(lse)
    if n == 0 or a == 0:
        return out, lse, tol, ltol
    m = visible(a, n, causal, window)
    for h in range(Hq):
        kh, vh = k[:, h // G], v[:, h // G]
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(m, q[:, h] @ kh.T * scale, -np.inf)
            mag = np.where(m, np.abs(q[:, h]) @ np.abs(kh).T * abs(scale), 0.0)
        for i in range(a):
            see = m[i]
            if not see.any():
                continue
            x = s[i, see]
            top = x.max()
            w = np.exp(x - top)
            l = w.sum()
            vv = vh[see]
            out[i, h] = w @ vv / l
            lse[i, h] = top + np.log(l)
            # a logit's error also holds one unit of float32 at its own size
            d = mag[i, see].max() * (D + 8) * 2.0 ** -24
            vmax = np.abs(vv).max()
            reach = w @ np.abs(vv) / l
            rel = 2.0 ** -11 + 2 * d + (see.sum() + 16) * 2.0 ** -24
            tol[i, h] = (unit * np.abs(out[i, h]) + reach * rel * (1 + unit)
                         + see.sum() * 2.0 ** -25 * vmax + (2.0 ** -25 if unit == UNIT["f16"] else 0))
            ltol[i, h] = d + (see.sum() + 16) * 2.0 ** -24 + abs(lse[i, h]) * 2.0 ** -22
    return out, lse, tol, ltol

"""Attention over held rows in float64 with the bound of each output's own roundings,
for the tests: kv_ref.attend's, but what the rounding of weights loses is counted token by
token."""
import numpy as np

import kv_ref as ref

# Below this part of a row's largest weight times value scale a weight is rounded to a
# fixed unit: 2^-25 below it (half of float16's smallest number, the largest weight being 2^9
# at least).
LOST = 2.0 ** -34


def attend(q, k, v, codes, scale, causal=True, window=0, unit=0.0):
    """q [a, Hq, D], k, v [n, H, D] as held, float64, codes [n, H, D] of v -> out, lse and
    the bounds of their errors.

    A weighted scale p_j (weight times value scale) is off by 2^-11 of itself or by LOST of
    the row's largest, and by no more than itself; that times its codes is the numerator's
    error.  Logits are float32 sums of D products (and a few operations more), exponentials and
    sums float32 (n 2^-24 and a few units), and the result is rounded once to its type."""
    a, Hq, D = q.shape
    n, H, _ = k.shape
    G = Hq // H
    out, tol = np.zeros((a, Hq, D)), np.zeros((a, Hq, D))
    lse, ltol = np.full((a, Hq), -np.inf), np.zeros((a, Hq))
    if n == 0 or a == 0:
        return out, lse, tol, ltol
    m = ref.visible(a, n, causal, window)
    for h in range(Hq):
        kh, vh, ch = k[:, h // G], v[:, h // G], np.abs(codes[:, h // G]).astype(np.float64)
        vs = np.abs(vh).max(-1) / np.maximum(ch.max(-1), 1)
        logits = q[:, h] @ kh.T * scale
        mags = np.abs(q[:, h]) @ np.abs(kh).T * abs(scale)
        for i in range(a):
            see = m[i]
            if not see.any():
                continue
            x = logits[i, see]
            w = np.exp(x - x.max())
            l = w.sum()
            p = w * vs[see]
            out[i, h] = w @ vh[see] / l
            lse[i, h] = x.max() + np.log(l)
            d = mags[i, see].max() * (D + 8) * 2.0 ** -24
            lost = np.maximum(p * 2.0 ** -11, np.minimum(p, p.max() * LOST)) @ ch[see] / l
            reach = p @ ch[see] / l
            sums = 2 * d + (see.sum() + 16) * 2.0 ** -24
            tol[i, h] = (unit * np.abs(out[i, h]) + (lost + reach * sums) * (1 + unit)
                         + (2.0 ** -25 if unit == ref.UNIT["f16"] else 0))
            ltol[i, h] = d + (see.sum() + 16) * 2.0 ** -24 + abs(lse[i, h]) * 2.0 ** -22
    return out, lse, tol, ltol

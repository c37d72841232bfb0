"""float64 restatement of rotary positions, for the tests."""
from fractions import Fraction

import numpy as np

PER_TURN = Fraction(0x28BE60DB9391054A7F09D5F47D4D3770, 1 << 128)  # 1 / (2 pi)
# unit roundoff of the types
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def angles(freq, pos):
    """[len(pos), len(freq)] angles in (-pi, pi], the product exact modulo a turn."""
    out = np.zeros((len(pos), len(freq)))
    for j, f in enumerate(freq):
        t = Fraction(float(f)) * PER_TURN
        for i, p in enumerate(pos):
            x = int(p) * t % 1
            out[i, j] = float(x - 1 if x > Fraction(1, 2) else x) * 2 * np.pi
    return out


def turn(x, pos, freq, rot, interleaved, amp=1.0, inverse=False, unit=0.0):
    """x [T, h, D] float64, and the bound of the error: sines and cosines are within 3 2^-24
    (two roundings of an argument of at most pi / 4, and of the last step of the series), two products
    with the amplitude and the sum add three roundings of float32, the result one of its
    type."""
    a = angles(freq, pos)[:, None, :]
    c, s = np.cos(a) * amp, np.sin(a) * amp
    if inverse:
        s = -s
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else \
        (slice(0, rot // 2), slice(rot // 2, rot))
    y, tol = x.copy(), np.zeros_like(x)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    big = (np.abs(x[..., lo]) + np.abs(x[..., hi])) * abs(amp) * 6 * 2.0 ** -24
    tol[..., lo] = tol[..., hi] = big
    tol[..., :rot] += unit * np.abs(y[..., :rot]) * (1 + 2.0 ** -10)
    if unit == UNIT["f16"]:
        tol[..., :rot] += 2.0 ** -25
    return y, tol

"""Angles and turned rows to the last bits of 64: what keys for an 8-bit cache are held to."""
from fractions import Fraction

import numpy as np

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")


def parts_of_two_pi():
    """2 pi as a sum of two numbers of 30 bits, whose products with whole numbers below 2^34 are exact in 64, and the rest."""
    parts, rest = [], 2 * PI
    for shift in (27, 57):
        p = Fraction(int(rest * 2 ** shift), 2 ** shift)
        parts.append(np.longdouble(p.numerator) / np.longdouble(p.denominator))
        rest -= p
    return parts + [np.longdouble(float(rest))]


def angles(positions, inv_freq):
    """positions * inv_freq less whole turns, in [-pi, pi] and fp64: the product of 31 and 24 bits and the turns below 2^33 are exact before."""
    assert np.finfo(np.longdouble).nmant >= 63
    a = positions.astype(np.longdouble)[:, None] * inv_freq.astype(np.longdouble)[None]
    assert abs(a).max() < 2.0 ** 33
    a1, a2, a3 = parts_of_two_pi()
    turns = np.rint(a / (a1 + a2))
    return (((a - turns * a1) - turns * a2) - turns * a3).astype(np.float64)


def turned(x, positions, inv_freq, scale):
    """Heads x [T, H, D] in 64 bits, all of D turned."""
    a = angles(positions, inv_freq)[:, None]
    h = x.shape[-1] // 2
    u, v = x[..., :h], x[..., h:]
    # in extended precision, rounded to 64 bits at the end
    c, s, scale = (np.asarray(t).astype(np.longdouble) for t in (np.cos(a), np.sin(a), np.float32(scale)))
    u, v = u.astype(np.longdouble), v.astype(np.longdouble)
    return np.concatenate([scale * (u * c - v * s), scale * (v * c + u * s)], -1).astype(np.float64)

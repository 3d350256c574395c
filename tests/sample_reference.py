"""Drawing a token a row in plain Python: weights from 80-bit exponentials rounded to whole multiples of 2^-bits, everything
after that in whole numbers of any size."""
from __future__ import annotations

from fractions import Fraction

import numpy as np


def bits_of(vocab):
    return min(50, 62 - (vocab - 1).bit_length())


def kept_weights(l, t=1.0, k=0, p=1.0, least=0.0):
    """{token: whole weight} of what a row's settings leave, or None where it has no token."""
    l = np.asarray(l, np.float64)
    tokens = np.flatnonzero(l > -np.inf)
    if len(tokens) == 0:
        return None
    order = tokens[np.argsort(-l[tokens], kind="stable")]
    if t == 0:
        return {int(order[0]): 1}
    top = l[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(l[order] == top, 0.0, np.where(np.isinf(top), -np.inf, l[order] - top)).astype(np.longdouble)
        ratio = np.exp(np.where(d == 0, 0, d / np.longdouble(t)))
    weight = [int(v) for v in np.rint(ratio * np.longdouble(2.0) ** bits_of(len(l)))]
    count = len(order) if k <= 0 else min(int(k), len(order))
    whole = sum(weight[:count])
    kept, before = {}, 0
    for i in range(count):
        if i and p < 1 and not Fraction(before) < Fraction(float(p)) * whole:
            break
        if i == 0 or ratio[i] >= np.longdouble(float(least)):
            kept[int(order[i])] = weight[i]
        before += weight[i]
    return kept


def draw(l, u, **settings):
    """(token, its share) of a row."""
    kept = kept_weights(l, **settings)
    if kept is None:
        return -1, 0.0
    total = sum(kept.values())
    target, run = Fraction(float(u)) * total, 0
    for i in sorted(kept):
        run += kept[i]
        if run > target:
            return i, float(Fraction(kept[i], total))
    raise AssertionError("u is below 1")

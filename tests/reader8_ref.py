"""Caches of 8 bits restated in 64 bits (numpy): e4m3 values, a head's exponent, and what a slot stands for.

Bounds: a stored element is off by at most half of e4m3's step there: 2^-4 of itself, or 2^-10 of its head's unit 2^e where it
is under 2^-6 of that; where the kernel's turned value is off by `err` before it is rounded, by that besides, and the step is that
of the larger of both.
"""
from __future__ import annotations

import numpy as np

LEAST = {"float16": -15, "bfloat16": -117}


def _table():
    b = np.arange(256)
    s, e, m = np.where(b >> 7, -1.0, 1.0), (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0)) * s
    v[(b & 0x7F) == 0x7F] = np.nan
    return v


VALUES = _table()
_POSITIVE = VALUES[:127]                     # 0 .. 448, rising


def to_e4m3(y):
    """The byte nearest to y (|y| <= 448), ties to the even one; NaN and infinities to NaN."""
    y = np.asarray(y, np.float64)
    a = np.where(np.isfinite(y), np.abs(y), 0)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POSITIVE[lo], _POSITIVE[hi] - a
    b = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    b = np.where(np.isfinite(y), b, 0x7F)
    return (b | (np.signbit(y) & np.isfinite(y)) * 0x80).astype(np.uint8)


def exponent(x, dtype):
    """The byte of each head of x (..., D): the least k + 127 with max |x| <= 448 2^k, at least the type's."""
    top = np.max(np.where(np.isfinite(x), np.abs(x), 0), axis=-1)
    k = np.full(top.shape, LEAST[dtype], np.int64)
    pos = top > 0
    g = np.ceil(np.log2(np.where(pos, top, 1) / 448.0)).astype(np.int64)
    g = np.where(448.0 * 2.0 ** (g - 1.0) >= top, g - 1, np.where(448.0 * 2.0 ** g.astype(np.float64) < top, g + 1, g))
    return (np.where(pos, np.maximum(k, g), k) + 127).astype(np.uint8)


MOST = {"float16": 61440.0, "bfloat16": 240.0 * 2.0 ** 120}       # the largest that is held: a finite value of the type


def limited(x, dtype):
    return np.where(np.isfinite(x), np.clip(x, -MOST[dtype], MOST[dtype]), x)


def hold(x, dtype):
    """x (..., D) -> e4m3 bytes, exponent bytes."""
    x = limited(x, dtype)
    e = exponent(x, dtype)
    return to_e4m3(x * 2.0 ** (127.0 - e.astype(np.float64))[..., None]), e


def held(b, e):
    """What bytes b under exponent bytes e (broadcast) stand for."""
    return VALUES[b] * np.where(e == 255, np.nan, 2.0 ** (e.astype(np.float64) - 127))


def pages_held(k, v, ks, vs):
    """64-bit pages of a cache: k (N, H, P, D), v (N, H, D, P), exponents (N, H, P)."""
    return held(k, ks[..., None]), held(v, vs[:, :, None])


def half_step(x, e, err=0.0):
    """Half of e4m3's step at x (..., D) under exponent bytes e (...), for values off by up to err."""
    unit = 2.0 ** (e.astype(np.float64) - 127)[..., None]
    y = (np.abs(x) + err) / unit
    return 0.5 * 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3) * unit

"""Rows of a 4-bit (MXFP4) cache as numpy sees them."""
from __future__ import annotations

import numpy as np

MXFP4 = 39
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def stored4(x: np.ndarray) -> np.ndarray:
    """f32 rows [..][1024] as the values that their 4-bit blocks stand for (NaN where the block has an infinity or NaN).

    A block is 32 values.  Its scale is the smallest power of two of which the largest value has at most 7, within
    2^-125 .. 2^125; a value is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 scales, halfway to the one of the even code, and 6
    above."""
    b = np.ascontiguousarray(x, np.float32).astype(np.float64).reshape(-1, 32)
    bad = ~np.isfinite(b).all(-1)
    b[bad] = 0.0
    big = np.abs(b).max(-1)
    f, e = np.frexp(big)  # big = f 2^e, f in [1/2, 1): at most 7 of 2^(e - 3) where f <= 7/8
    e = np.clip(np.where(big == 0, -125, e - 3 + (f > 0.875)), -125, 125)
    a = np.ldexp(np.abs(b), -e[:, None])
    code = np.searchsorted((LEVELS[1:] + LEVELS[:-1]) / 2, a)  # a level's upper half-way point is its own: right for the even codes
    tie = np.isin(a, (LEVELS[1:] + LEVELS[:-1]) / 2)
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    out = np.copysign(np.ldexp(LEVELS[code], e[:, None]), b)
    out[bad] = np.nan
    return out.astype(np.float32).reshape(np.shape(x))

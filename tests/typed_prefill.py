"""What a prompt piece's attention over typed rows is held to as a whole, and a
CPU form of its arithmetic."""
from __future__ import annotations

import numpy as np
from typed_rows import BF16, stored

# N(0, 1) queries, keys and values.  An operand x is kept as bf16 parts hi + lo, so
# a product loses lo * lo and each operand's rest.  A rounding's error is even
# over half a step, 2^-8 of the power of two below x: 0.42 2^-8 of x in the root mean
# square (1/sqrt(3), over the mantissa's size).  So lo * lo is 0.18 2^-16 of the
# product and a rest, lo's own rounding, 0.21 2^-16 of it at most.  In a score, a
# sum of 256 products of standard deviation 1/16, they add to sqrt(0.18^2 + 2 0.21^2)
# 2^-16 = 5.3e-6 of 1, and 32-bit sums 2.4e-6 as in typed_rows.NORMAL_TOL.  A
# weight's upper part is cut off, not rounded: its lower part is twice as large, and
# weight times value loses sqrt(0.36^2 + 0.36^2 + 0.21^2) 2^-16 = 8.4e-6.  An output, a sum of
# independent values, is off by the root of these squares' sum, 1.02e-5 of its 2-norm.
# Held to 1.6 times that: a head's scores may be spread a half wider than 1.
PREFILL_TOL = 1.6e-5


def parts(x: np.ndarray):
    """x as bf16 hi and lo, both as f32 values."""
    hi = stored(x, BF16)
    return hi, stored(x - hi, BF16)


def prefill_token(q, k, v, gate=None, lose=()):
    """One token's attention from bf16 parts with 32-bit sums; `lose` names parts that are left out ("q", "k", "p" or "v")."""
    f = np.float32
    out = np.empty((24, 256), f)

    def product(a, b, lost_a, lost_b):
        (ah, al), (bh, bl) = parts(a), parts(b)
        al, bl = al * f(not lost_a), bl * f(not lost_b)
        return (ah @ bh + (ah @ bl + al @ bh)).astype(f)

    for h in range(24):
        at = slice(256 * (h // 6), 256 * (h // 6) + 256)
        s = product(k[:, at], (q[h] * f(0.09016844)).astype(f), "k" in lose, "q" in lose)
        w = np.exp2(s - s.max()).astype(f)
        out[h] = product(w, v[:, at], "p" in lose, "v" in lose) / w.sum(dtype=f)
    if gate is not None:
        out = out / (f(1) + np.exp(-gate.reshape(24, 256)))
    return out.astype(f)

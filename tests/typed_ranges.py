"""Inputs of the typed cache's attention whose values differ by many orders,
and what their outputs are held to.

A row of large values may have little weight or none, and a row of small ones
nearly all of it: what a row adds is its weight times its values, and an error
is measured by what is added, not by the largest value in the cache.
"""
from __future__ import annotations

import numpy as np
from typed_rows import BF16, F16, NORMAL_TOL, Q8_K, off_by, stored

U = 2.0 ** -24


def attend_by_weight(q, k, v, ty):
    """typed_rows.attend with what small weights lose counted by what their rows add.

    A weight in bf16 parts has f32's exponents: nothing is lost before the
    parts are subnormal, 2^-125 of the largest.  In f16 parts, the lower one
    2^11 times as large, a weight is off by half of f16's smallest step over 2^11 --
    2^-36 of its unit -- where its parts are no longer normal: for F16 rows the
    largest weight of a chain is 2^7 units at least, so 2^-43 of the largest
    weight times the value; for Q8_K rows the largest weight times scale of a
    chain is 2^6 units at least, so 2^-42 of that times a quant, 127 at most:
    2^-42 of the largest weighted value.  Twice that for the joins."""
    n = k.shape[0]
    out, bound = np.empty((24, 256)), np.empty((24, 256))
    q, k, v = q.reshape(24, 256).astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    for h in range(24):
        kk, vv = k[:, 256 * (h // 6):256 * (h // 6) + 256], v[:, 256 * (h // 6):256 * (h // 6) + 256]
        s = kk @ q[h] / 16.0
        # a score's error by its own size, a weight's by its own score
        size = np.abs(kk) @ np.abs(q[h]) / 16.0
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vv
        top = float(((264 * size + np.abs(s)) * p).sum())  # the denominator's, by weight
        e = (264 * size + np.abs(s) + top + 8 + n + 16) * U + 2.0 ** -21
        least = {BF16: 2.0 ** -125 * np.abs(vv).max(), F16: 2.0 ** -42 * p.max() * np.abs(vv).max(),
                 Q8_K: 2.0 ** -41 * (p * np.abs(vv).max(1)).max()}[ty]
        bound[h] = (e * p) @ np.abs(vv) * 1.01 + n * least + 1e-44
    return out, bound


def check(got, want, bound, tol, heads=slice(None)):
    """Each value within its bound, and each kv head's outputs together within tol."""
    got, want = got.reshape(24, 256)[heads], want[heads]
    off = np.abs(got.astype(np.float64) - want)
    worst, norm = float((off / bound[heads]).max()), max(off_by(g, w) for g, w in zip(got, want))
    print(f"[bound] {worst:.3f} of the bound, 2-norm {norm:.2e} of {tol:.2e}", flush=True)
    assert np.all(np.isfinite(got)) and worst <= 1.0 and norm <= tol


def _normal(seed, P):
    rng = np.random.default_rng(seed)
    K, V = (rng.standard_normal((P, 1024)).astype(np.float32) for _ in range(2))
    Q = rng.standard_normal((24, 256)).astype(np.float32)
    # each head's first dim steers a row's score and no other's
    K[:, ::256] = 0.0
    Q[:, 0] = 8.0
    return rng, Q, K, V


def no_weight(seed, ratio, at, P=400):
    """One row of values `ratio` times as large, whose weight is e^-150 or so: nothing."""
    _, Q, K, V = _normal(seed, P)
    K[at, ::256] = -300.0
    V[at] *= np.float32(ratio)
    return Q, K, V, NORMAL_TOL


def little_weight(seed, low, high, base, P=400):
    """24 rows of low .. high binades less weight and as many more in size: each adds
    what the others do.  Their scores reach s = high log 2: 256 roundings of
    standard deviation s u / sqrt(3) at most off, in some sqrt(24 / 400) = 0.25 of
    the output; held to twice that besides N(0, 1)'s."""
    rng, Q, K, V = _normal(seed, P)
    t, b = rng.permutation(P)[:24], rng.uniform(low, high, 24)
    K[t, ::256] = (-2.0 * np.log(2.0) * b).astype(np.float32)[:, None]
    V[t] *= (2.0 ** b).astype(np.float32)[:, None]
    return Q, K, (V * np.float32(base)).astype(np.float32), NORMAL_TOL + 2 * 0.25 * 16 / np.sqrt(3) * high * np.log(2.0) * U


def one_heads_row(seed, ratio, at, P=400):
    """A row that takes all of every other head, and nothing of the rest."""
    _, Q, K, V = _normal(seed, P)
    Q[::2, 0] = -8.0
    K[at, ::256] = -300.0
    V[at] *= np.float32(ratio)
    return Q, K, V, NORMAL_TOL


def slope(seed, binades, base, rising, P=700):
    """Scores that rise (or fall) by `binades` over the rows, values that do the
    opposite: every row adds as much.  Scores reach s = binades log 2, off by 16 s u /
    sqrt(3); held to twice that besides N(0, 1)'s."""
    _, Q, K, V = _normal(seed, P)
    b = np.linspace(0.0, binades, P) if rising else np.linspace(binades, 0.0, P)
    K[:, ::256] = (2.0 * np.log(2.0) * b).astype(np.float32)[:, None]
    V *= (base * 2.0 ** -b).astype(np.float32)[:, None]
    return Q, K, V, NORMAL_TOL + 2 * 16 / np.sqrt(3) * binades * np.log(2.0) * U


# (type, name, arguments after the seed)
CASES = [(ty, "no_weight", (r, at)) for ty in ("q8_k", "bf16") for r, at in
         ((1e3, 399), (1e4, 7), (1e5, 200), (1e6, 0), (1e8, 37), (1e10, 350), (1e20, 100))]
CASES += [("f16", "no_weight", (1e4, 0)), ("f16", "no_weight", (1e4, 250))]
CASES += [(ty, "little_weight", (16, 26, 2.0 ** -12)) for ty in ("f16", "bf16", "q8_k")]
CASES += [(ty, "little_weight", a) for ty in ("bf16", "q8_k") for a in ((10, 40, 1.0), (30, 100, 1.0))]
CASES += [("f16", "one_heads_row", (1e4, 50))] + [(ty, "one_heads_row", (r, at)) for ty in ("bf16", "q8_k")
                                                  for r, at in ((1e8, 0), (1e8, 399), (1e25, 160), (1e-8, 30))]
CASES += [("f16", "slope", (24, 2.0 ** 10, up)) for up in (True, False)]
CASES += [(ty, "slope", (b, base, up)) for ty in ("bf16", "q8_k") for up in (True, False)
          for b, base in ((60, 1.0), (110, 1.0), (110, 2.0 ** 100))]
IDS = ["-".join([ty, name] + [str(a) for a in args]) for ty, name, args in CASES]
IDENT = {"f16": F16, "bf16": BF16, "q8_k": Q8_K}


def case(ty, name, args):
    Q, K, V, tol = globals()[name](len(str(args)) + len(name), *args)
    ident = IDENT[ty]
    return Q, K, V, stored(K, ident), stored(V, ident), tol


def heads_of(name):
    """The heads that a case's 2-norm limit is about: the others' one row is their value itself."""
    return slice(1, None, 2) if name == "one_heads_row" else slice(None)

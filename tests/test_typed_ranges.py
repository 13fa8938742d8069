"""The references of values of very different sizes, on the CPU: plain 32-bit
arithmetic stays within their limits, and weights that lose their small parts do
not."""
import numpy as np
import pytest
from typed_ranges import CASES, IDENT, IDS, attend_by_weight, case, check, heads_of


def _attend32(q, k, v, weights):
    """32-bit attention, 16 tokens at a time; weights(w, values) gives what each row is taken by."""
    f = np.float32
    out = np.empty((24, 256), f)
    for h in range(24):
        kk, vv = k[:, 256 * (h // 6):256 * (h // 6) + 256], v[:, 256 * (h // 6):256 * (h // 6) + 256]
        s = (kk @ q[h]) * f(0.0625)
        w = np.exp(s - s.max())
        p = weights(w, vv)
        total = np.zeros(256, f)
        for t in range(0, len(w), 16):
            total += p[t:t + 16] @ vv[t:t + 16]
        out[h] = total / w.sum(dtype=f)
    return out


def _whole(w, vv):
    return w


def _by_largest_scale(w, vv):
    """Two f16 parts of weight times scale over the largest scale's power of two."""
    scale = np.abs(vv).max(1) / np.float32(127.0)
    unit = np.exp2(np.ceil(np.log2(scale.max()))).astype(np.float32)
    x = w * np.float32(2.0 ** 7) * (scale / unit)
    hi = x.astype(np.float16).astype(np.float32)
    lo = (x - hi).astype(np.float16).astype(np.float32)
    return np.where(scale > 0, (hi + lo) / np.float32(2.0 ** 7) * (unit / np.where(scale > 0, scale, 1)), 0).astype(np.float32)


def _plain_f16_parts(w, vv):
    x = w * np.float32(2.0 ** 7)
    hi = x.astype(np.float16).astype(np.float32)
    return (hi + (x - hi).astype(np.float16).astype(np.float32)) / np.float32(2.0 ** 7)


@pytest.mark.parametrize("ty,name,args", CASES, ids=IDS)
def test_plain_arithmetic_holds(ty, name, args):
    Q, _, _, k, v, tol = case(ty, name, args)
    want, bound = attend_by_weight(Q, k, v, IDENT[ty])
    got = _attend32(Q, k, v, _whole)
    check(got, want, bound, tol, heads_of(name))


@pytest.mark.parametrize("ty,name,args,lose", [
    ("q8_k", "no_weight", (1e5, 200), _by_largest_scale), ("q8_k", "no_weight", (1e8, 37), _by_largest_scale),
    ("q8_k", "little_weight", (10, 40, 1.0), _by_largest_scale), ("q8_k", "one_heads_row", (1e8, 399), _by_largest_scale),
    ("q8_k", "slope", (60, 1.0, True), _by_largest_scale), ("f16", "little_weight", (16, 26, 2.0 ** -12), _plain_f16_parts)])
def test_lost_parts_are_noticed(ty, name, args, lose):
    Q, _, _, k, v, tol = case(ty, name, args)
    want, bound = attend_by_weight(Q, k, v, IDENT[ty])
    with pytest.raises(AssertionError):
        check(_attend32(Q, k, v, lose), want, bound, tol, heads_of(name))

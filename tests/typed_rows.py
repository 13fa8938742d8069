"""Plain references of the typed cache's rows and attention, in numpy and
64-bit arithmetic, and the bounds that its tests hold the kernels to."""
from __future__ import annotations

import numpy as np

F32, F16, Q8_K, BF16 = 0, 1, 15, 30
TYPES = {"f16": F16, "bf16": BF16, "q8_k": Q8_K}


def stored(x: np.ndarray, ty: int) -> np.ndarray:
    """f32 rows [..][1024] as the values that a cache of the type holds."""
    x = np.ascontiguousarray(x, np.float32)
    if ty == F32:
        return x.copy()
    if ty == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    if ty == BF16:
        # to the nearest multiple of the upper 16 bits' step, ties to the even one (finite values)
        b = x.view(np.uint32).astype(np.uint64)
        b = (b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000
        return b.astype(np.uint32).view(np.float32)
    b = x.reshape(-1, 256)
    m = np.take_along_axis(b, np.abs(b).argmax(-1)[:, None], -1)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inverse = np.float32(-127.0) / m
        # whole numbers: a quant of zero has no sign of its own
        q = np.nan_to_num(np.minimum(np.rint(inverse * b), np.float32(127.0))).astype(np.int32).astype(np.float32)
        scale = np.float32(1.0) / inverse
        # a size under 127 / 3.4e38 has no finite inverse scale: its scale is 0, whatever the quants
        q = np.where(np.isinf(inverse), np.float32(0.0), q)
    return np.where(m == 0, np.float32(0.0), q * scale).astype(np.float32).reshape(x.shape)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, gate=None):
    """One token's attention in 64 bits: q [24][256], k and v [n][1024] the
    stored values.  Returns the output [24][256] and a bound on what a kernel
    that keeps its sums, softmax statistics and products in 32 bits may be off.

    u = 2^-24.  A score is a sum of 256 products, formed from q split into
    parts that carry 22 bits or more: it is off by at most (256 + 8) u S in any
    order, S = sum |q k| / 16 (the split's 2^-22 on each term counted in the 8;
    scaling to base 2 and back two roundings more).  A weight is then off by a
    factor exp(+-e), e the largest such error plus 4 u for exp2 and its
    argument's rounding, |s| u; numerator and denominator each by e, and by
    (n + 16) u for their sums and the splits' rescalings; a weight's parts
    carry 2^-21 of it or better while they are normal halves.  Below those, a
    part is rounded to whole steps of 2^-24 (half of one off), and the largest
    weight of a chain is 2^7 at least (its reference lies at most 7 under its
    largest score): each weight is off by 2^-32 of the largest at most,
    whatever its own size, times its value -- for 8-bit rows, whose weight
    carries the value's scale over a power of two of up to twice the largest
    scale, times up to twice the largest value.  A term n 2^-31 pmax vmax
    covers both.  The gate's sigmoid 8 u."""
    u = 2.0 ** -24
    n = k.shape[0]
    out, bound = np.empty((24, 256)), np.empty((24, 256))
    q, k, v = q.reshape(24, 256).astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    for h in range(24):
        kk, vv = k[:, 256 * (h // 6):256 * (h // 6) + 256], v[:, 256 * (h // 6):256 * (h // 6) + 256]
        s = kk @ q[h] / 16.0
        big = float((np.abs(kk) @ np.abs(q[h])).max()) / 16.0
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vv
        e = 2.0 * ((264 * big + 4 + float(np.abs(s).max())) * u) + (n + 16) * u + 2.0 ** -21
        bound[h] = e * (p @ np.abs(vv)) * 1.01 + n * 2.0 ** -31 * p.max() * np.abs(vv).max() + 1e-37
    if gate is not None:
        sig = 1.0 / (1.0 + np.exp(-gate.reshape(24, 256).astype(np.float64)))
        out, bound = out * sig, bound * sig + 8 * u * np.abs(out * sig)
    return out, bound


def rope64(x: np.ndarray, positions) -> np.ndarray:
    """Rows [n][heads][256] in 64 bits, pairs (p, p + 32) turned by the model's f32 angles."""
    scale = np.float32(np.float32(10000000.0) ** np.float32(-2.0 / 64.0))
    theta, cols = np.array(positions, np.float32), []
    for _ in range(32):
        cols.append(theta.astype(np.float64))
        theta = (theta * scale).astype(np.float32)
    t = np.stack(cols, 1)[:, None, :]
    x = x.astype(np.float64)
    a, b = x[..., :32], x[..., 32:64]
    return np.concatenate((a * np.cos(t) - b * np.sin(t), a * np.sin(t) + b * np.cos(t), x[..., 64:]), -1)


def rms64(x: np.ndarray, w: np.ndarray) -> np.ndarray:
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w.astype(np.float64)


def off_by(got: np.ndarray, want: np.ndarray) -> float:
    """The 2-norm of the error over the result's."""
    d = got.reshape(-1).astype(np.float64) - want.reshape(-1)
    return float(np.linalg.norm(d) / np.linalg.norm(want))


# For N(0, 1) queries, keys and values the roundings add as random steps: a
# score is a sum of 256 products of standard deviation 1/16, its partial sums
# at most about 3 in size, so its 256 roundings of standard deviation 3 u /
# sqrt(3) at most give 28 u; q's, the weights' and the exponential's own few
# roundings 4 u more; sums over tokens, split into chains of some hundreds,
# as much again.  An output is a weighted sum of independent values, off by
# the root mean square of its weights' errors, 40 u = 2.4e-6 in all: held to
# twice that.
NORMAL_TOL = 80 * 2.0 ** -24

"""What q38_attn_observe keeps of a query: all of its bits whatever the number of
queries, and 16 of them over bf16 operands where the caller asks for two parts."""
import numpy as np
import pytest
from test_gpu_weights import Cache, U, typed
from typed_rows import BF16, stored

pytestmark = pytest.mark.gpu

LOG2 = np.float32(0.09016844005556021)  # 1 / 16 in units of log2
ONES = 8


def _queries(rng, n):
    """One dim of each head, the others 0: sizes near 960 whose products with LOG2 are a good half of 2^-18 of themselves more
    than the two bf16 values nearest to them and to the rest."""
    x = rng.uniform(930, 990, 200000).astype(np.float32)
    y = x * LOG2
    rest = y - stored(y, BF16)
    rest -= stored(rest, BF16)
    x = x[rest > 0.6 * 2.0 ** -18 * y][:24 * n]
    q = np.zeros((n, 24, 256), np.float32)
    q[:, :, 0] = x.reshape(n, 24)
    return q


def _sums(pkg, ctx, ty, P, Q):
    """Eight tokens of one key and P - 8 of another: scores of about 60 and of 0."""
    n = len(Q)
    K = np.zeros((P, 1024), np.float32)
    K[:ONES, ::256] = 1.0
    with Cache(pkg, ctx, ty, [P]) as c:
        c.kv.write(3, c.seqs[0], 0, P, ctx.array(K), ctx.array(K))
        c.kv.attn_observe(3, c.seqs[0], P - n, n, ctx.array(Q))
        got = c.weights(c.seqs[0], P)[0].astype(np.float64)
    want = np.zeros((P, 4))
    for u in range(n):
        # in 64 bits: the other tokens' e^-s each beside the eight
        end, low = P - n + u + 1, np.exp(-Q[u, :, 0].astype(np.float64) / 16.0)
        w = 1.0 / (ONES + (end - ONES) * low)
        want[:ONES] += w.reshape(4, 6).sum(1)
        want[ONES:end] += (w * low).reshape(4, 6).sum(1)
    return np.abs(got - want) / want


# A score is one product.  Its query times LOG2 is off by 2 u (the constant, the product); the three parts' sum is that
# number, and its difference from the reference, which is the same number or 0, is exact.  So a weight is off by 2 u S / 2^0 of
# itself, S = 62 its size in units of e, twice over for both scores of a difference; 8 u for the exponential, 24 u for the
# denominator (eight equal terms; the others, 2^-86 of it, leave it as it is) and its reciprocal, and the sum over 6 heads of n
# queries adds 7 n roundings.  What two parts leave is 0.6 2^-18 S = 1.4e-4 of a weight at least, all of one sign.
def _tol(n):
    return (4 * 62 + 32 + 7 * n) * U


@typed
@pytest.mark.parametrize("P,n", [(40, 1), (40, 16), (40, 17), (41, 33), (24593, 16), (24593, 17)])
def test_every_number_of_queries_keeps_their_bits(pkg, ctx, ty, P, n):
    Q = _queries(np.random.default_rng(n), n)
    off = _sums(pkg, ctx, ty, P, Q)
    print(f"[bound] {off.max() / _tol(n):.3f} of the bound", flush=True)
    # F16 and Q8_K rows: two parts of 11 bits, the lower one's own rounding 2^-22 of the query
    assert off.max() <= _tol(n) + (0.0 if ty in ("bf16", "mxfp4") else 2.0 ** -21 * 62)


@typed
@pytest.mark.parametrize("P,n", [(40, 1), (40, 17), (24593, 17)])
def test_two_parts_where_the_caller_asks(pkg, ctx, ty, P, n):
    Q = _queries(np.random.default_rng(n), n)
    whole = _sums(pkg, ctx, ty, P, Q)
    ctx.set_observe_parts(2)
    try:
        off = _sums(pkg, ctx, ty, P, Q)
    finally:
        ctx.set_observe_parts(3)
    if ty in ("bf16", "mxfp4"):
        # each part rounded to nearest, off by 2^-8 of what it stands for at most
        assert 1e-4 < off.max() <= _tol(n) + 2.0 ** -16 * 62
    else:
        assert np.array_equal(off, whole)
    assert np.array_equal(_sums(pkg, ctx, ty, P, Q), whole)


def test_parts_are_two_or_three(pkg, ctx):
    for parts in (-1, 0, 1, 4):
        with pytest.raises(pkg.Q38Error, match="2 or 3"):
            ctx.set_observe_parts(parts)

"""A prompt's queries observed where scores are far from zero: the sums against
64-bit arithmetic on the values that the stored rows stand for."""
import numpy as np
import pytest
from parity import decode_split
from test_gpu_weights import DECODE, OBSERVE, Cache, U, _held, _q, _rows, stored, typed, weights_of
from typed_rows import attend

pytestmark = pytest.mark.gpu

CASES = ["low", "low_rising", "low_falling", "rising", "falling", "peaked", "large", "tiny", "flat", "huge_q", "mixed_heads"]
#: a context whose scores are kept, one page of whose tokens a wave looks at, and one whose scores are formed twice
SHORT, LONG = 700, 24593


def _case(case, ty, P, n):
    """Rows and queries whose scores (q k / 16) lie at -300 (low), run from -400 to 0 and back, or up to 175 and back, spread
    over hundreds, or come from queries near the ends of the f32 range of sizes."""
    rng = np.random.default_rng(len(case) + P)
    K, Q = _rows(rng, P), _q(rng, n)
    unit = np.zeros(1024, np.float32)
    unit[::256] = 4.0
    ramp = np.linspace(0, 175, P, dtype=np.float32)[:, None]
    if case.startswith("low"):
        Q[:, :, 0] = -4.0
        by = 300.0 if case == "low" else ramp[::-1] * (16 / 7) if case == "low_rising" else ramp * (16 / 7)
        K += by * unit
    elif case in ("rising", "falling"):
        Q[:, :, 0] = 4.0
        K += (ramp if case == "rising" else ramp[::-1]) * unit
    elif case == "peaked":
        Q[:, :, 0] = 10.0
        K[P // 2] += 20 * unit
    elif case == "large":
        Q *= 50
    elif case == "tiny":
        Q *= 1e-12
    elif case == "flat":
        K[:] = K[0]
    elif case == "huge_q" and ty != "f16":
        Q *= 1e18
        K *= 1e-18
    elif case == "mixed_heads":
        Q *= (10.0 ** rng.uniform(-6, 1, (n, 24, 1))).astype(np.float32)
    return K, Q


def _observed(pkg, ctx, ty, K, Q):
    P, n = len(K), len(Q)
    with Cache(pkg, ctx, ty, [P]) as c:
        c.kv.write(3, c.seqs[0], 0, P, ctx.array(K), ctx.array(K))
        c.kv.attn_observe(3, c.seqs[0], P - n, n, ctx.array(Q))
        return c.weights(c.seqs[0], P)[0]


def _want(ty, K, Q, query):
    """The sums in 64 bits, and their bound: weights_of's of every query (1.05 times: exp(e) - 1 for errors e up to 0.09 of
    a score, where weights_of counts e), and the order of the additions."""
    P, n = len(K), len(Q)
    k = stored(K, ty)
    want, bound = np.zeros((P, 4)), np.zeros((P, 4))
    for u in range(n):
        w, e = weights_of(Q[u], k[:P - n + u + 1], query)
        want[:P - n + u + 1] += w
        bound[:P - n + u + 1] += 1.05 * e
    return want, bound + 7 * n * U * want


@typed
@pytest.mark.parametrize("P,n,case", [(SHORT, n, case) for n in (3, 20) for case in CASES] +
                         [(LONG, 2, case) for case in ("low", "low_rising", "low_falling", "falling", "large")])
def test_observe_score_ranges(pkg, ctx, ty, P, n, case):
    """Finite rows and queries leave finite sums, wherever their scores lie."""
    K, Q = _case(case, ty, P, n)
    want, bound = _want(ty, K, Q, OBSERVE[ty])
    _held(_observed(pkg, ctx, ty, K, Q), want, bound)


@typed
@pytest.mark.parametrize("case", CASES)
def test_decode_sums_score_ranges(pkg, ctx, ty, case):
    """The same of decode calls, in one split, in two and in many."""
    K, Q = _case(case, ty, SHORT, 1)
    want, bound = _want(ty, K, Q, DECODE)
    with Cache(pkg, ctx, ty, [SHORT]) as c:
        c.kv.write(3, c.seqs[0], 0, SHORT, ctx.array(K), ctx.array(K))
        for split in (4096, 352, 16):
            c.kv.weights_put(3, c.seqs, [0], [SHORT])
            with decode_split(ctx, split):
                c.kv.attn_decode(3, c.seqs, [SHORT - 1], ctx.array(Q), ctx.empty((24, 256)))
            _held(c.weights(c.seqs[0], SHORT)[0], want, bound)


@typed
def test_first_look_at_very_low_scores(pkg, ctx, ty):
    """One token and a few, all of whose scores lie below -128 in units of log2: the smallest powers there are."""
    for P in (1, 3, 5, 17):
        for low in (-88.0, -89.0, -200.0, -5000.0):
            K, Q = np.zeros((P, 1024), np.float32), np.zeros((1, 24, 256), np.float32)
            K[:, ::256] = 16.0
            Q[:, :, 0] = low
            # equal scores: six heads' weights of 1 / P
            got = _observed(pkg, ctx, ty, K, Q)
            assert np.all(np.abs(got.astype(np.float64) - 6.0 / P) <= 6.0 / P * (P + 40) * U), (P, low, got)


def _far_sizes(case, P, n):
    """Scores of ordinary size from queries near an end of the f32 range: their powers of two and the rows' scales, multiplied
    in one order or another, need not be within it."""
    rng = np.random.default_rng(P + n)
    K, Q = _rows(rng, P), rng.uniform(-2e38, 2e38, (n, 24, 256)).astype(np.float32)
    if case == "small_keys":
        return K * np.float32(1e-36), Q  # scores of some hundred
    # large keys, but where the queries are; or the other way round
    K *= 1e7
    K[:, ::256] = 0.0
    Q[:, :, 1:] = 0.0
    if case == "small_queries":
        K[:, ::256] = 1e38 * np.sign(rng.standard_normal((P, 4)))
        Q[:, :, 0] = rng.uniform(-1e-37, 1e-37, (n, 24))
    return K, Q


far_sizes = pytest.mark.parametrize("case", ["zero_products", "small_keys", "small_queries"])


@far_sizes
@pytest.mark.parametrize("P,n", [(SHORT, 3), (LONG, 2)])
def test_observe_queries_and_scales_of_far_sizes(pkg, ctx, case, P, n):
    K, Q = _far_sizes(case, P, n)
    want, bound = _want("q8_k", K, Q, OBSERVE["q8_k"])
    _held(_observed(pkg, ctx, "q8_k", K, Q), want, bound)


@far_sizes
def test_decode_queries_and_scales_of_far_sizes(pkg, ctx, case):
    """Outputs and sums of a decode call."""
    K, Q = _far_sizes(case, SHORT, 1)
    V = _rows(np.random.default_rng(1), SHORT)
    want, bound = _want("q8_k", K, Q, DECODE)
    out, off = attend(Q[0], stored(K, "q8_k"), stored(V, "q8_k"))
    with Cache(pkg, ctx, "q8_k", [SHORT]) as c:
        c.kv.write(3, c.seqs[0], 0, SHORT, ctx.array(K), ctx.array(V))
        o = ctx.empty((24, 256))
        for tracks in (True, False):
            c.kv.track_weights(tracks)
            c.kv.attn_decode(3, c.seqs, [SHORT - 1], ctx.array(Q), o)
            assert np.all(np.abs(o.download() - out) <= off)
            if tracks:
                _held(c.weights(c.seqs[0], SHORT)[0], want, bound)

"""The typed cache's references themselves, on the CPU: the roundings against
their definition and the engine's quantiser, the 64-bit attention against the engine's own
functions, and planted mistakes that the bounds have to notice."""
import numpy as np
import pytest
from typed_rows import BF16, F16, F32, NORMAL_TOL, Q8_K, attend, off_by, rms64, rope64, stored


def test_stored_rows(ref):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((6, 1024)) * np.array([1, 1e-20, 1e4, 0, 3, 1e30])[:, None]).astype(np.float32)
    q, _, s = ref.q8k_split(ref.quantize_q8_k(x), 6, 1024)
    assert np.array_equal(stored(x, Q8_K), (q.reshape(6, 4, 256) * s[:, :, None]).astype(np.float32).reshape(6, 1024))
    assert np.array_equal(stored(x, F32), x)
    for ty, bits in ((F16, 10), (BF16, 7)):
        r = stored(x[:1], ty).astype(np.float64)
        step = 2.0 ** (np.floor(np.log2(np.abs(x[:1]))) - bits)
        step = np.maximum(step, 2.0 ** -24 if ty == F16 else 0.0)
        assert np.all(r / step == np.rint(r / step)) and np.all(np.abs(r - x[:1]) <= step / 2)
    ties = np.float32(1.0) + np.arange(0, 1024, dtype=np.float32) * np.float32(2.0 ** -8)
    assert np.array_equal(stored(ties[None], BF16)[0], np.rint(ties * 128 * np.where(ties < 2, 1, np.where(ties < 4, .5, .25))) /
                          128 / np.where(ties < 2, 1, np.where(ties < 4, .5, .25)))


def test_attend_against_the_engine(ref):
    rng = np.random.default_rng(2)
    q, g = (rng.standard_normal((24, 256)).astype(np.float32) for _ in range(2))
    k, v = (rng.standard_normal((77, 1024)).astype(np.float32) for _ in range(2))
    want, bound = attend(q, k, v, g)
    got = ref.attn_heads(q, k, v, gate=g).reshape(24, 256)
    assert np.all(np.abs(got - want) <= bound) and off_by(got, want) <= NORMAL_TOL


def test_key_rows_against_the_engine(ref):
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((4, 256)).astype(np.float32), rng.standard_normal(256).astype(np.float32)
    want = rope64(rms64(x[None], w), [1234])[0]
    got = np.concatenate([ref.rmsnorm(r, w) for r in x])
    got = ref.rope(got.astype(np.float32), 4, 1234).reshape(4, 256)
    assert np.abs(got - want).max() <= 12 * 2.0 ** -24 * np.abs(want).max() * 3


@pytest.mark.parametrize("P", [17, 200, 1000, 3003])
@pytest.mark.parametrize("mistake", ["a page left out", "a token past the end", "two values swapped", "a head's query lo part lost",
                                     "another page's keys", "a scale of the next token"])
def test_planted_mistakes_leave_the_bound(P, mistake):
    rng = np.random.default_rng(P)
    q = rng.standard_normal((24, 256)).astype(np.float32)
    k, v = (stored(rng.standard_normal((P + 1, 1024)), Q8_K) for _ in range(2))
    want, bound = attend(q, k[:P], v[:P])
    if mistake == "a page left out":
        got, _ = attend(q, k[16:P], v[16:P])
    elif mistake == "a token past the end":
        got, _ = attend(q, k, v)
    elif mistake == "two values swapped":
        w = v[:P].copy()
        w[[3, 9]] = w[[9, 3]]
        got, _ = attend(q, k[:P], w)
    elif mistake == "a head's query lo part lost":
        r = q.copy()
        r[5] = stored(np.tile(r[5], 4)[None], BF16)[0, :256]
        got, _ = attend(r, k[:P], v[:P])
    elif mistake == "another page's keys":
        w = k[:P].copy()
        w[:1] = k[P:P + 1]
        got, _ = attend(q, w, v[:P])
    else:
        w = v[:P].copy()
        w[7] *= 1.05
        got, _ = attend(q, k[:P], w)
    assert (np.abs(got - want) / bound).max() > 1.0 or off_by(got, want) > 4 * NORMAL_TOL

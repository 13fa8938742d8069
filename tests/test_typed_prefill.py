"""The limits of tests/test_gpu_typed_prefill.py and of full_core's, on the CPU:
the kernels' arithmetic passes the very assertions, and mistakes do not."""
import numpy as np
import pytest
from test_gpu_typed_prefill import CORE_TOL, check_core, check_prefill, core_inputs, piece
from typed_prefill import PREFILL_TOL, prefill_token
from typed_rows import BF16, TYPES, attend, off_by, stored

PIECES = [(0, 33), (0, 200), (33, 7), (300, 65)]


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("base,n", [(0, 1)] + PIECES)
def test_the_arithmetic_holds(ty, base, n):
    x = piece(base, n, TYPES[ty])
    for t in {0, n // 2, n - 1}:
        end = base + t + 1
        check_prefill(prefill_token(x.q[t], x.k[:end], x.v[:end], x.g[t]), x, t)


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("base,n", PIECES)
@pytest.mark.parametrize("mistake", ["the query's lower part lost", "the key's", "the weight's", "the value's", "token 0 left out",
                                     "the last token left out", "a token too many", "two values swapped", "no gate"])
def test_mistakes_are_noticed(ty, base, n, mistake):
    x = piece(base, n, TYPES[ty])
    t = n // 2
    end = base + t + 1
    lost = {"the query's lower part lost": "q", "the key's": "k", "the weight's": "p", "the value's": "v"}.get(mistake, "")
    if ty == "bf16" and lost in ("k", "v") and lost:
        pytest.skip("bf16 rows have no lower part")
    a, b = (1, end) if mistake == "token 0 left out" else (0, end - 1) if mistake == "the last token left out" else \
        (0, end + 1) if mistake == "a token too many" else (0, end)
    v = x.v.copy()
    if mistake == "two values swapped":
        v[[0, t]] = v[[t, 0]]
    got = prefill_token(x.q[t], x.k[a:b], v[a:b], None if mistake == "no gate" else x.g[t], lost)
    with pytest.raises(AssertionError):
        check_prefill(got, x, t)


@pytest.mark.parametrize("ty", sorted(TYPES))
@pytest.mark.parametrize("P", [2, 40, 1500])
@pytest.mark.parametrize("mistake", ["", "the query rounded to f16", "the query rounded to bf16", "token 0 left out", "the new token left out"])
def test_full_cores_limit(ref, ty, P, mistake):
    q, k, v, g = core_inputs(ref, P, TYPES[ty])
    r = stored(q, TYPES["f16" if "f16" in mistake else "bf16"]) if "rounded" in mistake else q
    a, b = (1 if "token 0" in mistake else 0), (P - 1 if "new token" in mistake else P)
    got = attend(r, k[a:b], v[a:b], g)[0].astype(np.float32)
    if not mistake:
        check_core(got, *attend(q, k, v, g))
        assert off_by(got, attend(q, k, v, g)[0]) <= CORE_TOL
    else:
        with pytest.raises(AssertionError):
            check_core(got, *attend(q, k, v, g))


def test_limits():
    assert PREFILL_TOL < 2.0 ** -15 and CORE_TOL < 2.0 ** -15 and BF16 in TYPES.values()

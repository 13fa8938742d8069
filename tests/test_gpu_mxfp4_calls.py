"""Random calls and stored infinities on caches of 4-bit rows: the typed caches'
checks of them, with one type more."""
import importlib.util
import os

import numpy as np
import pytest
import typed_rows
from mxfp4_rows import MXFP4, stored4

pytestmark = pytest.mark.gpu


def _checks(name):
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), name + ".py")
    spec = importlib.util.spec_from_file_location("mxfp4_" + name, path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.TYPES = {"mxfp4": MXFP4}
    m.stored = lambda x, ty: stored4(x) if ty == MXFP4 else typed_rows.stored(x, ty)
    return m


CALLS, PAGES, BAD = (_checks(n) for n in ("test_gpu_kv_types_random", "test_gpu_typed_random_pages", "test_gpu_typed_infinities"))


def _spoiled(ty, which):
    """A bad element of a key reaches its kv head's heads, of a value the 32 dims that share its scale."""
    s = np.zeros((24, 256), bool)
    s[6 * BAD.HEAD:6 * BAD.HEAD + 6, slice(None) if which == "key" else slice(BAD.DIM // 32 * 32, BAD.DIM // 32 * 32 + 32)] = True
    return s


BAD._spoiled = _spoiled


@pytest.mark.parametrize("seed", range(6))
def test_random_calls(pkg, ctx, seed):
    CALLS.test_random_calls(pkg, ctx, "mxfp4", seed)


@pytest.mark.parametrize("seed", range(4))
def test_random_calls_on_placed_pages(pkg, ctx, seed):
    run = [f for n, f in vars(PAGES).items() if n.startswith("test_")]
    assert len(run) == 1
    run[0](pkg, ctx, "mxfp4", seed)


@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinities_stay_where_they_are(pkg, ctx, which, bad):
    BAD.test_they_stay_where_they_are(pkg, ctx, "mxfp4", which, bad)


@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinities_in_a_prefill(pkg, ctx, which, bad):
    BAD.test_prefill(pkg, ctx, "mxfp4", which, bad)

"""The reference of the 4-bit rows' tests, held to its definition (CPU)."""
import numpy as np
from mxfp4_rows import LEVELS, stored4


def test_each_value_is_the_nearest_of_its_block():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 1024)) * np.exp2(rng.integers(-60, 60, (64, 1)))).astype(np.float32)
    got = stored4(x).astype(np.float64).reshape(-1, 32)
    b = x.astype(np.float64).reshape(-1, 32)
    for row, have in zip(b, got):
        big = np.abs(row).max()
        unit = min(2.0 ** k for k in range(-130, 130) if big <= 7 * 2.0 ** k)
        grid = np.concatenate((-LEVELS, LEVELS)) * unit
        best = np.abs(row[:, None] - grid).min(-1)
        assert np.array_equal(np.abs(row - have), best)
        # no value is cut by more than half a step of the largest code
        assert best.max() <= unit


def test_ties_ends_and_zeros():
    x = np.zeros((1, 1024), np.float32)
    x[0, :16] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.5]
    want = [0, 1, 1, 2, 2, 4, 4, 6, 0, -1, -1, -2, -2, -4, -4, 6]
    assert np.array_equal(stored4(x)[0, :16], np.array(want, np.float32))
    x[0, 0] = np.float32(np.nextafter(np.float32(7.0), np.float32(8.0)))  # past 7: the scale doubles
    assert stored4(x)[0, 0] == 8.0 and stored4(x)[0, 1] == 1.0
    big = np.full((1, 1024), np.finfo(np.float32).max, np.float32)
    assert np.all(stored4(big) == np.float32(6 * 2.0 ** 125))
    assert not stored4(np.zeros((2, 1024), np.float32)).any()
    tiny = np.full((1, 1024), 2.0 ** -126, np.float32)
    assert np.all(stored4(tiny) == np.float32(2.0 ** -126)) and not stored4(tiny / np.float32(4)).any()
    x[0, 40] = np.inf
    assert np.isnan(stored4(x)[0, 32:64]).all() and not np.isnan(stored4(x)[0, :32]).any()

"""Integer lists across the binding: four bytes each, whatever holds them and however
many there are (CPU only)."""
import array

import numpy as np
import pytest


@pytest.mark.parametrize("n", [0, 1, 4, 63, 64, 65, 68, 70, 200])
@pytest.mark.parametrize("kind", [list, tuple, bytes, bytearray, "int32", "int64", "uint8", "float", "h", "q", "range", "bool"])
def test_integer_lists(pkg, n, kind):
    values = [(37 * i) % 128 for i in range(n)]
    if kind in ("int32", "int64", "uint8"):
        given = np.array(values, kind)
    elif kind == "float":
        given = [float(v) for v in values]
    elif kind in ("h", "q"):
        given = array.array(kind, values)
    elif kind == "range":
        given, values = range(n), list(range(n))
    elif kind == "bool":
        values = [v % 2 for v in values]
        given = [bool(v) for v in values]
    else:
        given = kind(values)
    got = pkg._i32(given)
    assert len(got) == 4 * n and np.frombuffer(got, np.int32).tolist() == values


@pytest.mark.parametrize("n", [3, 64, 65, 100])
def test_values_past_32_bits_convert_as_before(pkg, n):
    assert np.frombuffer(pkg._i32([2 ** 31 + 5] * n), np.int32).tolist() == [5 - 2 ** 31] * n
    assert np.frombuffer(pkg._i32([-1] * n), np.int32).tolist() == [-1] * n
    with pytest.raises((TypeError, ValueError)):
        pkg._i32(["x"] * n)

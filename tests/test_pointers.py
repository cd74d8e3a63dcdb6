"""Pointers of the binding's arguments: tensors, numpy arrays, whole numbers and None, each at the cost of a
lookup (a whole number is not tried as a tensor first)."""
import timeit

import numpy as np
import pytest

import vsl


def test_every_kind_of_pointer():
    torch = pytest.importorskip("torch")
    t, a = torch.zeros(4), np.zeros(4)
    assert vsl._ptr(t) == t.data_ptr() and vsl._ptr(a) == a.ctypes.data
    assert vsl._ptr(None) is None and vsl._ptr(1 << 40) == 1 << 40 and vsl._ptr(0) == 0
    assert vsl._ptr(type("Address", (int,), {})(48)) == 48
    for bad in ("16", 16.0, [16], np.int64(16)):
        with pytest.raises(TypeError):
            vsl._ptr(bad)


def test_whole_numbers_are_as_quick_as_none():
    def ns(x):
        return min(timeit.repeat(lambda: vsl._ptr(x), number=20000, repeat=9))
    assert ns(123456) < 4 * ns(None)

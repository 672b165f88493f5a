"""Mode and block lists as the library gets them."""
import numpy as np
import pytest

from hiptensor_b200 import _lib


class Label:
    """A mode that someone renames."""

    def __init__(self, n):
        self.n = n

    def __int__(self):
        return self.n


@pytest.mark.parametrize("marshal", [_lib.i32, _lib.u32])
def test_lists_are_what_they_hold_now(marshal):
    a = Label(5)
    modes = (a, 7)
    assert list(marshal(modes)) == [5, 7]
    a.n = 6
    assert list(marshal(modes)) == [6, 7]


@pytest.mark.parametrize("marshal", [_lib.i32, _lib.u32])
@pytest.mark.parametrize("modes", [(1, 2), [1, 2], (np.int64(1), np.array(2)), (np.array(1), 2), np.array([1, 2]), (True, 2.0), ()])
def test_lists_of_any_kind_of_number(marshal, modes):
    assert list(marshal(modes)) == [1, 2][: len(modes)]


def test_no_list():
    assert _lib.i32(None) is None and _lib.u32(None) is None

"""A test finds no error text that another one has left, in whatever order they run."""
from accelgcn import _lib


def test_a_refusal_leaves_its_text():
    assert _lib.load().agcn_dropout(None, 0, None, 0, 1, 0, 0, 0, 0.5, 0, 0, None, 0, None) == _lib.ERR_INVALID
    assert b"columns" in _lib.load().agcn_last_error()


def test_which_the_next_test_does_not_see():
    assert _lib.load().agcn_last_error() == b""

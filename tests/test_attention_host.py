"""Attention's host side, on a machine without a GPU."""
import pytest

from falkon_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    _lib.build()
    return _lib.load()


def test_wait_limits(lib):
    for ns in (-1, 2000000001):
        with pytest.raises(ValueError):
            _lib.attention_wait_limit(ns)
    for ns in (0, 2000000000, 1000000000):  # the last one is what a process starts with
        _lib.attention_wait_limit(ns)

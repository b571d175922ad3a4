"""Attention's host side, on a machine without a GPU."""
import glob
import os
import re

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


def test_loads_from_tensor_memory_end_where_they_begin():
    """A register that such a load is still to fill must not be moved or spilled: load and wait are one statement."""
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    loads = 0
    for path in sorted(glob.glob(os.path.join(csrc, "flk_attn*"))):
        if not path.endswith((".cu", ".cuh")):
            continue
        with open(path) as f:
            text = f.read()
        assert "tmem_ld" not in text, f"{path}: a load whose wait is a statement of its own"
        for statement in re.findall(r"asm volatile\((.*?)\);\n", text, flags=re.S):
            if "tcgen05.ld" in statement:
                loads += 1
                assert "tcgen05.wait::ld" in statement, path
    assert loads > 0

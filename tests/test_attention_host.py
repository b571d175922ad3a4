"""Attention's host side, on a machine without a GPU."""
import glob
import os
import re

import sys

import pytest
import torch

from falkon_b200 import _lib, mmv_ops  # noqa: F401


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


def test_labels_beyond_int32_do_not_fall_together():
    table = sys.modules["falkon_b200.mmv_ops.attention"]._table
    t = torch.tensor([[0, 2**31 - 1, 2**31, 2**31 + 5, 2**32, 2**62, -1, -(2**31), -(2**40)]])
    got = table("documents", t, t.shape, t.device, True)
    assert got.dtype == torch.int32 and got[0, :2].tolist() == [0, 2**31 - 1] and bool((got[0, 2:] < 0).all())
    got = table("kv_lens", t, t.shape, t.device)
    assert got[0].tolist() == [0] + [2**31 - 1] * 5 + [-1] + [-(2**31)] * 2

"""QA_PAGES_STRICT without a device: the flag, and the tests' own model of it."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import pages
from pages_strict import STRICT, strict_model
from test_pages import _fork, _refused


@pytest.mark.parametrize("flags,needle", [(STRICT, "null context"), (STRICT | pages.KEEP, "null context"), (2, "flags 0x2"), (8, "flags 0x8"), (2 | STRICT, "flags 0x2")])
def test_flags(pkg, flags, needle):
    assert pkg.PAGES_STRICT == STRICT and pkg.PAGES_KEEP == pages.KEEP
    _refused(pkg, pkg.lib().qa_pages_fork, _fork(pkg, flags=flags), needle)
    n = ctypes.c_size_t()
    assert pkg.lib().qa_pages_fork_workspace(ctypes.byref(_fork(pkg, flags=flags)), ctypes.byref(n)) == 0


def test_the_model_counts_what_rows_do_not_hold():
    refs, table = np.array([1, 1, 0, 0, 0, 0], np.int32), np.array([[0, 1]], np.int32)
    for have, grow, missing in ((32, 1, 2), (31, 1, 0), (31, 2, 2), (30, 18, 2), (30, 19, 4), (32, 0, 0), (0, 33, 2), (2 ** 31 - 1, 1, 2)):
        want = strict_model(refs, table, np.array([have], np.int32), [0, 0, -1], np.array([grow] * 3, np.int32), 16, 6)
        assert want[3] == missing, (have, grow)
        if missing:
            assert (want[0] == -1).all() and (want[1] == 0).all() and np.array_equal(want[2], refs) and want[4] == []
    assert strict_model(refs, table, np.array([32], np.int32), [0] * 40, np.full(40, 2 ** 31 - 1, np.int32), 16, 6)[3] == 2 ** 31 - 1

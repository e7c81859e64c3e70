"""qa_pages_fork and qa_pages_compact refuse buffers that overlap, before they look for a device: numbers that one part of a call
wrote for itself and another part wrote over would be taken for page numbers."""
from __future__ import annotations

import pytest

from test_pages import _compact, _fork, _refused

# where test_pages puts them, and their bytes: _fork's for 100 pages, 4 sources, 6 sequences of 8 pages, _compact's for 6
FORK_OUT = dict(table=(0x230000, 192), len=(0x240000, 24), refs=(0x100000, 400), missing=(0x260000, 4))
FORK_IN = dict(src_table=(0x200000, 128), src_len=(0x210000, 16), parent=(0x220000, 24), grow=(0x250000, 24))
COMPACT_OUT = dict(refs_out=(0x110000, 400), table_out=(0x210000, 192), map=(0x220000, 400), used=(0x230000, 4))
COMPACT_IN = dict(refs=(0x100000, 400), table=(0x200000, 192))


def _pairs(names):
    names = list(names)
    return [(a, b) for i, a in enumerate(names) for b in names[i + 1:]]


@pytest.mark.parametrize("a,b", _pairs(FORK_OUT))
def test_fork_outputs(pkg, a, b):
    """The first or the last number of one in the other, either way round; side by side they are taken."""
    fn = pkg.lib().qa_pages_fork
    for x, y in ((a, b), (b, a)):
        (at, n), (_, m) = FORK_OUT[x], FORK_OUT[y]
        for put in (at, at + n - 4, at - m + 4):
            _refused(pkg, fn, _fork(pkg, **{y: put}), "overlap")
        for put in (at + n, at - m):
            _refused(pkg, fn, _fork(pkg, **{y: put}), "null context")


@pytest.mark.parametrize("name", [*FORK_OUT, *FORK_IN])
def test_fork_workspace(pkg, name):
    at, n = {**FORK_OUT, **FORK_IN}[name]
    need = pkg.pages_fork_workspace(_fork(pkg))
    fn = pkg.lib().qa_pages_fork
    for put in (at, at - need // 16 * 16 + (0 if need % 16 else 16), at + (n - 1) // 16 * 16):
        _refused(pkg, fn, _fork(pkg, workspace=put, workspace_bytes=need), "overlap")
    for put in (at + (n + 15) // 16 * 16, at - (need + 15) // 16 * 16):
        _refused(pkg, fn, _fork(pkg, workspace=put, workspace_bytes=1 << 30), "null context")  # what a larger one has beyond is not written


def test_fork_of_nothing(pkg):
    """Lists without numbers may be anywhere."""
    fn = pkg.lib().qa_pages_fork
    _refused(pkg, fn, _fork(pkg, seqs=0, table=0x100000, len=0x100000), "null context")
    _refused(pkg, fn, _fork(pkg, src_seqs=0, src_table=0x100000, src_len=0x300000), "null context")
    _refused(pkg, fn, _fork(pkg, grow=None), "null context")


@pytest.mark.parametrize("a,b", _pairs(COMPACT_OUT))
def test_compact_outputs(pkg, a, b):
    fn = pkg.lib().qa_pages_compact
    for x, y in ((a, b), (b, a)):
        (at, n), (_, m) = COMPACT_OUT[x], COMPACT_OUT[y]
        for put in (at, at + n - 4, at - m + 4):
            _refused(pkg, fn, _compact(pkg, **{y: put}), "overlap")
        for put in (at + n, at - m):
            _refused(pkg, fn, _compact(pkg, **{y: put}), "null context")


@pytest.mark.parametrize("name", [*COMPACT_OUT, *COMPACT_IN])
def test_compact_workspace(pkg, name):
    at, n = {**COMPACT_OUT, **COMPACT_IN}[name]
    need = pkg.pages_compact_workspace(_compact(pkg))
    fn = pkg.lib().qa_pages_compact
    for put in (at, at - (need - 1) // 16 * 16, at + (n - 1) // 16 * 16):
        _refused(pkg, fn, _compact(pkg, workspace=put, workspace_bytes=need), "overlap")
    for put in (at + (n + 15) // 16 * 16, at - (need + 15) // 16 * 16):
        _refused(pkg, fn, _compact(pkg, workspace=put, workspace_bytes=1 << 30), "null context")


def test_compact_in_place(pkg):
    """In place, and without a map or a table."""
    fn = pkg.lib().qa_pages_compact
    _refused(pkg, fn, _compact(pkg, refs_out=0x100000, table_out=0x200000), "null context")
    _refused(pkg, fn, _compact(pkg, map=None), "null context")
    _refused(pkg, fn, _compact(pkg, seqs=0, table=0x110000, table_out=0x110000), "null context")

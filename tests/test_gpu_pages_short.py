"""qa_pages_fork without enough pages on an MI355X, in every form of the call: references that a launch of its own has changed,
sequences counted in the workspace, searches through many rounds.  All is as it was, and *missing is exact."""
from __future__ import annotations

import numpy as np
import pytest

from pages import Fork, Pool, fork_model, random_sequences

pytestmark = pytest.mark.gpu


def _short(ctx, pkg, pool, refs, table, length, parent, grow, short, **kw):
    """The call with `short` pages too few, the free ones that are left at the pool's end; then with just enough."""
    n, width = pool.num_pages, table.shape[1]
    free = np.nonzero(refs == 0)[0]
    refs = refs.copy()
    refs[free] = 1
    few = fork_model(refs, table, length, parent, grow, 16, n, **kw)[3] - short  # of the free pages
    assert 0 <= few <= len(free) - short
    refs[free[len(free) - few:]] = 0
    for spare in (0, short):
        if spare:
            refs[free[len(free) - few - spare:]] = 0
        want = fork_model(refs, table, length, parent, grow, 16, n, **kw)
        assert want[3] == short - spare
        call = Fork(ctx, pkg, pool, 16, refs, table, length, parent, grow, **kw).run()
        got = call.read()
        if not spare:
            assert got[3] == short and (got[0] == -1).all() and got[0].shape == (len(parent), width) and (got[1] == 0).all()
            assert np.array_equal(got[2], refs)
        for name, a, b in zip(("table", "len", "refs", "missing"), got, want):
            assert np.array_equal(a, b), (name, spare)
        pool.move(want[4])
        pool.check()
        call.free()


# One launch and a pool of several rounds; entries beyond one launch, at most 1024 sequences; more of them; long rows.
SHAPES = [(5, 4, 12, 20000), (600, 500, 8, 10000), (1024, 1024, 2, 5000), (1025, 900, 4, 9000), (3000, 2000, 3, 16000), (1500, 1400, 8, 30000), (2, 3, 2000, 12000)]


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("short", [1, 20])
@pytest.mark.parametrize("seqs,src,width,num_pages", SHAPES)
def test_without_enough_pages(ctx, pkg, seqs, src, width, num_pages, short, keep):
    r = np.random.default_rng(seqs + width)
    pool = Pool(ctx, pkg, num_pages, (64, 4), seed=6)
    most = min(8 * width, 200)
    table, length, refs = random_sequences(r, src, 16, width, num_pages, most)
    parent = r.integers(0, src, seqs).astype(np.int32)
    parent[1] = parent[0]
    if seqs > 10:
        parent[r.integers(0, seqs, 9)] = -1
    grow = r.integers(0 if seqs > 10 else 4 * width, 16 * width - most + 1, seqs).astype(np.int32)
    _short(ctx, pkg, pool, refs, table, length, parent, grow, short, window=30 if seqs == 3000 else 0, sinks=5, keep=keep)
    pool.free()

"""qa_pages_fork with QA_PAGES_STRICT for the tests: what it does, and the call."""
from __future__ import annotations

import numpy as np

import pages

STRICT = 4


def strict_model(refs, src_table, src_len, parent, grow, page, num_pages, before=0, table=None, **kw):
    """fork_model where growth behind the end of a row is a shortage; `before`: what *missing holds, which if not 0 leaves
    `table` and all but the lengths as they are."""
    if before:
        return table, np.zeros(len(parent), np.int32), refs.astype(np.int32), before, []
    width = src_table.shape[1]
    cap = min(width * page, 2 ** 30)
    past = 0
    for i, q in enumerate(parent):
        if 0 <= q < len(src_len) and grow is not None:
            want = min(max(int(src_len[q]), 0), cap) + max(0, int(grow[i]))
            past += max(0, -(-want // page) - cap // page)
    table, length, after, missing, pairs = pages.fork_model(refs, src_table, src_len, parent, grow, page, num_pages, **kw)
    if past:
        table, length, after, pairs = np.full_like(table, -1), np.zeros_like(length), refs.astype(np.int32), []
    return table, length, after, min(missing + past, 2 ** 31 - 1), pairs


def strict_fork(ctx, pkg, pool, page, refs, table, length, parent, grow, before=0, **kw):
    """The call, checked against the model: every number, every byte of the pool."""
    was = np.full((len(parent), table.shape[1]), 77, np.int32)  # (Fork's)
    want = strict_model(refs, table, length, parent, grow, page, pool.num_pages, before=before, table=was, **kw)
    call = pages.Fork(ctx, pkg, pool, page, refs, table, length, parent, grow, **kw)
    call.desc.flags |= STRICT
    ctx.upload(call.missing, np.array([before], np.int32))
    got = call.run().read()
    for name, a, b in zip(("table", "len", "refs", "missing"), got, want):
        assert np.array_equal(a, b), (name, a, b)
    pool.move(want[4])
    pool.check()
    call.free()
    return want

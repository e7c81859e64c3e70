"""The beam search of test_gpu_beam_search whose pool runs out of pages, its forks strict: two captured steps, replayed past the
shortage, leave what the same steps leave that stop there, and the pages can be given back."""
from __future__ import annotations

import numpy as np
import pytest

from hipgraph import Capture
from paged import BF16, E4M3, F16
from pages_strict import STRICT
from test_gpu_beam_search import BEAMS, GROUPS, HD, LAYERS, NKV, NQ, Search, narrow

pytestmark = pytest.mark.gpu


def _begin(ctx, pkg, dtype, cache, num_pages, width):
    s = Search(ctx, pkg, dtype, cache, num_pages, width, seed=1)
    r = np.random.default_rng(2)
    ctx.upload(s.score[1], np.tile(np.array([0.0] + [-np.inf] * (BEAMS - 1), np.float32), GROUPS))
    ctx.upload(s.parent, np.where(np.arange(s.S) % BEAMS == 0, np.arange(s.S), -1).astype(np.int32))
    for layer in range(LAYERS):
        ctx.upload(s.qkv[layer], narrow(r.standard_normal((s.S, (NQ + 2 * NKV) * HD)), dtype))
    return s


def _left(ctx, s):
    """(the number missing, references, every page)"""
    return (int(ctx.download(s.missing, (1,), np.int32)[0]), ctx.download(s.refs, (s.num_pages,), np.int32),
            [ctx.download(m, (m.nbytes,), np.uint8) for m in s.mem])


@pytest.mark.parametrize("num_pages,width", [(20, 12), (21, 12), (200, 3)], ids=["pages", "more-pages", "rows"])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4M3)], ids=["f16", "bf16-e4m3"])
def test_captured_search_past_a_shortage(pkg, dtype, cache, num_pages, width):
    with pkg.Context(0) as ctx:
        s = _begin(ctx, pkg, dtype, cache, num_pages, width)
        steps = 0
        while True:  # up to the first fork that is short
            live, source = s.tables[s.turn], s.turn
            s.fork(keep=STRICT)
            if ctx.download(s.missing, (1,), np.int32)[0]:
                break
            s.layers()
            s.select(5)
            steps += 1
            assert steps < 100
        assert steps > 2
        missing, refs, mem = _left(ctx, s)
        table = ctx.download(live, (s.S, s.width), np.int32)
        s.free()
    count = np.zeros(num_pages, np.int32)
    np.add.at(count, table[table >= 0], 1)
    assert np.array_equal(count, refs) and refs.sum() > 0
    with pkg.Context(0) as ctx:
        s = _begin(ctx, pkg, dtype, cache, num_pages, width)

        def two():
            for _ in range(2):
                s.fork(keep=STRICT)
                s.layers()
                s.select(5)
        two()
        with Capture(ctx.stream) as cap:
            two()
        for _ in range(steps // 2 + 3):
            cap.replay()
            ctx.download(s.logits, (s.S, 8))  # the program's own work between the replays
        cap.close()
        got = _left(ctx, s)
        assert got[0] == missing and np.array_equal(got[1], refs) and all(np.array_equal(a, b) for a, b in zip(got[2], mem))
        assert np.array_equal(ctx.download(s.tables[source], (s.S, s.width), np.int32), table)
        assert (ctx.download(s.tables[1 - source], (s.S, s.width), np.int32) == -1).all()
        assert all((ctx.download(x, (s.S,), np.int32) == 0).all() for x in s.lens)
        # from either table to no sequences: the one gives nothing, the other everything
        for turn in (1 - source, source):
            ctx.upload(s.missing, np.zeros(1, np.int32))
            d = pkg.PagesForkDesc(flags=STRICT, page=16, num_pages=s.num_pages, planes=s.planes, nplanes=len(s.mem), refs=int(s.refs), src_seqs=s.S, seqs=0,
                                  ldtable=s.width, src_table=int(s.tables[turn]), src_len=int(s.lens[turn]), missing=int(s.missing))
            ctx.pages_fork(s.workspace(d, pkg.pages_fork_workspace(d)))
            left = ctx.download(s.refs, (s.num_pages,), np.int32)
            assert np.array_equal(left, refs if turn != source else np.zeros_like(refs))
            assert ctx.download(s.missing, (1,), np.int32)[0] == 0
        s.free()

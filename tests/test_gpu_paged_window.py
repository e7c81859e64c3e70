"""qa_attention_paged_window on an MI355X against its definition in 64 bits (tests/paged_window.py), at the windows, sinks,
pages and batches where it can go wrong.  Tolerances: paged_window.assert_window."""
from __future__ import annotations

import numpy as np
import pytest

from hipgraph import Capture
from paged import BF16, E4M3, F16, STALE8, STALE16, Batch, attention, widen
from paged_window import assert_window, spoil_unseen, window_attention, window_desc

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)],
                                  ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])

BATCHES = [
    # rows, keys, page, nq, nkv, hd
    ([1], [1], 16, 16, 8, 128),
    ([1, 1, 1, 1], [700, 64, 65, 129], 16, 16, 8, 128),
    ([1] * 5, [2, 333, 640, 1000, 17], 64, 4, 2, 64),
    ([3, 0, 16], [300, 40, 16], 32, 6, 6, 64),
    ([40, 1, 0, 70], [400, 333, 12, 71], 32, 16, 8, 128),
    ([200], [863], 64, 3, 3, 128),
    ([130, 2], [130, 500], 16, 6, 2, 64),
    ([5], [3], 16, 2, 1, 128),          # fewer keys than rows: the first two have no position
    ([33, 300], [640, 900], 32, 10, 1, 64),
]
WINDOWS = [(1, 0), (1, 1), (16, 0), (63, 4), (64, 64), (65, 1), (130, 17), (300, 200), (7, 1000)]


@FORMATS
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("n,lens,page,nq,nkv,hd", BATCHES)
def test_window(ctx, pkg, dtype, cache, n, lens, page, nq, nkv, hd, window, sinks):
    """With everything that no row sees NaN or gone."""
    b = Batch(n, lens, page, nq, nkv, hd, dtype, cache, seed=sum(lens) + window)
    b.fill()
    spoil_unseen(b, window, sinks)
    b.upload(ctx)
    q = b.random_rows(nq * hd)
    assert_window(b, q, window_attention(ctx, pkg, b, q, window, sinks), window, sinks)
    b.free()


@FORMATS
@pytest.mark.parametrize("n,lens,window,sinks,rows", [
    ([1], [20011], 16000, 5, None), ([1, 1, 1], [9000, 130, 12097], 3000, 300, None), ([40], [9001], 6000, 70, (0, 17, 39)),
    ([700, 1], [2000, 9000], 500, 4, (0, 1, 350, 699)), ([1500], [4000], 100, 0, (0, 63, 64, 700, 1499)), ([20], [30000], 700, 20000, (0, 19))])
def test_long(ctx, pkg, dtype, cache, n, lens, window, sinks, rows):
    """Windows and sinks long enough to be split, in small parts of long caches."""
    b = Batch(n, lens, 32, 8, 4, 128, dtype, cache, seed=9)
    b.fill()
    spoil_unseen(b, window, sinks)
    b.upload(ctx)
    q = b.random_rows(8 * 128)
    assert_window(b, q, window_attention(ctx, pkg, b, q, window, sinks), window, sinks, rows=rows)
    b.free()


@FORMATS
@pytest.mark.parametrize("n,lens", [([1, 1, 40], [300, 4000, 900]), ([1], [9000]), ([90, 300], [90, 1500])])
@pytest.mark.parametrize("window,sinks", [(2 ** 30, 0), (20000, 7), (5, 2 ** 30)])
def test_all_keys_are_attention_paged(ctx, pkg, dtype, cache, n, lens, window, sinks):
    """A window or sinks over all keys: the same bits."""
    b = Batch(n, lens, 16, 4, 2, 128, dtype, cache, seed=5)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(4 * 128)
    assert np.array_equal(window_attention(ctx, pkg, b, q, window, sinks), attention(ctx, pkg, b, q))
    b.free()


@FORMATS
@pytest.mark.parametrize("n", [8, 90])
def test_keys_of_nan_in_front_of_a_window(ctx, pkg, dtype, cache, n):
    """A key that the first row alone sees may be NaN: that row is, and no other."""
    b = Batch([n], [200], 16, 2, 1, 64, dtype, cache, seed=42)
    b.fill()
    key = 200 - n - 59
    b.k[b.table[0, key // 16], :, key % 16] = STALE8 if cache == E4M3 else STALE16[dtype]
    b.upload(ctx)
    q = b.random_rows(2 * 64)
    got = window_attention(ctx, pkg, b, q, 60, 3)
    assert_window(b, q, got, 60, 3, rows=range(1, n))
    assert np.isnan(widen(got[0], dtype)).all()
    b.free()


@FORMATS
@pytest.mark.parametrize("page", [16, 32, 64])
def test_pages_that_are_none_inside(ctx, pkg, dtype, cache, page):
    """Holes among the keys that rows see, and sequences that lose all of them: zeros."""
    b = Batch([1, 1, 50, 2, 1], [200, 64, 130, 90, 700], page, 4, 2, 128, dtype, cache, seed=41)
    b.fill()
    b.table[0, 160 // page] = -1
    b.table[2, 64 // page] = b.num_pages
    b.table[1, :] = -3
    b.table[4, 576 // page:] = 2 ** 31 - 1
    b.upload(ctx)
    q = b.random_rows(4 * 128)
    for window, sinks in ((60, 0), (100, 20), (1, 0)):
        assert_window(b, q, window_attention(ctx, pkg, b, q, window, sinks), window, sinks)
    b.free()


@FORMATS
def test_many_sequences(ctx, pkg, dtype, cache):
    """150 sequences of no row, one, a few and many, over shared pages."""
    rng = np.random.default_rng(101)
    n = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 9, 17, 40, 90], 150)]
    lens = [int(rng.integers(k, 600)) for k in n]
    b = Batch.shared(n, lens, 16, 4, 2, 64, dtype, cache, seed=102)
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    assert_window(b, q, window_attention(ctx, pkg, b, q, 77, 9), 77, 9)
    b.free()


@FORMATS
@pytest.mark.parametrize("page,hd", [(16, 64), (64, 64), (32, 128)])
def test_single_tokens_behind_many_pages(ctx, pkg, dtype, cache, page, hd):
    """64 sequences whose keys are not split: a wave goes through its page ids 16 blocks at a time."""
    b = Batch.shared([1] * 64, [9000, 6097, 8192] + [60] * 60 + [8300], page, 16, 8, hd, dtype, cache, seed=103)
    b.table[[0, 63], 8000 // page] = -1
    b.upload(ctx)
    q = b.random_rows(16 * hd)
    assert_window(b, q, window_attention(ctx, pkg, b, q, 5000, 100), 5000, 100, seqs=(0, 1, 2, 30, 63))
    b.free()


@FORMATS
def test_lengths_past_the_bounds(ctx, pkg, dtype, cache):
    b = Batch([1, 4], [96, 64], 32, 4, 2, 64, dtype, cache, seed=44, extra_slots=0)
    b.fill()
    b.kv_len = np.array([2 ** 31 - 1, 64], np.int32)  # stands for max_len = 96
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    assert_window(b, q, window_attention(ctx, pkg, b, q, 20, 3), 20, 3)
    got = window_attention(ctx, pkg, b, q, 20, 3, max_rows=2)
    assert (got[3:5] == 0x3C01).all() and (got[:3] != 0x3C01).any(1).all()
    b.free()


@FORMATS
def test_captured_with_other_lengths(ctx, pkg, dtype, cache):
    """A captured call replayed on batches whose sequences are shorter and longer, within the bounds; two graphs, each with
    its own workspace."""
    big = Batch([1, 30, 1], [3000, 1500, 700], 32, 4, 2, 128, dtype, cache, seed=61)
    big.fill()
    big.upload(ctx)
    q = big.random_rows(4 * 128)
    dq = ctx.to_device(q)
    calls = []
    for window, sinks in ((1200, 40), (100, 0)):
        out = ctx.to_device(np.full(q.shape, 0x3C01, np.uint16))
        d = window_desc(pkg, big, dq, q.shape[1], out, q.shape[1], window, sinks)
        size = pkg.attention_paged_window_workspace(d)
        ws = ctx.to_device(np.full(max(size, 16), 0xFF, np.uint8))
        d.workspace, d.workspace_bytes = int(ws), size
        with Capture(ctx.stream) as cap:
            ctx.attention_paged_window(d)
        calls.append((window, sinks, out, ws, cap))
    for lens in ([3000, 1500, 700], [40, 30, 1], [1201, 1100, 699], [3000, 1500, 700]):
        big.len, big.kv_len = list(lens), np.array(lens, np.int32)
        ctx.upload(big.dev["kv_len"], big.kv_len)
        for window, sinks, out, _, cap in calls:
            cap.replay()
        eager = [window_attention(ctx, pkg, big, q, w, s) for w, s, *_ in calls]
        for (window, sinks, out, _, _), e in zip(calls, eager):
            got = ctx.download(out, q.shape)
            assert np.array_equal(got, e)
            assert_window(big, q, got, window, sinks, rows=(0, 7, 29))
    for _, _, out, ws, cap in calls:
        cap.close()
        out.free()
        ws.free()
    dq.free()
    big.free()

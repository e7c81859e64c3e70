"""qa_attention_paged_window with more than 16 q heads to a kv head on an MI355X: single tokens too go through the long sequences'
tiles, which begin and end inside a row.  Tolerances: paged_window.assert_window."""
from __future__ import annotations

import numpy as np
import pytest

from paged import BF16, E4M3, F16, Batch, attention
from paged_window import assert_window, spoil_unseen, window_attention

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)],
                                  ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])


@FORMATS
@pytest.mark.parametrize("nq,nkv,hd,page", [(17, 1, 128, 16), (32, 1, 64, 64), (40, 2, 128, 32), (100, 1, 64, 16), (129, 1, 128, 64)])
@pytest.mark.parametrize("n,lens,window,sinks", [
    ([1], [1], 1, 0), ([1, 1, 1], [700, 64, 129], 65, 4), ([1, 0, 2, 1], [333, 20, 130, 1000], 300, 70), ([5], [3], 16, 0), ([30, 1], [200, 640], 63, 1)])
def test_window(ctx, pkg, dtype, cache, nq, nkv, hd, page, n, lens, window, sinks):
    b = Batch(n, lens, page, nq, nkv, hd, dtype, cache, seed=nq + window)
    b.fill()
    spoil_unseen(b, window, sinks)
    b.upload(ctx)
    q = b.random_rows(nq * hd)
    assert_window(b, q, window_attention(ctx, pkg, b, q, window, sinks), window, sinks)
    b.free()


@FORMATS
@pytest.mark.parametrize("nq,nkv", [(24, 1), (66, 2)])
@pytest.mark.parametrize("n,lens,window,sinks,rows", [([1], [9001], 3000, 5, None), ([1] * 9, [5000, 17, 2000] * 3, 1500, 300, None), ([70], [4000], 2000, 0, (0, 1, 35, 69))])
def test_long(ctx, pkg, dtype, cache, nq, nkv, n, lens, window, sinks, rows):
    """Windows that are split over blocks and joined, of few blocks and of more."""
    b = Batch(n, lens, 32, nq, nkv, 128, dtype, cache, seed=nq)
    b.fill()
    spoil_unseen(b, window, sinks)
    b.upload(ctx)
    q = b.random_rows(nq * 128)
    assert_window(b, q, window_attention(ctx, pkg, b, q, window, sinks), window, sinks, rows=rows)
    b.free()


@FORMATS
def test_all_keys_are_attention_paged(ctx, pkg, dtype, cache):
    b = Batch([1, 3, 40], [4000, 70, 900], 16, 48, 2, 64, dtype, cache, seed=6)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(48 * 64)
    assert np.array_equal(window_attention(ctx, pkg, b, q, 2 ** 30, 0), attention(ctx, pkg, b, q))
    b.free()

"""qa_kv_append and qa_attention_paged on an MI355X where the batch's bounds, the
pages' contents or the formats' last bits decide (definitions: tests/paged.py)."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import rope_tables, ulp16
from paged import BF16, E4M3, F16, STALE8, STALE16, Batch, append, assert_attention, attention, attention_desc, e4m3_codes, e4m3_values, narrow, widen

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)],
                                  ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])


def _put(b, s, K, V, scale=2.0 ** -6):
    """Sequence s's keys: K, V [nkv, len, hd], exact in the cache's format (e4m3: at this scale)."""
    for i in range(-(-b.len[s] // b.page)):
        p, at = b.table[s, i], slice(i * b.page, (i + 1) * b.page)
        k, v = K[:, at], V[:, at].transpose(0, 2, 1)
        m = k.shape[1]
        if b.cache == E4M3:
            b.k_scale[p], b.v_scale[p] = scale, scale
            k, v = e4m3_codes(k / scale), e4m3_codes(v / scale)
        else:
            k, v = narrow(k, b.dtype), narrow(v, b.dtype)
        b.k[p, :, :m], b.v[p, :, :, :m] = k, v


@FORMATS
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,lens", [([1] * 24, list(range(3, 27))), ([1], [1500]), ([40], [300]), ([70, 1], [1500, 20])])
def test_probabilities_keep_their_last_bits(ctx, pkg, dtype, cache, hd, n, lens):
    """Two keys of nearly the same score with V = 1 and -1, the others' V 0: out = (p1 - p2) / sum p is 2^-13 of p1, and shows
    what was lost of either.  Scores are exact in f32 (one or two products of few bits).  What may be lost, over p1 / sum p:
      * p1, p2: the exponent's factor and rounding, 2^-25 (|arg| < 0.2; in f16, whose p carry a factor of 2^7, the
        exponent's last bit is 2^-22, times ln 2), exp2's 2^-23: 2.5 2^-23 for both (f16: 3 2^-23 more);
      * the terms in the product: f16 2^-22 each; three of bf16 nothing; two (bf16 pages, more than 16 rows and heads) 2^-18 each;
      * the sum of up to six products: 6 2^-24;
    then (keys + 16) 2^-24 of the result, the sum of p, and half a step of the output."""
    nq, nkv = 4, 2
    b = Batch(n, lens, 16, nq, nkv, hd, dtype, cache, seed=hd + sum(lens))
    b.stale()
    for s, m in enumerate(lens):
        K, V = np.zeros((nkv, m, hd)), np.zeros((nkv, m, hd))
        K[:, :, 0] = b.rng.integers(-8, 4, (nkv, m)) / 8.0
        K[:, 0, 0] = 1.0
        if m > 2:
            K[:, 1, 0] = K[:, 2, 0] = b.rng.integers(4, 8, nkv) / 8.0
            K[:, 1, 1], V[:, 1], V[:, 2] = 1.0, 1.0, -1.0
        _put(b, s, K, V)
    b.upload(ctx)
    x = np.zeros((b.tokens, nq, hd))
    x[..., 0] = b.rng.integers(64, 128, x.shape[:2]) / 128.0 * np.sqrt(hd / 64)  # 6 or 7 bits (sqrt 2 at hd 128: rounded to the format)
    x[..., 1] = 2.0 ** -10 * (1 + b.rng.integers(0, 128, x.shape[:2]) / 128.0)
    q = narrow(x.reshape(b.tokens, -1), dtype)
    got = widen(attention(ctx, pkg, b, q), dtype).reshape(b.tokens, nq, hd)
    x = widen(q, dtype).reshape(b.tokens, nq, hd)
    per_p = 2.5 * 2.0 ** -23 + 6 * 2.0 ** -24
    two = cache == BF16
    for s, m in enumerate(lens):
        K, _, _ = b.keys(s)
        for r in range(n[s]):
            t, see = b.row_start[s] + r, m - n[s] + r + 1
            if see < 3:
                continue
            lost = per_p + (5 * 2.0 ** -23 if cache == F16 else 2 * 2.0 ** -18 if two and n[s] * nq // nkv > 16 else 0.0)
            for h in range(nq):
                sc = K[h * nkv // nq, :see] @ x[t, h] / np.sqrt(hd)
                p = np.exp(sc - sc.max())
                want = (p[1] - p[2]) / p.sum()
                bound = lost * p[1] / p.sum() + abs(want) * (see + 16) * 2.0 ** -24
                bound += float(ulp16(np.array(abs(want) + bound), dtype)) / 2
                err = np.abs(got[t, h] - want).max()
                assert err <= bound, (s, r, h, err / bound)
    b.free()


def _rows(b):
    """qkv, norm weights, cosines and sines for b's rows."""
    qkv = b.random_rows((b.nq + 2 * b.nkv) * b.hd)
    w = [(1.0 + 0.2 * b.rng.standard_normal(b.hd)).astype(np.float32) for _ in range(2)]
    return (qkv, *w, *rope_tables(b.tokens, b.hd, 0, dtype=b.dtype))


def _nothing_as_zero(b, cache):
    """The cache with zeros where nothing was ever written (0 * NaN would reach the definition's sums)."""
    def nothing(a):  # (an e4m3 page that is rounded again keeps its NaN, but not their signs)
        return a & 0x7F == STALE8 if b.cache == E4M3 else a == STALE16[b.dtype]

    return {n: np.where(nothing(a), 0, a).astype(a.dtype) if n in ("k", "v") else np.nan_to_num(a, nan=1.0) for n, a in cache.items()}


@FORMATS
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n,lens,max_rows,cut", [([40], [45], 30, 0), ([5, 3, 1], [20, 70, 64], 2, 0), ([1, 40], [20, 45], 40, 5),
                                                 ([90, 1], [1500, 3], 20, 0), ([200], [200], 64, 0), ([1, 6], [7, 260], 3, 0)])
def test_slots_of_rows_left_out_are_not_looked_at(ctx, pkg, dtype, cache, page, n, lens, max_rows, cut):
    """Rows past max_rows or past `tokens`: what their slots and pages' scales hold (NaN: nothing was written yet) reaches no
    row that is kept, and they are left as they are."""
    b = Batch(n, lens, page, 4, 2, 64, dtype, cache, seed=sum(lens) + page, tail_rows=0 if cut else 2)
    b.fill([m - k for k, m in zip(n, lens)])
    b.upload(ctx)
    x, q, before = _rows(b), b.random_rows(4 * 64), b.read(ctx)
    b.tokens -= cut
    qkv, qn, kn, c, s = x
    append(ctx, pkg, b, qkv[: b.tokens], qn, kn, c[: b.tokens], s[: b.tokens], max_rows=max_rows)
    after = b.read(ctx)
    got = attention(ctx, pkg, b, q[: b.tokens], max_rows=max_rows)
    held = _nothing_as_zero(b, after)
    kept = [min(k, max_rows) for k in n]
    kept[-1] = min(kept[-1], n[-1] - cut)
    for sq in range(b.seqs):
        r0 = b.row_start[sq]
        assert (got[r0 + kept[sq]: r0 + n[sq]] == 0x3C01).all()
        for pos in range(lens[sq] - n[sq] + kept[sq], lens[sq]):
            p, at = b.table[sq, pos // page], pos % page
            for a, z in ((after["k"][p, :, at], before["k"][p, :, at]), (after["v"][p, :, :, at], before["v"][p, :, :, at])):
                assert np.array_equal(a & 0x7F, z & 0x7F) if cache == E4M3 else np.array_equal(a, z)  # NaN, whose sign may change
    out = np.concatenate([got, np.full((cut, got.shape[1]), 0x3C01, np.uint16)])  # the definition's batch is the whole one
    for sq in range(b.seqs):
        assert_attention(b, q, out, rows=range(kept[sq]), seqs=[sq], **held)
    b.free()


@FORMATS
@pytest.mark.parametrize("n,lens,page,max_rows", [([40, 1, 5], [70, 9, 64], 16, 4), ([90], [200], 32, 33), ([3, 0, 2, 2], [3, 5, 40, 2], 64, 1)])
def test_append_of_rows_past_max_rows(ctx, pkg, dtype, cache, n, lens, page, max_rows):
    """q, pages and scales are those of a call for each sequence that has its first max_rows rows alone; the other rows of
    q stay as they were."""
    b = Batch(n, lens, page, 6, 2, 64, dtype, cache, seed=sum(lens))
    b.fill([m - k for k, m in zip(n, lens)], kstd=0.3, vstd=0.3)
    b.upload(ctx)
    x, before = _rows(b), b.read(ctx)
    got, after = append(ctx, pkg, b, *x, max_rows=max_rows), b.read(ctx)
    for name, a in before.items():
        ctx.upload(b.dev[name], a)
    want = np.full_like(got, 0x1234)
    for s, k in enumerate(n):
        kept, r0 = min(k, max_rows), b.row_start[s]
        one = {name: ctx.to_device(a) for name, a in (("row_start", np.array([r0, r0 + kept], np.int32)), ("table", b.table[s]),
                                                      ("kv_len", np.array([lens[s] - k + kept], np.int32)))}
        q = append(ctx, pkg, b, *x, seqs=1, **{name: int(d) for name, d in one.items()})
        want[r0:r0 + kept] = q[r0:r0 + kept]
        for d in one.values():
            d.free()
    assert (want != 0x1234).any(1).sum() == sum(min(k, max_rows) for k in n)
    assert np.array_equal(got, want)
    each = b.read(ctx)
    assert all(np.array_equal(after[name], each[name], equal_nan=after[name].dtype == np.float32) for name in after)
    b.free()


@pytest.mark.parametrize("seqs", [63, 64, 65, 4000, 5000])
def test_append_finds_a_row_among_many_sequences(ctx, pkg, seqs):
    """Up to four rows a sequence, two of them kept: the kept ones' q and slots have the bits of a call with all of them."""
    rng = np.random.default_rng(seqs)
    n = [int(x) for x in rng.choice([0, 1, 2, 3, 4], seqs)]
    n[0], n[-1] = 0, 3
    b = Batch(n, [k + int(rng.integers(0, 9)) for k in n], 16, 2, 1, 64, F16, F16, seed=seqs + 1)
    b.stale()
    b.upload(ctx)
    x, before = _rows(b), b.read(ctx)
    all_q, whole = append(ctx, pkg, b, *x), b.read(ctx)
    for name, a in before.items():
        ctx.upload(b.dev[name], a)
    q, after = append(ctx, pkg, b, *x, max_rows=2), b.read(ctx)
    place = np.concatenate([np.arange(k) for k in n] + [np.full(b.tokens - sum(n), 9)])
    assert np.array_equal(q, np.where((place < 2)[:, None], all_q, 0x1234))
    k, v = before["k"].copy(), before["v"].copy()
    for s in range(seqs):
        for i in range(min(n[s], 2)):
            pos = b.len[s] - n[s] + i
            p, at = b.table[s, pos // 16], pos % 16
            k[p, :, at], v[p, :, :, at] = whole["k"][p, :, at], whole["v"][p, :, :, at]
    assert np.array_equal(after["k"], k) and np.array_equal(after["v"], v)
    b.free()


@FORMATS
@pytest.mark.parametrize("n,lens,max_rows", [([300, 1, 1], [300, 3000, 900], 300), ([1] * 20, [3000, 40] * 10, 16), ([1, 1, 1], [5000, 2, 1300], 1),
                                             ([90], [3000], 90), ([90, 1, 2], [3000, 2000, 100], 90), ([3, 8, 8], [4000, 4001, 8], 8)])
def test_workspace_is_all_that_is_written(ctx, pkg, dtype, cache, n, lens, max_rows):
    """Partial results of short and of long sequences, in either order: the call is right with exactly the bytes that it asks
    for, whatever they hold before, and nothing behind them changes."""
    b = Batch(n, lens, 32, 4, 2, 64, dtype, cache, seed=sum(lens))
    b.fill()
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    dq, do = ctx.to_device(q), ctx.to_device(np.full(q.shape, 0x3C01, np.uint16))
    d = attention_desc(pkg, b, dq, q.shape[1], do, q.shape[1], max_rows=max_rows)
    size = pkg.attention_paged_workspace(d)
    assert size > 0
    ws = ctx.to_device(np.concatenate([np.full(size, 0xFF, np.uint8), np.full(8192, 0xA5, np.uint8)]))
    d.workspace, d.workspace_bytes = int(ws), size
    ctx.attention_paged(d)
    got = ctx.download(do, q.shape)
    assert (ctx.download(ws, (8192,), np.uint8, size) == 0xA5).all()
    assert_attention(b, q, got)
    for x in (dq, do, ws):
        x.free()
    b.free()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,lens,cut", [([1, 40], [20, 45], 5), ([1, 6], [20, 30], 3)])
def test_append_to_e4m3_leaves_the_slots_of_rows_past_the_batch(ctx, pkg, dtype, n, lens, cut):
    """The last rows lie past `tokens`.  Their slots hold finite values: in a page whose first slot is new its codes stay as they
    are, whatever its scale becomes; in a page that held rows before they are rounded again with it."""
    b = Batch(n, lens, 16, 4, 2, 64, dtype, E4M3, seed=sum(lens), tail_rows=0)
    b.fill(kstd=0.3, vstd=0.3)
    b.upload(ctx)
    (qkv, qn, kn, c, s), before = _rows(b), b.read(ctx)
    b.tokens -= cut
    append(ctx, pkg, b, qkv[: b.tokens], qn, kn, c[: b.tokens], s[: b.tokens])
    after = b.read(ctx)
    first, page = lens[1] - n[1], (lens[1] - cut) // 16
    assert (lens[1] - 1) // 16 == page
    p, at = b.table[1, page], np.arange(lens[1] - cut, lens[1]) % 16
    fresh = first <= page * 16
    assert fresh == (n[1] == 40)
    for name, axis in (("k", 1), ("v", 2)):
        old, now = (x[name + "_scale"][p].astype(np.float64) for x in (before, after))
        assert (now > old).all()  # these rows' values are smaller than the new ones
        held, got = (np.take(x[name][p], at, axis) for x in (before, after))
        want = held if fresh else e4m3_codes(e4m3_values(held) * (old / now)[:, None, None])
        assert np.array_equal(got, want), name
    b.free()


@FORMATS
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_wave_goes_through_several_windows_of_pages(ctx, pkg, dtype, cache, page, hd):
    """One token behind 20011 keys under a bound of 2^20, which leaves the keys in one part: each of four waves goes through 78
    blocks of 64 keys, whose pages are looked up 16 blocks at a time.  Pages in the third and fourth windows are none."""
    b = Batch([1], [20011], page, 4, 2, hd, dtype, cache, seed=hd + page, tail_rows=0, extra_slots=2 ** 20 // page)
    b.fill()
    b.table[0, [9001 // page, 15000 // page, 20000 // page]] = -1
    b.upload(ctx)
    q = b.random_rows(4 * hd)
    size = pkg.attention_paged_workspace(attention_desc(pkg, b, 0, 4 * hd, 0, 4 * hd, max_len=2 ** 20))
    parts = size // (4 * (hd + 2) * 4)
    assert parts * 4 * (hd + 2) * 4 == size and 2 ** 20 // parts > 20011  # no part ends before the keys do
    assert_attention(b, q, attention(ctx, pkg, b, q, max_len=2 ** 20))
    b.free()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,lens", [([1, 1], [37, 700]), ([40], [100])])
def test_scales_at_the_ends_of_their_range(ctx, pkg, dtype, n, lens):
    """K scales of the smallest normal number (all scores round to 0) and of 2^100 with K of zeros: every key that a row sees has
    the same weight, the ones that it does not see none."""
    for scale, k in ((2.0 ** -126, None), (2.0 ** 100, 0)):
        b = Batch(n, lens, 16, 4, 2, 64, dtype, E4M3, seed=sum(lens))
        b.fill()
        b.k_scale[:] = scale
        if k is not None:
            b.k[:] = k
        b.upload(ctx)
        q = b.random_rows(4 * 64)
        assert_attention(b, q, attention(ctx, pkg, b, q))
        b.free()

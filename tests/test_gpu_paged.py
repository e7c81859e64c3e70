"""qa_mrope_rows, qa_kv_append and qa_attention_paged on an MI355X against their
definitions in 64 bits (tests/paged.py), at the sizes, tables and contents where
they can go wrong.

Tolerances, derived:
  * rotary rows: half a step of the 16-bit format around the f64 cosine, plus
    the rounding to f32 before it (2^-24 relative) and 2^-50 for the f64
    evaluation of angles up to 2^31 (relative to the angle: 2^-52 * 2^31 * 2 for
    the far ones, given there).
  * q and K: inv = 1 / sqrt(mean + eps) in f32 is off by at most (hd / 2 + 3) 2^-24
    (half the sum's gamma_hd, sqrt, divide, mean), each product and the
    rotation's sum by 2^-24: (hd / 2 + 10) 2^-24 (|a cos| + |b sin|); then half a
    step of the 16-bit format, or of e4m3 at the page's scale.
  * V, and a page that is rounded again: equal codes.
  * attention: paged.assert_attention.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import paged
from conftest import rope_tables, ulp16
from hipgraph import Capture, hip
from paged import (BF16, E4M3, F16, STALE8, STALE16, Batch, append, assert_attention, attention, e4m3_codes, e4m3_step, e4m3_values, narrow,
                   scale_for, widen)

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)],
                                  ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])
DTYPES = pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])


# ------------------------------------------------------------ rotary rows

def _mrope(ctx, pkg, dtype, pos, hd, sec, inter, theta=1e6, pad=3):
    axes, n = pos.shape
    sec = list(sec) + [0] * (3 - axes)
    p = ctx.to_device(np.pad(pos.astype(np.int32), ((0, 0), (0, pad)), constant_values=77))
    c, s = (ctx.to_device(np.full((n + 1, hd), 9.0, np.float32)) for _ in range(2))
    ctx.mrope_rows(pkg.MropeDesc(dtype=dtype, flags=pkg.MROPE_INTERLEAVED if inter else 0, tokens=n, hd=hd, axes=axes, sec0=sec[0], sec1=sec[1],
                                 sec2=sec[2], theta=theta, pos=int(p), ldpos=n + pad, cos=int(c), sin=int(s)))
    out = [ctx.download(x, (n + 1, hd), np.float32) for x in (c, s)]
    for x in (p, c, s):
        x.free()
    assert all((x[n] == 9.0).all() for x in out)  # the row behind the last is not written
    return [x[:n] for x in out]


def _axes_of(hd, axes, sec, inter):
    if not inter:
        return np.repeat(np.arange(axes), sec)
    return np.array([j % axes if j < axes * sec[j % axes] else 0 for j in range(hd // 2)])


@DTYPES
@pytest.mark.parametrize("hd,sec,inter,n", [
    (128, (64,), False, 1), (128, (64,), True, 5), (128, (24, 20, 20), True, 300), (128, (16, 24, 24), False, 257), (64, (12, 20), False, 33),
    (64, (12, 20), True, 64), (8, (2, 1, 1), True, 3), (256, (128,), False, 9), (256, (0, 100, 28), False, 19), (128, (64, 0, 0), True, 7),
    (128, (0, 32, 32), True, 40), (24, (5, 4, 3), True, 200), (200, (100,), False, 31), (88, (20, 24), True, 47)])
def test_mrope_rows(ctx, pkg, dtype, hd, sec, inter, n):
    rng = np.random.default_rng(hd + n)
    pos = rng.integers(0, 5000, (len(sec), n))
    got = _mrope(ctx, pkg, dtype, pos, hd, sec, inter)
    ang = pos[_axes_of(hd, len(sec), sec, inter)].T / 1e6 ** (2.0 * np.arange(hd // 2) / hd)
    for x, f in zip(got, (np.cos, np.sin)):
        want = f(ang)
        assert np.array_equal(x[:, : hd // 2], x[:, hd // 2:])
        assert (np.abs(x[:, : hd // 2] - want) <= ulp16(want, dtype) / 2 + np.abs(want) * 2.0 ** -24 + 2.0 ** -50).all()


@DTYPES
def test_mrope_far_and_negative_positions(ctx, pkg, dtype):
    pos = np.array([[2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, -1, 0, 10 ** 9 + 7]])
    got = _mrope(ctx, pkg, dtype, pos, 128, (64,), False)
    # the angle as the definition forms it, in 80-bit arithmetic behind the f64 product
    ang = (pos[0][:, None].astype(np.float64) * (1.0 / 1e6 ** (2.0 * np.arange(64) / 128))[None]).astype(np.longdouble)
    for x, f in zip(got, (np.cos, np.sin)):
        want = f(ang).astype(np.float64)
        # pow's last place moves an angle by 2^-52 of itself
        assert (np.abs(x[:, :64] - want) <= ulp16(want, dtype) / 2 + np.abs(want) * 2.0 ** -24 + np.abs(ang).astype(np.float64) * 2.0 ** -51).all()


@DTYPES
@pytest.mark.parametrize("axes,inter", [(1, False), (3, True), (2, False)])
def test_mrope_of_equal_axes_is_rope_tables(ctx, pkg, dtype, axes, inter):
    hd, n = 128, 200
    sec = [64 - 20 * (axes - 1)] + [20] * (axes - 1)
    c, s = _mrope(ctx, pkg, dtype, np.tile(np.arange(n), (axes, 1)), hd, sec, inter)
    wc, ws = pkg.rope_tables(n, hd, 1e6, dtype)
    assert np.array_equal(c, wc) and np.array_equal(s, ws)


# ----------------------------------------------------------------- append

def _inputs(b, std=2.0):
    qkv = b.random_rows((b.nq + 2 * b.nkv) * b.hd, std)
    qn, kn = ((1.0 + 0.2 * b.rng.standard_normal(b.hd)).astype(np.float32) for _ in range(2))
    c, s = rope_tables(b.tokens + 90, b.hd, 0, dtype=b.dtype)
    at = b.rng.permutation(b.tokens + 90)[: b.tokens]  # any positions: a row's own cos and sin
    return qkv, qn, kn, np.ascontiguousarray(c[at]), np.ascontiguousarray(s[at])


def _turned(b, x, w, c, s):
    """RMSNorm and rotation of x [rows, heads, hd] in 64 bits, and the f32 error's bound."""
    h = b.hd // 2
    y = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + paged.EPS) * w.astype(np.float64)
    c, s = c.astype(np.float64)[:, None], s.astype(np.float64)[:, None]
    swapped = np.concatenate([-y[..., h:], y[..., :h]], -1)
    return y * c + swapped * s, (h + 10) * 2.0 ** -24 * (np.abs(y * c) + np.abs(swapped * s))


def _check_append(b, before, after, q, inputs, q0=0x1234, checked_scales=True):
    """Everything qa_kv_append leaves, against the definition."""
    qkv, qn, kn, c, s = inputs
    x = widen(qkv, b.dtype).reshape(b.tokens, -1, b.hd)
    lo, hi = b.row_start[0], b.row_start[-1]
    assert (q[:lo] == q0).all() and (q[hi:] == q0).all()
    want, err = _turned(b, x[:, : b.nq], qn, c, s)
    got = widen(q, b.dtype).reshape(b.tokens, b.nq, b.hd)
    assert (np.abs(got - want) <= err + ulp16(np.abs(want) + err, b.dtype) / 2)[lo:hi].all()
    kw, kerr = _turned(b, x[:, b.nq: b.nq + b.nkv], kn, c, s)
    vbits = qkv.reshape(b.tokens, -1, b.hd)[:, b.nq + b.nkv:]
    model = {n: a.copy() for n, a in before.items()}  # what no row of this batch touches
    for sq in range(b.seqs):
        n, m = b.n[sq], b.len[sq]
        pos = m - n + np.arange(n)
        for i in sorted({int(p) // b.page for p in pos if p >= 0}):
            p = b.table[sq, i]
            if not 0 <= p < b.num_pages:
                continue
            rows = b.row_start[sq] + np.nonzero((pos >= 0) & (pos // b.page == i))[0]
            slots = pos[rows - b.row_start[sq]] % b.page
            a, z = slots[0], slots[-1] + 1
            k, kt, v = kw[rows].transpose(1, 0, 2), kerr[rows].transpose(1, 0, 2), vbits[rows].transpose(1, 2, 0)
            if b.cache != E4M3:
                got = widen(after["k"][p, :, a:z], b.dtype)
                assert (np.abs(got - k) <= kt + ulp16(np.abs(k) + kt, b.dtype) / 2).all()
                model["k"][p, :, a:z], model["v"][p, :, :, a:z] = after["k"][p, :, a:z], v
                continue
            vf = widen(np.ascontiguousarray(v), b.dtype)
            for name, y in (("k", k), ("v", vf)):
                fin = np.where(np.isfinite(y), np.abs(y), 0.0)
                need = scale_for(fin.max((1, 2)))
                old = np.zeros(b.nkv) if a == 0 else np.nan_to_num(before[name + "_scale"][p].astype(np.float64), nan=0.0, posinf=0.0)
                now = np.maximum(np.maximum(old, 0), need)
                assert np.array_equal(after[name + "_scale"][p].astype(np.float64), now), (name, p)
                model[name + "_scale"][p] = now
                if a > 0:  # the page is rounded again where its scale grew
                    for h in range(b.nkv):
                        if now[h] != old[h]:
                            model[name][p, h] = e4m3_codes(e4m3_values(before[name][p, h]) * (old[h] / now[h]))
                if name == "v":
                    with np.errstate(invalid="ignore"):
                        model["v"][p, :, :, a:z] = e4m3_codes(vf / now[:, None, None])
                else:
                    g = e4m3_values(after["k"][p, :, a:z])
                    r = k / now[:, None, None]
                    t = kt / now[:, None, None]
                    assert (np.abs(g - r) <= t + e4m3_step(np.minimum(np.abs(r) + t, 448.0)) / 2).all()
                    model["k"][p, :, a:z] = after["k"][p, :, a:z]
    for n in model:
        same = (model[n] == after[n]) | (np.isnan(model[n]) & np.isnan(after[n]) if model[n].dtype == np.float32 else False)
        if n in ("k", "v") and b.cache == E4M3:  # a NaN keeps no sign
            same |= (model[n] & 0x7F == 0x7F) & (after[n] & 0x7F == 0x7F)
        assert same.all(), (n, np.argwhere(~same)[:4])


APPEND = [
    # rows, keys, page, nq, nkv, hd
    ([1], [1], 16, 16, 8, 128),
    ([1, 1, 1], [16, 17, 15], 16, 16, 8, 128),          # last and first slot of a page
    ([1] * 5, [1, 64, 65, 130, 200], 64, 4, 2, 64),
    ([40, 1, 0, 70], [40, 33, 12, 101], 32, 16, 8, 128),  # prompts, a step, no rows
    ([200], [263], 64, 3, 3, 128),
    ([130, 2], [130, 50], 16, 6, 2, 64),
    ([0, 0], [5, 0], 16, 2, 1, 128),
    ([5], [3], 16, 2, 1, 128),                            # fewer keys than rows: the first two have no position
    ([33, 17], [64, 96], 32, 10, 1, 64),
]


@FORMATS
@pytest.mark.parametrize("n,lens,page,nq,nkv,hd", APPEND)
def test_append(ctx, pkg, dtype, cache, n, lens, page, nq, nkv, hd):
    b = Batch(n, lens, page, nq, nkv, hd, dtype, cache, seed=sum(lens) + page)
    # earlier keys are smaller than the new rows: e4m3 scales have to grow
    b.fill([max(0, m - k) for m, k in zip(lens, n)], kstd=0.3, vstd=0.3)
    b.upload(ctx)
    before, x = b.read(ctx), _inputs(b)
    q = append(ctx, pkg, b, *x)
    _check_append(b, before, b.read(ctx), q, x)
    b.free()


@DTYPES
def test_append_keeps_a_large_scale(ctx, pkg, dtype):
    """Rows that are smaller than what their page holds leave scale and page alone."""
    b = Batch([1, 3], [20, 40], 32, 4, 2, 128, dtype, E4M3, seed=3)
    b.fill([19, 37], kstd=50.0, vstd=50.0)
    b.upload(ctx)
    before, x = b.read(ctx), _inputs(b)
    q = append(ctx, pkg, b, *x)
    after = b.read(ctx)
    _check_append(b, before, after, q, x)
    for s, i in ((0, 0), (1, 1)):
        p = b.table[s, i]
        assert np.array_equal(after["k_scale"][p], before["k_scale"][p]) and np.array_equal(after["v_scale"][p], before["v_scale"][p])
    b.free()


def test_append_scales_that_are_no_powers_of_two(ctx, pkg):
    """A page filled with other scales keeps a larger one, and is rounded again from it when it grows."""
    for std in (0.05, 30.0):
        b = Batch([2, 1], [30, 17], 32, 4, 2, 128, F16, E4M3, seed=8)
        b.fill([28, 16], kstd=std, vstd=std, pow2=False)
        b.upload(ctx)
        before, x = b.read(ctx), _inputs(b)
        q = append(ctx, pkg, b, *x)
        after = b.read(ctx)
        # ratios that are no powers of two round an f32 product once more than the restatement's double
        for name in ("k", "v"):
            for s, i, held in ((0, 0, 28), (1, 0, 16)):
                p = b.table[s, i]
                part = (slice(None), slice(0, held)) if name == "k" else (slice(None), slice(None), slice(0, held))
                old = before[name + "_scale"][p].astype(np.float64)[:, None, None]
                now = after[name + "_scale"][p].astype(np.float64)[:, None, None]
                r = e4m3_values(before[name][p][part]) * (old / now)
                assert (np.abs(e4m3_values(after[name][p][part]) - r) <= e4m3_step(r) * (0.5 + 2.0 ** -18)).all()
                assert (now >= old).all()
        b.free()


@DTYPES
@pytest.mark.parametrize("hd", [64, 128])
def test_append_rounds_keys_to_e4m3_once(ctx, pkg, dtype, hd):
    """1500 keys a head: every code and scale is that of the 64-bit value.  The kernel's f64 is 2^-44 off at the most and a
    value is within that of a step's middle with a chance of 2^-40: none of 2^20 is."""
    b = Batch([1500], [1500], 32, 4, 4, hd, dtype, E4M3, seed=15)
    b.stale()
    b.upload(ctx)
    qkv, qn, kn, c, s = _inputs(b, 1.0)
    append(ctx, pkg, b, qkv, qn, kn, c, s)
    after = b.read(ctx)
    x = widen(qkv, dtype).reshape(b.tokens, -1, hd)[:1500, 4:8]
    k = _turned(b, x, kn, c[:1500], s[:1500])[0]
    for i in range(-(-1500 // 32)):
        p, part = b.table[0, i], k[32 * i:32 * i + 32].transpose(1, 0, 2)
        scale = scale_for(np.abs(part).max((1, 2)))
        assert np.array_equal(after["k_scale"][p], scale)
        assert np.array_equal(after["k"][p][:, : part.shape[1]], e4m3_codes(part / scale[:, None, None]))
    b.free()


def test_append_infinities_and_nan(ctx, pkg):
    """V with infinities and NaN in e4m3: the largest value and NaN, no part in the scale; in 16 bits as they are."""
    for cache in (E4M3, F16):
        b = Batch([20], [20], 16, 2, 1, 64, F16, cache, seed=5)
        b.stale()
        b.upload(ctx)
        qkv, qn, kn, c, s = _inputs(b)
        rows = qkv.reshape(b.tokens, -1, 64)
        rows[3, -1, 5], rows[4, -1, 6], rows[17, -1, 9], rows[18, -1, :] = 0x7C00, 0xFC00, 0x7E00, 0
        before = b.read(ctx)
        q = append(ctx, pkg, b, qkv, qn, kn, c, s)
        after = b.read(ctx)
        _check_append(b, before, after, q, (qkv, qn, kn, c, s))
        if cache == E4M3:
            p0, p1 = b.table[0, :2]
            assert after["v"][p0, 0, 5, 3] == 0x7E and after["v"][p0, 0, 6, 4] == 0xFE and after["v"][p1, 0, 9, 1] & 0x7F == 0x7F
        b.free()


def test_append_of_zeros_and_of_extremes(ctx, pkg):
    """A page of zeros, and bf16 values near both ends of f32's range, in e4m3."""
    for std in (0.0, 1e-37, 3e37):
        b = Batch([18, 1], [18, 40], 16, 2, 1, 64, BF16, E4M3, seed=6)
        b.stale()
        b.upload(ctx)
        qkv, qn, kn, c, s = _inputs(b, 1.0)
        v = (std * b.rng.standard_normal((b.tokens, 64))).clip(-3e38, 3e38)
        qkv.reshape(b.tokens, -1, 64)[:, -1] = narrow(v, BF16)
        before = b.read(ctx)
        q = append(ctx, pkg, b, qkv, qn, kn, c, s)
        _check_append(b, before, b.read(ctx), q, (qkv, qn, kn, c, s))
        b.free()


@FORMATS
def test_append_leaves_out_what_has_no_place(ctx, pkg, dtype, cache):
    """Pages that are none, rows past max_rows, and rows before the first sequence."""
    b = Batch([1, 40, 3, 6], [20, 45, 3, 30], 16, 4, 2, 64, dtype, cache, seed=12)
    b.table[1, 1], b.table[1, 2], b.table[2, 0] = -1, b.num_pages, 2 ** 31 - 1
    b.row_start[0] = 1  # the first sequence's only row is no one's
    b.n[0] = 0
    b.fill([20, 5, 0, 24], kstd=0.3, vstd=0.3)
    b.upload(ctx)
    before, x = b.read(ctx), _inputs(b)
    q = append(ctx, pkg, b, *x)
    _check_append(b, before, b.read(ctx), q, x)
    b.free()


# -------------------------------------------------------------- attention

ATTENTION = [
    # rows, keys, page, nq, nkv, hd
    ([1], [1], 16, 16, 8, 128),
    ([1], [17], 16, 16, 8, 128),
    ([1, 1, 1, 1], [15, 16, 63, 64], 16, 16, 8, 128),
    ([1, 1, 1], [65, 127, 129], 32, 4, 4, 128),
    ([1, 1], [256, 257], 64, 8, 2, 64),
    ([1], [1500], 16, 16, 8, 128),
    ([1] * 9, [3, 700, 64, 1, 300, 255, 512, 90, 1025], 32, 6, 2, 128),   # three heads to a kv head
    ([1, 2, 0, 5], [40, 70, 9, 5], 16, 16, 1, 128),                       # 16 heads to a kv head
    ([2, 1], [300, 31], 64, 20, 1, 64),                                   # 20: more than a tile's rows
    ([100], [100], 16, 16, 8, 128),
    ([64, 33], [64, 240], 64, 4, 2, 128),
    ([257, 1, 1], [300, 600, 2], 32, 6, 2, 64),
    ([1, 130], [900, 1100], 16, 3, 3, 128),
    ([7], [4], 16, 4, 2, 128),                                            # fewer keys than rows: three rows of zeros
    ([3, 4], [0, 2], 32, 4, 2, 64),
    ([0, 0], [5, 0], 16, 2, 1, 128),
    ([31, 17, 1, 16, 15], [31, 80, 81, 16, 47], 16, 10, 2, 64),
    ([1, 3], [70, 40], 16, 200, 1, 64),                                   # a row's heads in several tiles
]


@FORMATS
@pytest.mark.parametrize("n,lens,page,nq,nkv,hd", ATTENTION)
def test_attention(ctx, pkg, dtype, cache, n, lens, page, nq, nkv, hd):
    b = Batch(n, lens, page, nq, nkv, hd, dtype, cache, seed=sum(lens) + nq)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(nq * hd)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@FORMATS
@pytest.mark.parametrize("n,lens,rows", [([1], [20011], None), ([1, 1, 1], [9000, 130, 4097], None), ([40], [9001], (0, 17, 39)),
                                         ([700, 1], [2000, 3000], (0, 1, 350, 699))])
def test_attention_long(ctx, pkg, dtype, cache, n, lens, rows):
    """Long keys: many splits, joined."""
    b = Batch(n, lens, 32, 8, 4, 128, dtype, cache, seed=9)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(8 * 128)
    assert_attention(b, q, attention(ctx, pkg, b, q), rows=rows)
    b.free()


@FORMATS
@pytest.mark.parametrize("n,lens", [([1, 1], [700, 90]), ([90], [400])])
def test_attention_peaked_scores(ctx, pkg, dtype, cache, n, lens):
    """Score spread of ~6: the running maximum moves often."""
    b = Batch(n, lens, 16, 8, 4, 128, dtype, cache, seed=21)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(8 * 128, 6.0)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@DTYPES
def test_attention_other_scales(ctx, pkg, dtype):
    """Scales that are no powers of two, and pages whose scales lie far apart."""
    b = Batch([1, 30], [300, 150], 16, 4, 2, 128, dtype, E4M3, seed=31)
    b.fill(pow2=False)
    far = b.rng.choice(np.array([2.0 ** -30, 2.0 ** -4, 1.0, 3.0], np.float32), b.v_scale.shape)
    b.v_scale = (b.v_scale * far).astype(np.float32)
    b.upload(ctx)
    q = b.random_rows(4 * 128)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@FORMATS
@pytest.mark.parametrize("page", [16, 32, 64])
def test_attention_pages_that_are_none(ctx, pkg, dtype, cache, page):
    """Keys on such pages do not count, whole sequences of them give zeros."""
    b = Batch([1, 1, 50, 2, 1], [200, 64, 130, 90, 700], page, 4, 2, 128, dtype, cache, seed=41)
    b.fill()
    b.table[0, 1], b.table[2, 0], b.table[2, 1] = -1, b.num_pages, -2 ** 31
    b.table[1, :] = -3
    b.table[4, : 256 // page] = 2 ** 31 - 1
    b.upload(ctx)
    q = b.random_rows(4 * 128)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@FORMATS
def test_attention_of_lengths_past_the_bounds(ctx, pkg, dtype, cache):
    """kv_len past max_len, and rows past max_rows: held to the bounds, without an access outside the buffers."""
    b = Batch([1, 4], [96, 64], 32, 4, 2, 64, dtype, cache, seed=44, extra_slots=0)
    b.fill()
    b.kv_len = np.array([2 ** 31 - 1, 64], np.int32)  # stands for max_len = 96
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    got = attention(ctx, pkg, b, q, max_rows=2)
    assert (got[3:5] == 0x3C01).all() and (got[:3] != 0x3C01).any(1).all()
    b.free()


@FORMATS
def test_rows_past_the_batch_are_left_out(ctx, pkg, dtype, cache):
    """The last sequence's last five rows lie past `tokens`: the others have the same positions, keys and bits as with
    them, and nothing stands in for those."""
    b = Batch([1, 40], [20, 45], 16, 4, 2, 64, dtype, cache, seed=46, tail_rows=0)
    b.fill(kstd=0.3, vstd=0.3)
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    want = attention(ctx, pkg, b, q)
    before, (qkv, qn, kn, c, s) = b.read(ctx), _inputs(b)
    b.tokens -= 5
    assert np.array_equal(attention(ctx, pkg, b, q[:36]), want[:36])
    append(ctx, pkg, b, qkv[:36], qn, kn, c[:36], s[:36])
    after = b.read(ctx)
    p = b.table[1, 2]  # positions 32 .. 44: 40 .. 44 keep what they held, at the page's scale
    if cache == E4M3:
        held = e4m3_values(before["v"][p, :, :, 8:13]) * before["v_scale"][p].astype(np.float64)[:, None, None]
        now = e4m3_values(after["v"][p, :, :, 8:13]) * after["v_scale"][p].astype(np.float64)[:, None, None]
        if (after["v_scale"][p] == before["v_scale"][p]).all():
            assert np.array_equal(held, now)
        new = widen(qkv, dtype).reshape(41, -1, 64)[28:36, 6:].transpose(1, 2, 0)
        got = e4m3_values(after["v"][p, :, :, :8]) * after["v_scale"][p].astype(np.float64)[:, None, None]
        step = e4m3_step(new / after["v_scale"][p].astype(np.float64)[:, None, None]) * after["v_scale"][p].astype(np.float64)[:, None, None]
        assert (np.abs(got - new) <= step / 2).all()
    else:
        assert np.array_equal(after["v"][p, :, :, 8:], before["v"][p, :, :, 8:])
        assert np.array_equal(after["v"][p, :, :, :8], qkv.reshape(41, -1, 64)[28:36, 6:].transpose(1, 2, 0))
    b.free()


def test_attention_shared_pages_and_repeats(ctx, pkg):
    """A prefix in two tables, the same page twice in one; the same call again gives the same bits."""
    b = Batch([1, 1, 60], [100, 130, 160], 16, 8, 4, 128, F16, F16, seed=51)
    b.fill()
    b.table[1, :6] = b.table[0, :6]
    b.table[2, 3] = b.table[2, 2]
    b.upload(ctx)
    q = b.random_rows(8 * 128)
    got = attention(ctx, pkg, b, q)
    assert_attention(b, q, got)
    assert np.array_equal(attention(ctx, pkg, b, q), got)
    b.free()


@FORMATS
def test_attention_of_many_sequences(ctx, pkg, dtype, cache):
    """150 sequences of no row, one, a few and many, in any order."""
    rng = np.random.default_rng(101)
    n = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 9, 17, 40, 90], 150)]
    lens = [int(rng.integers(k, 300)) for k in n]
    b = Batch.shared(n, lens, 16, 4, 2, 64, dtype, cache, seed=102)
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@FORMATS
@pytest.mark.parametrize("page,hd", [(16, 64), (64, 64), (32, 128)])
def test_attention_of_single_tokens_behind_many_pages(ctx, pkg, dtype, cache, page, hd):
    """64 sequences, whose keys are not split: a wave goes through its page ids 16 blocks at a time.  A page in
    the middle is none."""
    b = Batch.shared([1] * 64, [9000, 4097, 8192] + [60] * 60 + [8300], page, 16, 8, hd, dtype, cache, seed=103)
    b.table[[0, 63], 5000 // page] = -1
    b.upload(ctx)
    q = b.random_rows(16 * hd)
    assert_attention(b, q, attention(ctx, pkg, b, q), seqs=(0, 1, 2, 30, 63))
    b.free()


@FORMATS
@pytest.mark.parametrize("page,hd", [(16, 64), (64, 128)])
def test_attention_of_single_tokens_behind_pages_in_one_part(ctx, pkg, dtype, cache, page, hd):
    """32 sequences of 8 kv heads behind up to 5000 keys: no call needs a workspace, a wave has up to 20 blocks."""
    b = Batch.shared([1] * 32, [5000, 4097, 4352, 4353] + [60] * 27 + [4800], page, 16, 8, hd, dtype, cache, seed=108)
    b.table[[0, 31], 4500 // page] = -1
    b.upload(ctx)
    q = b.random_rows(16 * hd)
    assert pkg.attention_paged_workspace(paged.attention_desc(pkg, b, 0, 16 * hd, 0, 16 * hd)) == 0
    assert_attention(b, q, attention(ctx, pkg, b, q), seqs=(0, 1, 2, 3, 30, 31))
    b.free()


@FORMATS
@pytest.mark.parametrize("page,hd", [(16, 64), (64, 64), (32, 128)])
def test_attention_of_rows_behind_many_pages(ctx, pkg, dtype, cache, page, hd):
    """The same for 17 and more rows: 128 sequences of 2 kv heads."""
    b = Batch.shared([17] * 127 + [20], [9000, 4500] + [60] * 125 + [8300], page, 2, 2, hd, dtype, cache, seed=104)
    b.table[[0, 127], 5000 // page] = -1
    b.upload(ctx)
    q = b.random_rows(2 * hd)
    assert_attention(b, q, attention(ctx, pkg, b, q), seqs=(0, 1, 77, 127))
    b.free()


@FORMATS
@pytest.mark.parametrize("page,hd", [(16, 64), (32, 64), (64, 64), (16, 128), (32, 128), (64, 128)])
def test_attention_of_long_tiles(ctx, pkg, dtype, cache, page, hd):
    """6000 rows of 8 kv heads: tiles of 128 rows, with few and many keys, whole and not, beside a single token."""
    b = Batch.shared([100] * 58 + [1, 130, 257], [4500, 100, 2100] + [130] * 55 + [700, 140, 600], page, 8, 8, hd, dtype, cache, seed=105)
    b.table[0, 4096 // page] = -1
    b.upload(ctx)
    q = b.random_rows(8 * hd)
    assert_attention(b, q, attention(ctx, pkg, b, q), seqs=(0, 1, 2, 40, 58, 59, 60), rows=(0, 1, 63, 64, 99, 127, 128, 129, 255, 256))
    b.free()


@FORMATS
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_many_split_sequences(ctx, pkg, dtype, cache, hd):
    """100 sequences of one kv head, single tokens and 20 rows in turn, whose keys are split: the join finds them past
    the first 64."""
    rng = np.random.default_rng(109)
    lens = [2500, 2400] + [int(rng.integers(20, 2500)) for _ in range(98)]
    b = Batch.shared([1, 20] * 50, lens, 16, 2, 1, hd, dtype, cache, seed=110)
    b.upload(ctx)
    q = b.random_rows(2 * hd)
    assert pkg.attention_paged_workspace(paged.attention_desc(pkg, b, 0, 2 * hd, 0, 2 * hd)) > 0
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@FORMATS
def test_attention_of_short_sequences_in_a_batch_with_no_room_for_them(ctx, pkg, dtype, cache):
    """max_rows * seqs rows: the sizes say that every sequence has 20 rows, row_start says otherwise."""
    b = Batch([20, 5, 20], [90, 300, 20], 16, 4, 2, 64, dtype, cache, seed=106, tail_rows=15)
    assert b.seqs * b.max_rows == b.tokens
    b.fill()
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    assert_attention(b, q, attention(ctx, pkg, b, q))
    b.free()


@FORMATS
@pytest.mark.parametrize("n", [16, 90])
def test_attention_keys_of_nan_behind_a_row(ctx, pkg, dtype, cache, n):
    """A key that a row does not see may be NaN: the rows before it have the same bits as without."""
    b = Batch([n], [200], 16, 2, 2, 64, dtype, cache, seed=107)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(2 * 64)
    want = attention(ctx, pkg, b, q)
    p, at = b.table[0, 199 // 16], 199 % 16
    k = b.k.copy()
    k[p, :, at] = STALE8 if cache == E4M3 else STALE16[dtype]
    ctx.upload(b.dev["k"], k)
    got = attention(ctx, pkg, b, q)
    assert np.array_equal(got[: n - 1], want[: n - 1])
    assert np.isnan(widen(got[n - 1], dtype)).all()
    b.free()


@FORMATS
def test_pages_past_four_gigabytes(ctx, pkg, dtype, cache):
    """A pool of over 2^32 bytes of K: append to and attend over its last pages."""
    each = 1 if cache == E4M3 else 2
    b = Batch([20, 1], [20, 40], 64, 4, 2, 128, dtype, cache, seed=61)
    small = b.num_pages
    page_bytes = b.nkv * b.page * b.hd * each
    b.fill([0, 39])
    total = 2 ** 32 // page_bytes + small
    b.upload(ctx)
    for name in ("k", "v"):
        b.dev[name].free()
        b.dev[name] = ctx.alloc(total * page_bytes)
        ctx.upload(b.dev[name], getattr(b, name), (total - small) * page_bytes)
    if cache == E4M3:
        for name in ("k_scale", "v_scale"):
            b.dev[name].free()
            b.dev[name] = ctx.to_device(np.concatenate([np.ones((total - small, b.nkv), np.float32), getattr(b, name)]))
    table = np.where((b.table >= 0) & (b.table < small), b.table + total - small, b.table).astype(np.int32)
    b.dev["table"].free()
    b.dev["table"] = ctx.to_device(table)

    def read():
        out = {n: ctx.download(b.dev[n], getattr(b, n).shape, getattr(b, n).dtype, (total - small) * page_bytes) for n in ("k", "v")}
        if cache == E4M3:
            out.update({n: ctx.download(b.dev[n], (small, b.nkv), np.float32, (total - small) * b.nkv * 4) for n in ("k_scale", "v_scale")})
        return out

    before, x = read(), _inputs(b)
    q = append(ctx, pkg, b, *x, num_pages=total)
    after = read()
    _check_append(b, before, after, q, x)
    rows = b.random_rows(4 * 128)
    assert_attention(b, rows, attention(ctx, pkg, b, rows, num_pages=total), **after)
    b.free()


# ------------------------------------------------- the operators together

@FORMATS
def test_prompts_then_steps(ctx, pkg, dtype, cache):
    """mrope rows -> append -> attention, as a layer loop runs them: three prompts in one batch,
    one of them in two parts, then steps of one token each; after every batch the attention over
    the cache as it is on the device, and at the end the whole cache against its definition."""
    nq, nkv, hd, page, sec = 8, 4, 128, 16, (24, 20, 20)
    plan = [[50, 7, 1], [30, 1, 1], [1, 1, 1], [1, 1, 1], [1, 0, 1]]
    done, rng = [0, 0, 0], np.random.default_rng(71)
    total = [sum(x) for x in zip(*plan)]
    pool = Batch([0] * 3, total, page, nq, nkv, hd, dtype, cache, seed=72)
    pool.stale()
    pool.upload(ctx)
    w = [(1.0 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    for n in plan:
        done = [d + k for d, k in zip(done, n)]
        b = Batch(n, done, page, nq, nkv, hd, dtype, cache, seed=73 + done[0])
        b.table, b.ldtable, b.num_pages = pool.table, pool.ldtable, pool.num_pages
        b.k, b.v, b.k_scale, b.v_scale = pool.k, pool.v, pool.k_scale, pool.v_scale
        b.dev = dict(pool.dev, row_start=ctx.to_device(b.row_start), kv_len=ctx.to_device(b.kv_len))
        at = np.concatenate([np.arange(d - k, d) for d, k in zip(done, n)] + [np.zeros(b.tokens - sum(n), np.int64)])
        pos = np.stack([at, at // 3, at % 7])
        c, s = _mrope(ctx, pkg, dtype, pos, hd, sec, True)
        qkv = b.random_rows((nq + 2 * nkv) * hd)
        before = b.read(ctx)
        q = append(ctx, pkg, b, qkv, *w, c, s)
        after = b.read(ctx)
        _check_append(b, before, after, q, (qkv, *w, c, s))
        assert_attention(b, q, attention(ctx, pkg, b, q), **after)
        b.dev["row_start"].free()
        b.dev["kv_len"].free()
    pool.free()


def test_graph_replays_follow_the_lengths(ctx, pkg):
    """A captured append + attention, replayed while lengths, rows and tables change on the device,
    with eager calls between, gives the eager results."""
    nq, nkv, hd, page, seqs = 8, 4, 128, 16, 3
    b = Batch([1] * seqs, [600, 300, 40], page, nq, nkv, hd, F16, E4M3, seed=81, tail_rows=0, extra_slots=2, spare_pages=70)
    b.stale()  # every page holds something: the tables below name any of them
    b.k, b.v = (e4m3_codes(20.0 * b.rng.standard_normal(x)) for x in b.shapes())
    b.k_scale, b.v_scale = (np.full((b.num_pages, nkv), x, np.float32) for x in (0.0625, 0.03125))
    b.upload(ctx)
    qkv, qn, kn, c, s = _inputs(b)
    d_in = [ctx.to_device(x) for x in (qkv, qn, kn, c, s)]
    d_q, d_o = ctx.alloc(seqs * nq * hd * 2), ctx.alloc(seqs * nq * hd * 2)
    kv = b.kv(pkg, max_len=b.ldtable * page)
    ap = pkg.KvAppendDesc(dtype=F16, flags=0, tokens=seqs, nqh=nq, eps=paged.EPS, qkv=int(d_in[0]), ldqkv=qkv.shape[1], qn_w=int(d_in[1]),
                          kn_w=int(d_in[2]), cos=int(d_in[3]), sin=int(d_in[4]), q_out=int(d_q), ldq=nq * hd, kv=ctypes.pointer(kv))
    at = pkg.PagedAttentionDesc(dtype=F16, flags=0, tokens=seqs, nqh=nq, q=int(d_q), ldq=nq * hd, kv=ctypes.pointer(kv), out=int(d_o), ldo=nq * hd,
                                workspace=None, workspace_bytes=0)
    size = pkg.attention_paged_workspace(at)
    ws = ctx.alloc(max(16, size))
    at.workspace, at.workspace_bytes = int(ws), size
    with Capture(ctx.stream) as cap:
        ctx.kv_append(ap)
        ctx.attention_paged(at)
    try:
        for lens, start in (([600, 300, 40], [0, 1, 2, 3]), ([17, 620, 1], [0, 1, 2, 3]), ([640, 16, 33], [0, 1, 1, 2]), ([5, 6, 7], [0, 0, 0, 0]),
                            ([601, 301, 41], [0, 1, 2, 3])):
            table = b.rng.permutation(b.num_pages)[: seqs * b.ldtable].reshape(seqs, -1).astype(np.int32)
            ctx.upload(b.dev["table"], table)
            ctx.upload(b.dev["kv_len"], np.array(lens, np.int32))
            ctx.upload(b.dev["row_start"], np.array(start, np.int32))
            state = b.read(ctx)
            outs = []
            for go in (cap.replay, lambda: (ctx.kv_append(ap), ctx.attention_paged(at), ctx.sync())):
                for n, a in state.items():
                    ctx.upload(b.dev[n], a)
                ctx.upload(d_o, np.full(seqs * nq * hd, 0x3C01, np.uint16))
                go()
                outs.append((ctx.download(d_o, (seqs, nq * hd)), b.read(ctx)))
            assert np.array_equal(outs[0][0], outs[1][0]) and all(np.array_equal(outs[0][1][k], outs[1][1][k]) for k in state)
            assert (outs[0][0][start[-1]:] == 0x3C01).all()
            b.table, b.row_start, b.n, b.len = table, np.array(start), list(np.diff(start)), lens
            got = ctx.download(d_q, (seqs, nq * hd))
            assert_attention(b, got, outs[0][0], **outs[0][1])
            if start[-1] == 0:
                assert all(np.array_equal(outs[0][1][k], state[k]) for k in state)
    finally:
        cap.close()
    for x in d_in + [d_q, d_o, ws]:
        x.free()
    b.free()


def test_graph_replays_of_prompts(ctx, pkg):
    """A captured attention over bounds of 120 rows and 3000 keys, replayed on other batches with eager
    calls between: the eager results."""
    b = Batch([120, 60, 1], [3000, 60, 900], 32, 4, 2, 128, BF16, BF16, seed=83, tail_rows=40)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(4 * 128)
    dq, do = ctx.to_device(q), ctx.alloc(q.nbytes)
    d = paged.attention_desc(pkg, b, dq, q.shape[1], do, q.shape[1])
    size = pkg.attention_paged_workspace(d)
    assert size  # split: the join is captured too
    ws = ctx.to_device(np.full(size, 0xFF, np.uint8))
    d.workspace, d.workspace_bytes = int(ws), size
    with Capture(ctx.stream) as cap:
        ctx.attention_paged(d)
    try:
        for n, lens in (([120, 60, 1], [3000, 60, 900]), ([1, 1, 1], [2999, 1, 33]), ([16, 17, 120], [16, 60, 900]), ([0, 0, 0], [3000, 0, 5]),
                        ([90, 0, 120], [1025, 60, 120]), ([120, 60, 1], [3000, 60, 900])):
            b.n, b.len = n, lens
            b.row_start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
            ctx.upload(b.dev["row_start"], b.row_start)
            ctx.upload(b.dev["kv_len"], np.array(lens, np.int32))
            outs = []
            for go in (cap.replay, lambda: (ctx.attention_paged(d), ctx.sync())):
                ctx.upload(do, np.full(q.shape, 0x3C01, np.uint16))
                go()
                outs.append(ctx.download(do, q.shape))
            assert np.array_equal(*outs)
            assert_attention(b, q, outs[0], rows=(0, 1, 16, 59, 89, 119))
    finally:
        cap.close()
    for x in (dq, do, ws):
        x.free()
    b.free()


def test_two_contexts_at_once(ctx, pkg):
    """Two contexts' calls on one GPU at the same time, a workspace each: each gets its own result."""
    b = Batch([1, 1], [5000, 3000], 32, 8, 4, 128, F16, F16, seed=91)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(8 * 128)
    want = attention(ctx, pkg, b, q)
    with pkg.Context(0) as other:
        work = []
        for c in (ctx, other):
            dq, do = ctx.to_device(q), ctx.to_device(np.zeros_like(q))
            d = paged.attention_desc(pkg, b, dq, q.shape[1], do, q.shape[1])
            size = pkg.attention_paged_workspace(d)
            ws = ctx.alloc(max(16, size))
            d.workspace, d.workspace_bytes = int(ws), size
            work.append((c, d, do, (dq, do, ws)))
        for _ in range(20):
            for c, d, _, _ in work:
                c.attention_paged(d)
        for c, _, _, _ in work:
            c.sync()
        n = b.row_start[-1]
        for _, _, do, bufs in work:
            assert np.array_equal(ctx.download(do, q.shape)[:n], want[:n])
            for x in bufs:
                x.free()
    b.free()


def test_nothing_to_do(ctx, pkg):
    """No rows, no sequences, no bound: nothing is written, no buffer is needed."""
    b = Batch([2], [20], 16, 4, 2, 64, F16, F16, seed=95)
    b.fill()
    b.upload(ctx)
    q = b.random_rows(4 * 64)
    for kw in (dict(seqs=0), dict(max_rows=0)):
        assert (attention(ctx, pkg, b, q, **kw) == 0x3C01).all()
    got = attention(ctx, pkg, b, q, max_len=0)  # no key: zeros
    assert (got[:2] == 0).all() and (got[2:] == 0x3C01).all()
    before = b.read(ctx)
    x = _inputs(b)
    append(ctx, pkg, b, *x, max_rows=0)
    append(ctx, pkg, b, *x, max_len=0)
    after = b.read(ctx)
    assert all(np.array_equal(before[n], after[n]) for n in before)
    d = pkg.MropeDesc(dtype=F16, flags=0, tokens=0, hd=64, axes=1, sec0=32, theta=1e4, pos=16, ldpos=0, cos=16, sin=16)
    ctx.mrope_rows(d)
    assert hip().hipStreamSynchronize(ctypes.c_void_p(ctx.stream)) == 0
    b.free()

"""qa_attention_paged_window for the tests: the call, and the definition in 64 bits."""
from __future__ import annotations

import ctypes

import numpy as np

from conftest import _attention_bound_rows, ulp16
from paged import BF16, E4M3, STALE8, STALE16, widen


def window_desc(pkg, b, q, ldq, out, ldo, window, sinks, **kv):
    return pkg.PagedWindowDesc(dtype=b.dtype, flags=0, tokens=b.tokens, nqh=b.nq, q=int(q), ldq=ldq, kv=ctypes.pointer(b.kv(pkg, **kv)),
                               out=int(out), ldo=ldo, window=window, sinks=sinks, workspace=None, workspace_bytes=0)


def window_attention(ctx, pkg, b, q, window, sinks, pad=8, out0=0x3C01, **kv):
    """qa_attention_paged_window of q [tokens, nq hd]: out rows."""
    ld = q.shape[1] + pad
    dq, do = ctx.to_device(np.pad(q, ((0, 0), (0, pad)))), ctx.to_device(np.full((b.tokens, ld), out0, np.uint16))
    d = window_desc(pkg, b, dq, ld, do, ld, window, sinks, **kv)
    size = pkg.attention_paged_window_workspace(d)
    ws = ctx.to_device(np.full(size + 64, 0xFF, np.uint8))  # NaN: nothing may be read before it is written
    if size:
        d.workspace, d.workspace_bytes = int(ws), size
    ctx.attention_paged_window(d)
    out = ctx.download(do, (b.tokens, ld))
    assert (ctx.download(ws, (size + 64,), np.uint8)[size:] == 0xFF).all() and (out[:, q.shape[1]:] == out0).all()
    for x in (dq, do, ws):
        x.free()
    return np.ascontiguousarray(out[:, : q.shape[1]])


def visible(m, n, rows, window, sinks):
    """[rows, m]: the keys that rows (of n, behind m - n) see."""
    p = m - n + np.asarray(rows)[:, None]
    j = np.arange(m)[None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def spoil_unseen(b, window, sinks, entries=True):
    """What no row of a sequence sees becomes NaN, and pages of which it sees nothing become none, other sequences' or
    pages of NaN with NaN scales, as the table says."""
    r = np.random.default_rng(b.tokens)
    for s in range(b.seqs):
        m, n = b.len[s], b.n[s]
        seen = visible(m, n, range(n), window, sinks).any(0) if n and m else np.zeros(m, bool)
        for i in range(-(-m // b.page)):
            p, at = b.table[s, i], np.arange(i * b.page, min(m, (i + 1) * b.page))
            if not 0 <= p < b.num_pages:
                continue
            hide = np.ones(b.page, bool)
            hide[at[seen[at]] - i * b.page] = False
            b.k[p][:, hide] = STALE8 if b.cache == E4M3 else STALE16[b.dtype]
            b.v[p][:, :, hide] = STALE8 if b.cache == E4M3 else STALE16[b.dtype]
            if hide.all():
                if b.cache == E4M3:
                    b.k_scale[p] = b.v_scale[p] = np.nan
                if entries:
                    b.table[s, i] = r.choice(np.array([p, -1, -9, b.num_pages, 2 ** 31 - 1]))


def assert_window(b, q, got, window, sinks, out0=0x3C01, rows=None, seqs=None, **cache):
    """paged.assert_attention with the window's mask: every row within the bound of conftest._attention_bound_rows and half
    a step of the output; rows without keys zeros, rows of no sequence what they were."""
    assert (got[b.row_start[-1]:] == out0).all()
    for s in range(b.seqs) if seqs is None else seqs:
        K, V, on = b.keys(s, **cache)
        r0, n, m = b.row_start[s], b.n[s], b.len[s]
        pick = range(n) if rows is None else [r for r in rows if r < n]
        if not pick:
            continue
        vis = visible(m, n, pick, window, sinks) & on[None]
        K, V = (np.where(vis.any(0)[None, :, None], x, 0.0) for x in (K, V))  # what nobody sees may be NaN
        full = vis.any(1)
        x = widen(q[r0:r0 + n][pick], b.dtype).reshape(len(pick), b.nq, b.hd)
        y = widen(got[r0:r0 + n][pick], b.dtype).reshape(len(pick), b.nq, b.hd)
        assert (got[r0:r0 + n][pick][~full] & 0x7FFF == 0).all()
        if not full.any():
            continue
        for h in range(b.nq):
            k, v = K[h * b.nkv // b.nq], V[h * b.nkv // b.nq]
            sc = np.where(vis[full], x[full, h] @ k.T / np.sqrt(b.hd), -np.inf)
            p = np.exp(sc - sc.max(1, keepdims=True))
            want = p @ v / p.sum(1, keepdims=True)
            bound = _attention_bound_rows(x[full, h], k, v, vis[full], BF16 if b.cache == E4M3 else b.dtype, "split")
            bound = bound + ulp16(np.abs(want) + bound, b.dtype) / 2
            err = np.abs(y[full, h] - want)
            assert np.isfinite(err).all() and (err <= bound).all(), (s, h, float((err / bound).max()))

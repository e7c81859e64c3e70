"""A packed batch over a paged cache for the tests of qa_kv_append and
qa_attention_paged: random pages, tables and rows, and the operators' definition
in 64 bits.  E4M3 is restated here on numpy (`e4m3_codes`, `e4m3_values`)."""
from __future__ import annotations

import ctypes

import numpy as np

from conftest import _attention_bound_rows, ulp16

F16, BF16, E4M3 = 0, 1, 2
EPS = 1e-6
STALE16 = {F16: 0x7E55, BF16: 0x7FD5}  # NaN: what unused slots hold
STALE8 = 0x7F


def widen(bits, dtype):
    """16-bit bits as float64."""
    if dtype == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def narrow(x, dtype):
    """float64 to the nearest 16-bit value's bits (x is near no tie of the double rounding in these tests' inputs)."""
    x = np.asarray(x, np.float32)
    if dtype == F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def e4m3_values(codes):
    c = codes.astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, np.ldexp(8.0 + m, e - 10), np.ldexp(m * 1.0, -9))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return np.where(c & 0x80, -v, v)


def e4m3_step(x):
    """Spacing of e4m3 at |x|."""
    return np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)


def e4m3_codes(x):
    """float64 (|x| <= 448 after saturation) to the nearest e4m3, ties to even, NaN kept."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    step = e4m3_step(a)
    r = np.round(a / step) * step  # numpy rounds halves to even
    e = np.floor(np.log2(np.maximum(r, 2.0 ** -6))).astype(np.int64)
    code = np.where(r < 2.0 ** -6, np.round(r * 512).astype(np.int64), ((e + 7) << 3) + (np.round(r / np.exp2(e - 3.0)).astype(np.int64) & 7))
    code = np.where(np.isnan(x), 0x7F, code)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def scale_for(amax):
    """The least power of two p with amax <= 448 p, in [2^-110, 2^120]."""
    amax = np.asarray(amax, np.float64)
    e = np.ceil(np.log2(np.maximum(amax, 2.0 ** -130) / 448.0))
    return np.exp2(np.clip(e, -110, 120))


class Batch:
    """n[s] new rows and len[s] keys of each sequence, pages in random places."""

    def __init__(self, n, lens, page, nq, nkv, hd, dtype, cache, seed, tail_rows=2, spare_pages=2, extra_slots=2):
        self.n, self.len = list(n), list(lens)
        self.page, self.nq, self.nkv, self.hd, self.dtype, self.cache = page, nq, nkv, hd, dtype, cache
        self.rng = np.random.default_rng(seed)
        self.seqs = len(self.n)
        self.row_start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.tokens = int(self.row_start[-1]) + tail_rows  # rows behind the last sequence
        self.kv_len = np.array(self.len, np.int32)
        pages = [-(-k // page) for k in self.len]
        self.num_pages = sum(pages) + spare_pages
        order = self.rng.permutation(self.num_pages)
        self.ldtable = max(pages + [0]) + extra_slots
        # entries that no key needs are no pages at all, or other sequences'
        self.table = self.rng.choice(np.array([-1, -7, 2 ** 31 - 1, 0, self.num_pages - 1]), (self.seqs, self.ldtable)).astype(np.int32)
        at = 0
        for s, k in enumerate(pages):
            self.table[s, :k] = order[at:at + k]
            at += k
        self.max_rows, self.max_len = max(self.n + [0]), max(self.len + [0])
        self.k = self.v = self.k_scale = self.v_scale = None

    @classmethod
    def shared(cls, n, lens, *args, **kw):
        """Many sequences over one's pages: each table names the pages of the longest."""
        b = cls([0], [max(lens)], *args, tail_rows=0, **kw)
        b.fill()
        b.n, b.len, b.seqs = list(n), list(lens), len(n)
        b.row_start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        b.tokens, b.kv_len = int(b.row_start[-1]) + 2, np.array(b.len, np.int32)
        b.table = np.tile(b.table, (b.seqs, 1))
        b.max_rows = max(n)
        return b

    def shapes(self):
        return (self.num_pages, self.nkv, self.page, self.hd), (self.num_pages, self.nkv, self.hd, self.page)

    def stale(self):
        """A cache of which nothing is written yet."""
        ks, vs = self.shapes()
        if self.cache == E4M3:
            self.k, self.v = np.full(ks, STALE8, np.uint8), np.full(vs, STALE8, np.uint8)
            self.k_scale, self.v_scale = (np.full((self.num_pages, self.nkv), np.nan, np.float32) for _ in range(2))
        else:
            self.k, self.v = np.full(ks, STALE16[self.dtype], np.uint16), np.full(vs, STALE16[self.dtype], np.uint16)

    def fill(self, counts=None, kstd=1.0, vstd=0.6, pow2=True):
        """Keys 0 .. counts[s] - 1 of each sequence (all of them by default) random, the rest stale."""
        counts = self.len if counts is None else counts
        self.stale()
        for s, count in enumerate(counts):
            for i in range(-(-count // self.page)):
                p, m = self.table[s, i], min(self.page, count - i * self.page)
                if not 0 <= p < self.num_pages:
                    continue
                k = kstd * self.rng.standard_normal((self.nkv, m, self.hd))
                v = vstd * self.rng.standard_normal((self.nkv, self.hd, m))
                if self.cache == E4M3:
                    ks, vs = scale_for(np.abs(k).max((1, 2))), scale_for(np.abs(v).max((1, 2)))
                    if not pow2:
                        ks, vs = (np.float32(x * self.rng.uniform(1.0, 1.9, self.nkv)).astype(np.float64) for x in (ks, vs))
                    self.k_scale[p], self.v_scale[p] = ks, vs
                    self.k[p, :, :m], self.v[p, :, :, :m] = e4m3_codes(k / ks[:, None, None]), e4m3_codes(v / vs[:, None, None])
                else:
                    self.k[p, :, :m], self.v[p, :, :, :m] = narrow(k, self.dtype), narrow(v, self.dtype)

    def random_rows(self, width, std=1.0):
        return narrow(std * self.rng.standard_normal((self.tokens, width)), self.dtype)

    def keys(self, s, k=None, v=None, k_scale=None, v_scale=None):
        """K, V [nkv, len, hd] of sequence s in 64 bits and which keys there are (their page is one)."""
        k, v = (self.k if k is None else k), (self.v if v is None else v)
        k_scale, v_scale = (self.k_scale if k_scale is None else k_scale), (self.v_scale if v_scale is None else v_scale)
        m = self.len[s]
        K, V, on = np.zeros((self.nkv, m, self.hd)), np.zeros((self.nkv, m, self.hd)), np.zeros(m, bool)
        for i in range(-(-m // self.page)):
            p, a, b = self.table[s, i], i * self.page, min(m, (i + 1) * self.page)
            if not 0 <= p < self.num_pages:
                continue
            on[a:b] = True
            if self.cache == E4M3:
                K[:, a:b] = e4m3_values(k[p, :, : b - a]) * k_scale[p].astype(np.float64)[:, None, None]
                V[:, a:b] = (e4m3_values(v[p, :, :, : b - a]) * v_scale[p].astype(np.float64)[:, None, None]).transpose(0, 2, 1)
            else:
                K[:, a:b], V[:, a:b] = widen(k[p, :, : b - a], self.dtype), widen(v[p, :, :, : b - a], self.dtype).transpose(0, 2, 1)
        return K, V, on

    # ---- device side

    def upload(self, ctx):
        self.dev = {n: ctx.to_device(getattr(self, n)) for n in ("table", "row_start", "kv_len", "k", "v")}
        if self.cache == E4M3:
            self.dev.update(k_scale=ctx.to_device(self.k_scale), v_scale=ctx.to_device(self.v_scale))

    def kv(self, pkg, **kw):
        d = {n: int(b) for n, b in self.dev.items()}
        d.update(dtype=self.cache, page=self.page, nkvh=self.nkv, hd=self.hd, num_pages=self.num_pages, ldtable=self.ldtable,
                 seqs=self.seqs, max_rows=self.max_rows, max_len=self.max_len)
        return pkg.PagedKV(**{**d, **kw})

    def read(self, ctx):
        """The cache as it is on the device."""
        out = {n: ctx.download(self.dev[n], getattr(self, n).shape, getattr(self, n).dtype)
               for n in ("k", "v") + (("k_scale", "v_scale") if self.cache == E4M3 else ())}
        return out

    def free(self):
        for b in self.dev.values():
            b.free()


def append(ctx, pkg, b, qkv, qn, kn, cos, sin, pad=8, q0=0x1234, **kv):
    """qa_kv_append of qkv [tokens, width] into b's pages: q rows [tokens, nq hd]."""
    width, ldq = qkv.shape[1], b.nq * b.hd + pad
    bufs = [ctx.to_device(a) for a in (np.pad(qkv, ((0, 0), (0, pad))), qn, kn, cos, sin, np.full((b.tokens, ldq), q0, np.uint16))]
    q, w, w2, c, s, o = bufs
    ctx.kv_append(pkg.KvAppendDesc(dtype=b.dtype, flags=0, tokens=b.tokens, nqh=b.nq, eps=EPS, qkv=int(q), ldqkv=width + pad, qn_w=int(w),
                                   kn_w=int(w2), cos=int(c), sin=int(s), q_out=int(o), ldq=ldq, kv=ctypes.pointer(b.kv(pkg, **kv))))
    out = ctx.download(o, (b.tokens, ldq))
    for x in bufs:
        x.free()
    assert (out[:, b.nq * b.hd:] == q0).all()  # the stride's padding is not written
    return np.ascontiguousarray(out[:, : b.nq * b.hd])


def attention_desc(pkg, b, q, ldq, out, ldo, **kv):
    return pkg.PagedAttentionDesc(dtype=b.dtype, flags=0, tokens=b.tokens, nqh=b.nq, q=int(q), ldq=ldq, kv=ctypes.pointer(b.kv(pkg, **kv)),
                                  out=int(out), ldo=ldo, workspace=None, workspace_bytes=0)


def attention(ctx, pkg, b, q, pad=8, out0=0x3C01, **kv):
    """qa_attention_paged of q [tokens, nq hd]: out rows."""
    ld = q.shape[1] + pad
    dq, do = ctx.to_device(np.pad(q, ((0, 0), (0, pad)))), ctx.to_device(np.full((b.tokens, ld), out0, np.uint16))
    d = attention_desc(pkg, b, dq, ld, do, ld, **kv)
    size = pkg.attention_paged_workspace(d)
    ws = ctx.to_device(np.full((size + 15) // 4 * 4, 0xFF, np.uint8)) if size else None  # NaN: nothing may be read before it is written
    if ws is not None:
        d.workspace, d.workspace_bytes = int(ws), size
    ctx.attention_paged(d)
    out = ctx.download(do, (b.tokens, ld))
    for x in (dq, do, ws):
        if x is not None:
            x.free()
    assert (out[:, q.shape[1]:] == out0).all()
    return np.ascontiguousarray(out[:, : q.shape[1]])


def assert_attention(b, q, got, out0=0x3C01, rows=None, seqs=None, **cache):
    """Every row within the derived bound of the definition in 64 bits: the f32
    score and accumulation errors and the two-term probabilities of
    conftest._attention_bound_rows (bf16 terms over an e4m3 cache), and half a
    step of the output.  Rows without keys are zeros, rows of no sequence what
    they were.  rows, seqs: those to look at (all of them)."""
    assert (got[b.row_start[-1]:] == out0).all()
    worst = 0.0
    for s in range(b.seqs) if seqs is None else seqs:
        K, V, on = b.keys(s, **cache)
        r0, n, m = b.row_start[s], b.n[s], b.len[s]
        pick = range(n) if rows is None else [r for r in rows if r < n]
        if not pick:
            continue
        vis = (np.arange(m)[None] <= (m - n + np.array(pick))[:, None]) & on[None]
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
            worst = max(worst, float((err / bound).max()))
    return worst

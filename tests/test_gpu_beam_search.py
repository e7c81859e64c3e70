"""A beam search over paged caches, every call of it as it would be used: qa_mrope_rows, qa_kv_append and
qa_attention_paged_window over two layers, qa_linear to logits, qa_beam_select, qa_pages_fork; then compaction and a move to
another pool, and the search goes on.  Checked at every step against a search in 64 bits that keeps whole keys and values for
each beam: the same parents, tokens and lengths, attention within paged_window's bound."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from conftest import _attention_bound_rows, ulp16
from hipgraph import Capture
from paged import BF16, E4M3, EPS, F16, e4m3_values, narrow, widen
from paged_window import visible

pytestmark = pytest.mark.gpu

PAGE, NQ, NKV, HD, LAYERS, VOCAB = 16, 4, 2, 64, 2, 1000
GROUPS, BEAMS = 3, 4
WINDOW, SINKS = 40, 5


class Search:
    """The device's side of a search, step by step."""

    def __init__(self, ctx, pkg, dtype, cache, num_pages, width, seed):
        self.ctx, self.pkg, self.dtype, self.cache, self.num_pages, self.width = ctx, pkg, dtype, cache, num_pages, width
        r = np.random.default_rng(seed)
        self.S = GROUPS * BEAMS
        es = 1 if cache == E4M3 else 2
        self.sizes = [NKV * PAGE * HD * es] * 2 + ([NKV * 4] * 2 if cache == E4M3 else [])
        self.pool(num_pages)
        put = ctx.to_device
        self.tables = [put(np.full((self.S, width), -1, np.int32)) for _ in range(2)]
        self.lens = [put(np.zeros(self.S, np.int32)) for _ in range(2)]
        self.refs, self.missing = put(np.zeros(num_pages, np.int32)), put(np.zeros(1, np.int32))
        self.grow = put(np.ones(self.S, np.int32))
        self.row_start = put(np.arange(self.S + 1, dtype=np.int32))
        self.w = put(narrow(r.standard_normal((VOCAB, NQ * HD)) * 0.6, dtype))
        self.qn, self.kn = (put((1 + 0.1 * r.standard_normal(HD)).astype(np.float32)) for _ in range(2))
        self.out, self.q = (put(np.zeros((self.S, NQ * HD), np.uint16)) for _ in range(2))
        self.cos, self.sin = (put(np.zeros((self.S, HD), np.float32)) for _ in range(2))
        self.pos = put(np.zeros(self.S, np.int32))
        self.qkv = [put(np.zeros((self.S, (NQ + 2 * NKV) * HD), np.uint16)) for _ in range(LAYERS)]
        self.logits = put(np.zeros((self.S, VOCAB), np.uint16))
        self.score = [put(np.zeros(self.S, np.float32)) for _ in range(2)]
        self.done = [put(np.zeros(self.S, np.int32)) for _ in range(2)]
        self.parent, self.token = put(np.zeros(self.S, np.int32)), put(np.zeros(self.S, np.int32))
        self.turn, self.ws = 0, {}

    def pool(self, num_pages):
        self.num_pages = num_pages
        self.mem = [self.ctx.to_device(np.full(num_pages * n, 0x7F, np.uint8)) for _ in range(LAYERS) for n in self.sizes]
        self.planes = (self.pkg.PagePlane * len(self.mem))(*[(int(m), self.sizes[i % len(self.sizes)]) for i, m in enumerate(self.mem)])

    def workspace(self, d, size):
        """A buffer for each kind of call, kept (a captured call's stays where it is)."""
        kind = type(d).__name__
        if kind not in self.ws or self.ws[kind].nbytes < size:
            self.ws[kind] = self.ctx.to_device(np.full(max(size, 16), 0xFF, np.uint8))
        d.workspace, d.workspace_bytes = int(self.ws[kind]), size
        return d

    def fork(self, parent=None, keep=0):
        """tables[turn], lens[turn] -> the others; turns."""
        pkg, a, b = self.pkg, self.turn, 1 - self.turn
        d = pkg.PagesForkDesc(flags=keep, page=PAGE, num_pages=self.num_pages, planes=self.planes, nplanes=len(self.mem), refs=int(self.refs), src_seqs=self.S,
                              seqs=self.S, ldtable=self.width, src_table=int(self.tables[a]), src_len=int(self.lens[a]), parent=int(parent or self.parent),
                              table=int(self.tables[b]), len=int(self.lens[b]), grow=int(self.grow), window=WINDOW, sinks=SINKS, missing=int(self.missing))
        self.ctx.pages_fork(self.workspace(d, pkg.pages_fork_workspace(d)))
        self.turn = b

    def kv(self, layer):
        m = self.mem[layer * len(self.sizes):]
        e4m3 = self.cache == E4M3
        return self.pkg.PagedKV(dtype=self.cache, page=PAGE, nkvh=NKV, hd=HD, num_pages=self.num_pages, k=int(m[0]), v=int(m[1]),
                                k_scale=int(m[2]) if e4m3 else None, v_scale=int(m[3]) if e4m3 else None, table=int(self.tables[self.turn]),
                                ldtable=self.width, seqs=self.S, row_start=int(self.row_start), kv_len=int(self.lens[self.turn]), max_rows=1,
                                max_len=self.width * PAGE)

    def layers(self):
        """The rows' step through the layers; logits of the last one's attention."""
        pkg, ctx = self.pkg, self.ctx
        ctx.mrope_rows(pkg.MropeDesc(dtype=self.dtype, flags=0, tokens=self.S, hd=HD, axes=1, sec0=HD // 2, sec1=0, sec2=0, theta=1e6, pos=int(self.pos),
                                     ldpos=self.S, cos=int(self.cos), sin=int(self.sin)))
        for layer in range(LAYERS):
            kv = self.kv(layer)
            ctx.kv_append(pkg.KvAppendDesc(dtype=self.dtype, flags=0, tokens=self.S, nqh=NQ, eps=EPS, qkv=int(self.qkv[layer]), ldqkv=(NQ + 2 * NKV) * HD,
                                           qn_w=int(self.qn), kn_w=int(self.kn), cos=int(self.cos), sin=int(self.sin), q_out=int(self.q), ldq=NQ * HD,
                                           kv=ctypes.pointer(kv)))
            d = pkg.PagedWindowDesc(dtype=self.dtype, flags=0, tokens=self.S, nqh=NQ, q=int(self.q), ldq=NQ * HD, kv=ctypes.pointer(kv), out=int(self.out),
                                    ldo=NQ * HD, window=WINDOW, sinks=SINKS)
            ctx.attention_paged_window(self.workspace(d, pkg.attention_paged_window_workspace(d)))
        ctx.linear(pkg.linear_desc(self.dtype, self.S, VOCAB, NQ * HD, self.out, self.w, self.logits))

    def select(self, end):
        pkg, a, b = self.pkg, self.turn, 1 - self.turn
        d = pkg.BeamDesc(dtype=self.dtype, flags=0, groups=GROUPS, beams=BEAMS, width=BEAMS, vocab=VOCAB, logits=int(self.logits), ldl=VOCAB,
                         score=int(self.score[a]), done=int(self.done[a]), end=end, parent=int(self.parent), token=int(self.token), score_out=int(self.score[b]),
                         done_out=int(self.done[b]))
        self.ctx.beam_select(self.workspace(d, pkg.beam_select_workspace(d)))

    def free(self):
        for b in list(self.ctx._bufs):
            b.free()


def _beams_want(x, score, done, end):
    out = []
    for g in range(GROUPS):
        found = []
        for b in range(g * BEAMS, (g + 1) * BEAMS):
            if not np.isfinite(score[b]):
                continue
            if done[b]:
                found.append((-score[b], b, end))
                continue
            lse = x[b].max() + np.log(np.exp(x[b] - x[b].max()).sum())
            found += [(-(score[b] + x[b, t] - lse), b, int(t)) for t in np.lexsort((np.arange(VOCAB), -x[b]))[:BEAMS]]
        out += (sorted(found) + [(np.inf, -1, -1)] * BEAMS)[:BEAMS]
    s, p, t = zip(*out)
    return np.array(p), np.array(t), -np.array(s)


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])
def test_beam_search(pkg, dtype, cache):
    with pkg.Context(0) as ctx:
        s = Search(ctx, pkg, dtype, cache, 60, 12, seed=dtype * 4 + cache)
        r = np.random.default_rng(7)
        end = 3
        # the first sequences: the first of each group, with no keys; the others are none
        ctx.upload(s.score[1], np.tile(np.array([0.0] + [-np.inf] * (BEAMS - 1), np.float32), GROUPS))
        ctx.upload(s.parent, np.where(np.arange(s.S) % BEAMS == 0, np.arange(s.S), -1).astype(np.int32))
        rows = [[[] for _ in range(s.S)] for _ in range(LAYERS)]  # each beam's (K, V) of every position, as the cache has them
        here = np.arange(s.S)
        parent = np.where(here % BEAMS == 0, here, -1)
        peak = 0
        for step in range(70):
            s.fork()
            a = s.turn
            table, length = ctx.download(s.tables[a], (s.S, s.width), np.int32), ctx.download(s.lens[a], (s.S,), np.int32)
            refs = ctx.download(s.refs, (s.num_pages,), np.int32)
            assert ctx.download(s.missing, (1,), np.int32)[0] == 0
            rows = [[list(layer[p]) if p >= 0 else [] for p in parent] for layer in rows]
            want_len = np.array([len(rows[0][i]) + 1 if parent[i] >= 0 else 0 for i in range(s.S)])
            assert np.array_equal(length, want_len)
            count = np.zeros(s.num_pages, np.int32)
            np.add.at(count, table[table >= 0], 1)
            assert np.array_equal(count, refs)
            for i in range(s.S):  # what is written next is its own; what no window reaches is given back
                if length[i]:
                    assert refs[table[i, (length[i] - 1) // PAGE]] == 1
                    first = max(0, length[i] - 1 - WINDOW + 1) // PAGE
                    assert all((table[i, j] >= 0) == (j * PAGE < length[i] and (j >= first or j * PAGE < SINKS)) for j in range(s.width))
            peak = max(peak, int((refs > 0).sum()))
            ctx.upload(s.pos, np.maximum(length - 1, 0).astype(np.int32))
            x = [narrow(1.5 * r.standard_normal((s.S, (NQ + 2 * NKV) * HD)), dtype) for _ in range(LAYERS)]
            for layer in range(LAYERS):
                ctx.upload(s.qkv[layer], x[layer])
            s.layers()
            # the appended keys and values, read back from each sequence's page
            got = [ctx.download(m, (s.num_pages * s.sizes[i % len(s.sizes)],), np.uint8) for i, m in enumerate(s.mem)]
            keys = []
            for layer in range(LAYERS):
                m = got[layer * len(s.sizes):]
                if cache == E4M3:
                    ks, vs = (y.view(np.float32).reshape(s.num_pages, NKV).astype(np.float64) for y in m[2:4])
                    K = e4m3_values(m[0].reshape(-1, NKV, PAGE, HD)) * ks[..., None, None]
                    V = (e4m3_values(m[1].reshape(-1, NKV, HD, PAGE)) * vs[..., None, None]).transpose(0, 1, 3, 2)
                else:
                    K = widen(m[0].view(np.uint16).reshape(-1, NKV, PAGE, HD), dtype)
                    V = widen(m[1].view(np.uint16).reshape(-1, NKV, HD, PAGE), dtype).transpose(0, 1, 3, 2)
                keys.append((K, V))
                for i in range(s.S):
                    if not length[i]:
                        continue
                    p, slot = table[i, (length[i] - 1) // PAGE], (length[i] - 1) % PAGE
                    rows[layer][i].append((K[p, :, slot], V[p, :, slot]))
                    v = widen(np.ascontiguousarray(x[layer][i].reshape(-1, HD)[NQ + NKV:]), dtype)
                    step_v = np.abs(v) * 2.0 ** -4 + 2.0 ** -9 if cache == E4M3 else 0.0  # half a step of e4m3, or of what its scale leaves
                    assert (np.abs(V[p, :, slot] - v) <= step_v).all()
                    if cache != E4M3 or dtype == F16:
                        # everything that the sequence sees is what its ancestors wrote (e4m3 pages may since have been rounded to a larger scale)
                        for j in np.nonzero(visible(length[i], 1, [0], WINDOW, SINKS)[0])[0]:
                            at = table[i, j // PAGE]
                            k0, v0 = rows[layer][i][j]
                            near = 2.0 ** -2 if cache == E4M3 else 0.0
                            assert (np.abs(K[at, :, j % PAGE] - k0) <= near * np.abs(k0) + near).all() and (np.abs(V[at, :, j % PAGE] - v0) <= near * np.abs(v0) + near).all()
            out, q = ctx.download(s.out, (s.S, NQ * HD)), ctx.download(s.q, (s.S, NQ * HD))
            K, V = keys[-1]
            for i in range(s.S):
                if not length[i]:
                    continue
                see = np.nonzero(visible(length[i], 1, [0], WINDOW, SINKS)[0])[0]
                k, v = (np.stack([y[table[i, j // PAGE], :, j % PAGE] for j in see], 1) for y in (K, V))  # [nkv, keys, hd]
                for h in range(NQ):
                    qh = widen(q[i:i + 1, h * HD:(h + 1) * HD], dtype)
                    kh, vh = k[h * NKV // NQ], v[h * NKV // NQ]
                    sc = qh @ kh.T / np.sqrt(HD)
                    p = np.exp(sc - sc.max())
                    want = p @ vh / p.sum()
                    bound = _attention_bound_rows(qh, kh, vh, np.ones((1, len(see)), bool), BF16 if cache == E4M3 else dtype, "split")
                    bound = bound + ulp16(np.abs(want) + bound, dtype) / 2
                    assert (np.abs(widen(out[i:i + 1, h * HD:(h + 1) * HD], dtype) - want) <= bound).all()
            s.select(end)
            score, done = ctx.download(s.score[a], (s.S,), np.float32), ctx.download(s.done[a], (s.S,), np.int32)
            parent, token = ctx.download(s.parent, (s.S,), np.int32), ctx.download(s.token, (s.S,), np.int32)
            total = ctx.download(s.score[1 - a], (s.S,), np.float32)
            p, t, v = _beams_want(widen(ctx.download(s.logits, (s.S, VOCAB)), dtype), score.astype(np.float64), done, end)
            assert np.array_equal(parent, p) and np.array_equal(token, t)
            on = p >= 0
            assert (np.abs(total[on] - v[on]) <= 1e-5 + 2.0 ** -23 * np.abs(v[on])).all()
            assert np.array_equal(ctx.download(s.done[1 - a], (s.S,), np.int32), on & (((p >= 0) & (done[np.maximum(p, 0)] != 0)) | (t == end)))
            # (select writes what the next turn reads: fork's turn comes first)
            if step == 30:
                _compact(ctx, pkg, s, table, refs)
            if step == 50:
                _move(ctx, pkg, s)
        assert peak < 60
        s.free()


def _compact(ctx, pkg, s, table, refs):
    """The sequences' pages to the front of the pool, in place: tables and references as the model has them."""
    from pages import compact_model
    d = pkg.PagesCompactDesc(flags=0, num_pages=s.num_pages, planes=s.planes, nplanes=len(s.mem), refs=int(s.refs), refs_out=int(s.refs), seqs=s.S, ldtable=s.width,
                             table=int(s.tables[s.turn]), table_out=int(s.tables[s.turn]), map=None, used=int(s.missing))
    ctx.pages_compact(s.workspace(d, pkg.pages_compact_workspace(d)))
    want = compact_model(refs, table)
    assert np.array_equal(ctx.download(s.refs, refs.shape, np.int32), want[0]) and np.array_equal(ctx.download(s.tables[s.turn], table.shape, np.int32), want[1])
    ctx.upload(s.missing, np.zeros(1, np.int32))


def _move(ctx, pkg, s):
    """All pages to a larger pool, under the same numbers."""
    old, planes, n = s.mem, s.planes, s.num_pages
    refs = ctx.download(s.refs, (n,), np.int32)
    s.pool(n + 20)
    pairs = ctx.to_device(np.repeat(np.arange(n, dtype=np.int32), 2))
    ctx.pages_copy(pkg.PagesCopyDesc(flags=0, nplanes=len(old), src=planes, src_pages=n, dst=s.planes, dst_pages=n + 20, pairs=int(pairs), npairs=n))
    s.refs = ctx.to_device(np.concatenate([refs, np.zeros(20, np.int32)]))


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4M3)], ids=["f16", "bf16-e4m3"])
def test_captured_steps(pkg, dtype, cache):
    """Two steps (their buffers take turns) in one graph, replayed: the same bits as the same steps run one by one."""
    ends = []
    for captured in (False, True):
        with pkg.Context(0) as ctx:
            s = Search(ctx, pkg, dtype, cache, 80, 12, seed=1)
            r = np.random.default_rng(2)
            ctx.upload(s.score[1], np.tile(np.array([0.0] + [-np.inf] * (BEAMS - 1), np.float32), GROUPS))
            ctx.upload(s.parent, np.where(np.arange(s.S) % BEAMS == 0, np.arange(s.S), -1).astype(np.int32))
            for layer in range(LAYERS):
                ctx.upload(s.qkv[layer], narrow(r.standard_normal((s.S, (NQ + 2 * NKV) * HD)), dtype))

            def steps():
                for _ in range(2):
                    s.fork()
                    s.layers()
                    s.select(5)
            if captured:
                steps()  # (what grows grows outside of a capture)
                with Capture(ctx.stream) as cap:
                    steps()
                for _ in range(9):
                    cap.replay()
                    ctx.download(s.logits, (s.S, VOCAB))  # the program's own work between the replays
                cap.close()
            else:
                for _ in range(10):
                    steps()
            ends.append([ctx.download(b, (b.nbytes,), np.uint8) for b in [*s.tables, *s.lens, s.refs, s.logits, s.out, *s.score, *s.done, s.parent, s.token, *s.mem]])
            s.free()
    assert all(np.array_equal(a, b) for a, b in zip(*ends))

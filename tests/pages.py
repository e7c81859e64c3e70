"""What qa_pages_fork and qa_pages_compact do, in Python, one sequence and page after the other, and a pool of
random pages for their tests."""
from __future__ import annotations

import ctypes

import numpy as np

KEEP = 1


def fork_model(refs, src_table, src_len, parent, grow, page, num_pages, window=0, sinks=0, keep=False):
    """(table, len, refs, missing, pairs of pages to copy) behind the call, from the description in qa.h."""
    refs = refs.astype(np.int64).copy()
    src_seqs, width = src_table.shape
    cap = min(width * page, 2 ** 30)
    have = [min(max(int(x), 0), cap) for x in src_len]
    ok = lambda p: 0 <= p < num_pages  # noqa: E731
    table, length, last = [], [], []
    for i, q in enumerate(parent):
        on = 0 <= q < src_seqs
        row, n = [-1] * width, have[q] if on else 0
        for j in range(width):
            reached = window <= 0 or j * page < sinks or (j + 1) * page > n - window + 1
            if on and j * page < n and reached and ok(src_table[q, j]):
                row[j] = int(src_table[q, j])
        more = max(0, int(grow[i])) if on and grow is not None else 0
        table.append(row)
        length.append((n, min(n + more, cap)))
        last.append(row[n // page] if n % page and length[i][1] > n else -1)
    before = refs.copy()
    for row in ([] if keep else src_table.tolist()):
        for p in row:
            if ok(p):
                refs[p] -= 1
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    free = [p for p in range(num_pages) if refs[p] <= 0]
    writers = {p: [i for i, x in enumerate(last) if x == p] for p in set(last) if p >= 0}
    whole = {p: refs[p] == len(w) for p, w in writers.items()}
    wanted, pairs = [], []
    for i, (n, to) in enumerate(length):
        p = last[i]
        if p >= 0 and not (whole[p] and writers[p][0] == i):
            wanted.append((i, n // page, p))
        wanted += [(i, j, None) for j in range(-(-n // page), -(-to // page))]
    if len(wanted) > len(free):
        return np.full((len(parent), width), -1, np.int32), np.zeros(len(parent), np.int32), before.astype(np.int32), len(wanted) - len(free), []
    for d, (i, j, old) in zip(free, wanted):
        table[i][j] = d
        refs[d] = 1
        if old is not None:
            refs[old] -= 1
            pairs.append((old, d))
    return (np.array(table, np.int32).reshape(len(parent), width), np.array([b for _, b in length], np.int32), refs.astype(np.int32), 0, pairs)


def compact_model(refs, table):
    """(refs, table, map, used, pairs) behind the call."""
    used = [p for p, r in enumerate(refs) if r > 0]
    n = len(used)
    gaps = [p for p in range(n) if refs[p] <= 0]
    pairs = list(zip([p for p in used if p >= n], gaps))
    name = {p: p for p in used}
    name.update(pairs)
    out = np.zeros(len(refs), np.int32)
    for p, d in name.items():
        out[d] = refs[p]
    return (out, np.array([[name.get(int(p), -1) for p in row] for row in table], np.int32).reshape(table.shape),
            np.array([name.get(p, -1) for p in range(len(refs))], np.int32), n, pairs)


class Pool:
    """Planes of random bytes on the device: bytes[i] of each page in plane i, and a page behind the last."""

    def __init__(self, ctx, pkg, num_pages, sizes, seed=0):
        r = np.random.default_rng(seed)
        self.ctx, self.num_pages, self.sizes = ctx, num_pages, list(sizes)
        self.host = [r.integers(0, 256, (num_pages + 1, n), np.uint8) for n in sizes]
        self.dev = [ctx.to_device(x) for x in self.host]
        self.planes = (pkg.PagePlane * len(self.dev))(*[(int(d), n) for d, n in zip(self.dev, self.sizes)])

    def move(self, pairs, src=None):
        """The model's planes with the pairs copied."""
        for x, y in zip(self.host, (src or self).host):
            if len(pairs):
                a, d = np.array(pairs).T
                x[d] = y[a]

    def check(self):
        for d, x in zip(self.dev, self.host):
            assert np.array_equal(self.ctx.download(d, x.shape, np.uint8), x)

    def free(self):
        for d in self.dev:
            d.free()


def _guarded(ctx, a, tail=3):
    """An int32 array on the device with `tail` numbers behind it that no call may write."""
    return ctx.to_device(np.concatenate([np.asarray(a, np.int32).ravel(), np.full(tail, 0x5A5A5A5A, np.int32)]))


def _back(ctx, buf, shape, tail=3):
    n = int(np.prod(shape))
    x = ctx.download(buf, (n + tail,), np.int32)
    assert (x[n:] == 0x5A5A5A5A).all()
    return x[:n].reshape(shape)


class Fork:
    """A qa_pages_fork call's buffers on the device."""

    def __init__(self, ctx, pkg, pool, page, refs, src_table, src_len, parent, grow, window=0, sinks=0, keep=False):
        self.ctx, self.pkg, self.pool = ctx, pkg, pool
        self.seqs, self.width = len(parent), src_table.shape[1]
        put = lambda a: _guarded(ctx, a)  # noqa: E731
        self.refs, self.src, self.len0, self.parent = put(refs), put(src_table), put(src_len), put(parent)
        self.grow = put(grow) if grow is not None else None
        self.table, self.len, self.missing = put(np.full((self.seqs, self.width), 77)), put(np.full(self.seqs, 77)), put([77])
        self.desc = pkg.PagesForkDesc(flags=KEEP if keep else 0, page=page, num_pages=pool.num_pages, planes=pool.planes, nplanes=len(pool.dev),
                                      refs=int(self.refs), src_seqs=src_table.shape[0], seqs=self.seqs, ldtable=self.width, src_table=int(self.src),
                                      src_len=int(self.len0), parent=int(self.parent), table=int(self.table), len=int(self.len),
                                      grow=int(self.grow) if self.grow else None, window=window, sinks=sinks, missing=int(self.missing))
        self.size = pkg.pages_fork_workspace(self.desc)
        self.ws = ctx.to_device(np.full(self.size + 64, 0xA5, np.uint8))
        self.desc.workspace, self.desc.workspace_bytes = int(self.ws), self.size

    def run(self):
        self.ctx.pages_fork(self.desc)
        return self

    def read(self):
        assert (self.ctx.download(self.ws, (self.size + 64,), np.uint8)[self.size:] == 0xA5).all()
        return (_back(self.ctx, self.table, (self.seqs, self.width)), _back(self.ctx, self.len, (self.seqs,)),
                _back(self.ctx, self.refs, (self.pool.num_pages,)), int(_back(self.ctx, self.missing, (1,))[0]))

    def free(self):
        for b in (self.refs, self.src, self.len0, self.parent, self.grow, self.table, self.len, self.missing, self.ws):
            if b is not None:
                b.free()


def compact(ctx, pkg, pool, refs, table, in_place=False, with_map=True):
    """qa_pages_compact: (refs, table, map, used)."""
    r, t = _guarded(ctx, refs), _guarded(ctx, table)
    ro, to = (r, t) if in_place else (_guarded(ctx, np.full(refs.shape, 77)), _guarded(ctx, np.full(table.shape, 77)))
    m, u = _guarded(ctx, np.full(refs.shape, 77)), _guarded(ctx, [77])
    d = pkg.PagesCompactDesc(flags=0, num_pages=pool.num_pages, planes=pool.planes, nplanes=len(pool.dev), refs=int(r), refs_out=int(ro),
                             seqs=table.shape[0], ldtable=table.shape[1], table=int(t), table_out=int(to), map=int(m) if with_map else None, used=int(u))
    size = pkg.pages_compact_workspace(d)
    ws = ctx.to_device(np.full(size + 64, 0xA5, np.uint8))
    d.workspace, d.workspace_bytes = int(ws), size
    ctx.pages_compact(d)
    out = (_back(ctx, ro, refs.shape), _back(ctx, to, table.shape), _back(ctx, m, refs.shape), int(_back(ctx, u, (1,))[0]))
    assert (ctx.download(ws, (size + 64,), np.uint8)[size:] == 0xA5).all()
    for b in {r, t, ro, to, m, u, ws}:
        b.free()
    return out


def random_sequences(r, seqs, page, width, num_pages, most, shared=0.5):
    """Tables of sequences of 0 .. most keys whose pages lie anywhere and are in part those of the sequence before, and
    their references."""
    order = iter(r.permutation(num_pages).tolist())
    table, length = np.full((seqs, width), -1, np.int32), []
    for s in range(seqs):
        n = int(r.integers(0, most + 1))
        cols = -(-n // page)
        same = 0
        if s and r.random() < shared:
            same = min(cols, length[-1] // page)  # full pages of the one before
        table[s, :same] = table[s - 1, :same]
        table[s, same:cols] = [next(order) for _ in range(cols - same)]
        length.append(n)
    refs = np.zeros(num_pages, np.int32)
    np.add.at(refs, table[table >= 0], 1)
    return table, np.array(length, np.int32), refs


def pairs_desc(pkg, src, dst, pairs, n):
    return pkg.PagesCopyDesc(flags=0, nplanes=len(src.dev), src=src.planes, src_pages=src.num_pages, dst=dst.planes, dst_pages=dst.num_pages,
                             pairs=ctypes.c_void_p(int(pairs)), npairs=n)

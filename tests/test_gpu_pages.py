"""qa_pages_fork, qa_pages_compact and qa_pages_copy on an MI355X against tests/pages.py: every number and every byte is
the same, what lies behind the buffers is left alone, whatever tables, lengths and parents hold."""
from __future__ import annotations

import numpy as np
import pytest

import pages
from hipgraph import Capture
from pages import Fork, Pool, compact, compact_model, fork_model, random_sequences

pytestmark = pytest.mark.gpu

SIZES = (4096, 4096, 32, 4)  # a layer's K and V pages and their scales, one of a single head


def _fork(ctx, pkg, pool, page, refs, table, length, parent, grow, **kw):
    want = fork_model(refs, table, length, parent, grow, page, pool.num_pages, **kw)
    call = Fork(ctx, pkg, pool, page, refs, table, length, parent, grow, **kw).run()
    got = call.read()
    for name, a, b in zip(("table", "len", "refs", "missing"), got, want):
        assert np.array_equal(a, b), (name, a, b)
    pool.move(want[4])
    pool.check()
    call.free()
    return want


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 4), (100, 33), (5000, 3)])
def test_fork(ctx, pkg, page, window, sinks):
    """Branches, ends and growth of sequences that share pages; several steps behind each other."""
    r = np.random.default_rng(page + window)
    pool = Pool(ctx, pkg, 400, SIZES, seed=page)
    table, length, refs = random_sequences(r, 9, page, 14, 400, 10 * page)
    for step in range(4):
        parent = r.integers(0, len(length), int(r.integers(1, 12))).astype(np.int32)
        if step == 2:
            parent[r.integers(0, len(parent))] = -1
        grow = r.choice(np.array([0, 1, 1, 1, 2, page, 2 * page + 1], np.int32), len(parent))
        table, length, refs, missing, _ = _fork(ctx, pkg, pool, page, refs, table, length, parent, grow, window=window, sinks=sinks)
        assert missing == 0
    pool.free()


@pytest.mark.parametrize("keep", [False, True])
def test_fork_shares_what_nobody_writes_on(ctx, pkg, keep):
    """Children that do not grow share the last page too; the first to go on alone later keeps it, the others copy."""
    pool = Pool(ctx, pkg, 12, SIZES, seed=3)
    refs = np.zeros(12, np.int32)
    refs[[7, 2]] = 1
    table = np.array([[7, 2, -1, -1]], np.int32)
    length = np.array([25], np.int32)
    parent = np.zeros(3, np.int32)
    table, length, refs, _, pairs = _fork(ctx, pkg, pool, 16, refs, table, length, parent, None, keep=keep)
    assert pairs == [] and refs[7] == 3 + keep and refs[2] == 3 + keep
    # two of the three write; the third holds the page as it is
    t2, l2, r2, _, pairs = _fork(ctx, pkg, pool, 16, refs, table, length, np.array([0, 1, 2], np.int32), np.array([1, 0, 4], np.int32))
    assert len(pairs) == 2
    # all that hold it write: the first keeps it
    _, _, _, _, pairs = _fork(ctx, pkg, pool, 16, refs, table, length, np.array([2, 1, 0], np.int32), np.array([1, 1, 1], np.int32))
    assert len(pairs) == 2 + keep
    pool.free()


def test_fork_gives_back(ctx, pkg):
    """No children: every page is free again, reserved ones too.  No sources: nothing but empty sequences."""
    pool = Pool(ctx, pkg, 40, SIZES, seed=4)
    r = np.random.default_rng(4)
    table, length, refs = random_sequences(r, 5, 16, 8, 40, 60)
    table[0, 7] = 39  # reserved behind its keys
    refs[39] += 1
    _, _, after, _, _ = _fork(ctx, pkg, pool, 16, refs, table, length, np.zeros(0, np.int32), np.zeros(0, np.int32))
    assert (after == 0).all()
    _fork(ctx, pkg, pool, 16, refs, table, length, np.array([-1, 5, 2 ** 31 - 1, -2 ** 31], np.int32), np.array([3, 3, 3, 3], np.int32))
    _fork(ctx, pkg, pool, 16, np.zeros(40, np.int32), np.zeros((0, 8), np.int32), np.zeros(0, np.int32), np.array([0, 1], np.int32), None)
    pool.free()


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("short", [1, 3])
def test_fork_without_enough_pages_changes_nothing(ctx, pkg, keep, short):
    r = np.random.default_rng(5)
    table, length, refs = random_sequences(r, 6, 16, 20, 50, 100)
    parent = np.array([0, 0, 1, 2, 3, 3, 5], np.int32)
    grow = np.array([1, 2, 40, 1, 1, 17, 33], np.int32)
    pool = Pool(ctx, pkg, 50, SIZES, seed=5)
    # take free pages away until `short` too few are left
    free = [int(p) for p in np.nonzero(refs == 0)[0]]
    while fork_model(refs, table, length, parent, grow, 16, 50, keep=keep)[3] < short:
        refs[free.pop()] = 1
    got = _fork(ctx, pkg, pool, 16, refs, table, length, parent, grow, keep=keep)
    assert got[3] == short and (got[0] == -1).all() and (got[1] == 0).all() and np.array_equal(got[2], refs)
    pool.free()


@pytest.mark.parametrize("seed", range(6))
def test_fork_of_anything(ctx, pkg, seed):
    """Entries, lengths, parents and growths out of every range."""
    r = np.random.default_rng(100 + seed)
    pool = Pool(ctx, pkg, 64, SIZES, seed=seed)
    wild = np.array([-2 ** 31, -7, -1, 0, 1, 5, 15, 16, 17, 63, 64, 100, 2 ** 31 - 1], np.int64)
    table = r.choice(np.concatenate([wild, r.integers(0, 60, 30)]), (7, 5)).astype(np.int32)
    length = r.choice(wild, 7).astype(np.int32)
    refs = np.zeros(64, np.int32)
    inside = table[(table >= 0) & (table < 64)]
    np.add.at(refs, inside, 1)
    refs[r.integers(0, 60, 4)] += 1  # held by others
    parent = r.choice(np.concatenate([wild, np.arange(7), np.arange(7)]), 11).astype(np.int32)
    grow = r.choice(wild, 11).astype(np.int32)
    for keep in (False, True):
        _fork(ctx, pkg, pool, 16, refs, table, length, parent, grow, window=int(r.choice([0, 3, 40])), sinks=int(r.choice([0, 20])), keep=keep)
        _fork(ctx, pkg, pool, 64, refs, table, length, parent, np.minimum(grow, 40), keep=keep)
    pool.free()


def test_fork_of_many(ctx, pkg):
    """More sequences than one round of the block, a pool of several rounds with its free pages behind."""
    r = np.random.default_rng(7)
    pool = Pool(ctx, pkg, 21000, (64, 4), seed=7)
    table, length, refs = random_sequences(r, 1500, 16, 14, 21000, 190, shared=0.3)
    refs[:9000] += 1  # somebody's, so that new pages lie far behind
    parent = r.integers(0, 1500, 2300).astype(np.int32)
    grow = r.integers(0, 30, 2300).astype(np.int32)
    _fork(ctx, pkg, pool, 16, refs, table, length, parent, grow)
    _fork(ctx, pkg, pool, 16, refs, table, length, np.full(2300, 3, np.int32), grow, keep=True)  # one source's children
    pool.free()


@pytest.mark.parametrize("seqs,src,width", [(1024, 1024, 2), (1025, 3, 2), (3, 1025, 2), (1, 1, 2048), (1, 1, 2049), (512, 512, 4), (512, 513, 4), (1030, 1030, 9)])
def test_fork_around_the_small_calls(ctx, pkg, seqs, src, width):
    """Both sides of the sizes that one block takes, and of those whose shared pages are counted in LDS."""
    r = np.random.default_rng(seqs + width)
    total = src * width + seqs * 3 + 50
    pool = Pool(ctx, pkg, total, (16, 4), seed=1)
    table = np.full((src, width), -1, np.int32)
    length = r.integers(0, 16 * width - 3, src).astype(np.int32)
    order = iter(r.permutation(total).tolist())
    for q in range(src):
        for j in range(-(-int(length[q]) // 16)):
            table[q, j] = table[q - 1, j] if q % 3 == 2 and length[q] == length[q - 1] else next(order)
    refs = np.zeros(total, np.int32)
    np.add.at(refs, table[table >= 0], 1)
    parent = r.integers(0, src, seqs).astype(np.int32)
    _fork(ctx, pkg, pool, 16, refs, table, length, parent, r.integers(0, 3, seqs).astype(np.int32))
    _fork(ctx, pkg, pool, 16, refs, table, length, np.full(seqs, src - 1, np.int32), np.ones(seqs, np.int32), window=20, sinks=3, keep=True)
    pool.free()


def test_fork_of_a_wide_table(ctx, pkg):
    """One sequence that takes thousands of pages at once."""
    pool = Pool(ctx, pkg, 9000, (16,), seed=8)
    refs = np.zeros(9000, np.int32)
    refs[::3] = 1
    table = np.full((2, 5000), -1, np.int32)
    table[0, :2] = [0, 3]
    _fork(ctx, pkg, pool, 16, refs, table, np.array([20, 0], np.int32), np.array([1, 0, 0], np.int32), np.array([5000, 60000, 16], np.int32), keep=True)
    pool.free()


def test_fork_at_the_limit_of_sequences(ctx, pkg):
    n = 8192
    pool = Pool(ctx, pkg, 2 * n + 10, (32,), seed=9)
    table = np.arange(n, dtype=np.int32)[:, None].repeat(3, 1)
    table[:, 1:] = -1
    refs = np.zeros(2 * n + 10, np.int32)
    refs[:n] = 1
    parent = np.random.default_rng(9).integers(0, n, n).astype(np.int32)
    _fork(ctx, pkg, pool, 16, refs, table, np.full(n, 9, np.int32), parent, np.ones(n, np.int32))
    pool.free()


def test_fork_captured(ctx, pkg):
    """Two steps that take turns, captured once: each replay is the next two steps, also with other parents."""
    r = np.random.default_rng(10)
    pool = Pool(ctx, pkg, 300, SIZES, seed=10)
    table, length, refs = random_sequences(r, 6, 16, 12, 300, 100)
    parent, grow = np.array([0, 0, 1, 3, 5, 5], np.int32), np.ones(6, np.int32)
    a = Fork(ctx, pkg, pool, 16, refs, table, length, parent, grow)
    b = Fork(ctx, pkg, pool, 16, refs, table, length, parent, grow)
    b.desc.refs, b.desc.src_table, b.desc.src_len, b.desc.table, b.desc.len = a.desc.refs, a.desc.table, a.desc.len, a.desc.src_table, a.desc.src_len
    b.desc.parent = a.desc.parent
    with Capture(ctx.stream) as cap:
        ctx.pages_fork(a.desc)
        ctx.pages_fork(b.desc)
    for step in range(4):
        if step == 2:
            parent = np.array([5, 4, 3, 2, 1, 1], np.int32)
            ctx.upload(a.parent, parent)
        cap.replay()
        for _ in range(2):
            table, length, refs, missing, pairs = fork_model(refs, table, length, parent, grow, 16, 300)
            pool.move(pairs)
            assert missing == 0
        pool.check()
        assert np.array_equal(pages._back(ctx, a.src, table.shape), table)
        assert np.array_equal(pages._back(ctx, a.len0, length.shape), length)
        assert np.array_equal(pages._back(ctx, a.refs, refs.shape), refs)
    cap.close()
    for x in (a, b):
        x.free()
    pool.free()


# ------------------------------------------------------------ compaction

@pytest.mark.parametrize("num_pages,used", [(1, 0), (1, 1), (2, 1), (7, 3), (90, 70), (1000, 0), (1000, 1000), (4096, 100), (4097, 2000), (9000, 4096), (9000, 8999),
                                            (20000, 9999)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(ctx, pkg, num_pages, used, in_place):
    r = np.random.default_rng(num_pages + used)
    pool = Pool(ctx, pkg, num_pages, (64, 1024, 4) if num_pages > 500 else SIZES, seed=used)
    refs = np.zeros(num_pages, np.int32)
    refs[r.permutation(num_pages)[:used]] = r.integers(1, 5, used)
    free = refs == 0
    refs[free] = r.choice(np.array([0, 0, 0, -2], np.int32), free.sum())
    wild = np.array([-2 ** 31, -1, num_pages, 2 ** 31 - 1], np.int64)
    table = np.concatenate([wild, r.integers(0, num_pages, 60)])[r.integers(0, 64, (9, 7))].astype(np.int32)
    want = compact_model(refs, table)
    got = compact(ctx, pkg, pool, refs, table, in_place)
    for name, a, b in zip(("refs", "table", "map", "used"), got, want):
        assert np.array_equal(a, b), name
    pool.move(want[4])
    pool.check()
    pool.free()


@pytest.mark.parametrize("num_pages,entries", [(300, 16384), (300, 16385), (4096, 1), (4097, 1), (4096, 40000)])
def test_compact_around_the_small_pools(ctx, pkg, num_pages, entries):
    """Both sides of the sizes that one block takes."""
    r = np.random.default_rng(entries)
    pool = Pool(ctx, pkg, num_pages, (48,), seed=3)
    refs = (r.random(num_pages) < 0.6).astype(np.int32)
    table = r.integers(-1, num_pages, (1, entries)).astype(np.int32)
    want = compact_model(refs, table)
    for a, b in zip(compact(ctx, pkg, pool, refs, table, True), want):
        assert np.array_equal(a, b)
    pool.move(want[4])
    pool.check()
    pool.free()


def test_compact_without_map_table_or_planes(ctx, pkg):
    pool = Pool(ctx, pkg, 50, (), seed=1)
    refs = np.zeros(50, np.int32)
    refs[[49, 3, 20]] = [2, 1, 7]
    got = compact(ctx, pkg, pool, refs, np.zeros((0, 4), np.int32), with_map=False)
    assert list(got[0][:4]) == [1, 7, 2, 0] and (got[0][3:] == 0).all()
    assert (got[2] == 77).all() and got[3] == 3
    pool.free()


# ------------------------------------------------------------ copies

@pytest.mark.parametrize("sizes", [(16,), (4,), (12, 4096), (1008, 1024, 1040), (4080, 4096, 4112, 65536), (36864, 20, 8208)])
@pytest.mark.parametrize("n", [0, 1, 37])
def test_copy(ctx, pkg, sizes, n):
    """Page sizes around the kernels' pieces; from one pool into another and back into the first."""
    r = np.random.default_rng(sum(sizes) + n)
    a, b = Pool(ctx, pkg, 50, sizes, seed=1), Pool(ctx, pkg, 41, sizes, seed=2)
    pairs = np.stack([r.integers(0, 50, n), r.permutation(41)[:n]], 1).astype(np.int32)
    p = ctx.to_device(np.concatenate([pairs.ravel(), [0, 0]]).astype(np.int32))
    ctx.pages_copy(pages.pairs_desc(pkg, a, b, p, n))
    b.move(pairs.tolist(), a)
    a.check()
    b.check()
    half = np.stack([np.arange(0, 20), np.arange(20, 40)], 1).astype(np.int32)
    q = ctx.to_device(half)
    ctx.pages_copy(pages.pairs_desc(pkg, a, a, q, 20))
    a.move(half.tolist())
    a.check()
    for x in (a, b, p, q):
        x.free()


def test_copy_of_planes_in_one_buffer(ctx, pkg):
    """Every layer's scales in one tensor: planes that begin at any 4 bytes, also from and to different ones."""
    n, layers, size = 7, 5, 12  # 84 bytes a layer
    r = np.random.default_rng(6)
    for words, sizes in ((3, (12,)), (1, (2048,)), (0, (4096,))):
        size, extra = sizes[0], 4 * words
        host = [r.integers(0, 256, 64 + layers * (n * size + extra), np.uint8) for _ in range(2)]
        dev = [ctx.to_device(x) for x in host]
        at = [[8 * k + i * (n * size + extra) for i in range(layers)] for k in range(2)]
        src, dst = ((pkg.PagePlane * layers)(*[(int(d) + o, size) for o in at[k]]) for k, d in enumerate(dev))
        pairs = np.array([[0, 6], [5, 1], [3, 3]], np.int32)
        p = ctx.to_device(pairs)
        ctx.pages_copy(pkg.PagesCopyDesc(flags=0, nplanes=layers, src=src, src_pages=n, dst=dst, dst_pages=n, pairs=int(p), npairs=3))
        for i in range(layers):
            for a, b in pairs:
                host[1][at[1][i] + b * size: at[1][i] + (b + 1) * size] = host[0][at[0][i] + a * size: at[0][i] + (a + 1) * size]
        assert np.array_equal(ctx.download(dev[1], host[1].shape, np.uint8), host[1])
        for x in dev + [p]:
            x.free()


def test_copy_leaves_out_what_is_no_page(ctx, pkg):
    a, b = Pool(ctx, pkg, 9, SIZES, seed=1), Pool(ctx, pkg, 5, SIZES, seed=2)
    pairs = np.array([[0, 5], [9, 0], [-1, 1], [3, -1], [8, 4], [2 ** 31 - 1, 2], [2, 2 ** 31 - 1], [-2 ** 31, 3]], np.int32)
    p = ctx.to_device(pairs)
    ctx.pages_copy(pages.pairs_desc(pkg, a, b, p, len(pairs)))
    b.move([(8, 4)], a)
    b.check()
    for x in (a, b, p):
        x.free()


@pytest.mark.parametrize("planes", [127, 128, 129, 300])
def test_copy_of_many_planes(ctx, pkg, planes):
    """More planes than one launch takes."""
    sizes = [(1024, 2048, 16, 4)[i % 4] for i in range(planes)]
    a, b = Pool(ctx, pkg, 6, sizes, seed=1), Pool(ctx, pkg, 6, sizes, seed=2)
    p = ctx.to_device(np.array([[5, 0], [1, 3]], np.int32))
    ctx.pages_copy(pages.pairs_desc(pkg, a, b, p, 2))
    b.move([(5, 0), (1, 3)], a)
    b.check()
    for x in (a, b, p):
        x.free()


def test_copy_past_32_bits(ctx, pkg):
    """Pages behind the first 4 GB of a plane."""
    size, n = 1 << 20, 4200
    buf = ctx.alloc(size * n)
    r = np.random.default_rng(1)
    x, y = (r.integers(0, 256, size, np.uint8) for _ in range(2))
    ctx.upload(buf, x, 5 * size)
    ctx.upload(buf, y, (n - 1) * size)
    planes = (pkg.PagePlane * 1)((int(buf), size))
    p = ctx.to_device(np.array([[5, n - 2], [n - 1, 7]], np.int32))
    ctx.pages_copy(pkg.PagesCopyDesc(flags=0, nplanes=1, src=planes, src_pages=n, dst=planes, dst_pages=n, pairs=int(p), npairs=2))
    assert np.array_equal(ctx.download(buf, (size,), np.uint8, (n - 2) * size), x)
    assert np.array_equal(ctx.download(buf, (size,), np.uint8, 7 * size), y)
    buf.free()
    p.free()

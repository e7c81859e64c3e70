"""qa_pages_fork with QA_PAGES_STRICT on an MI355X: growth that a row of the table cannot hold is a shortage, no
sequence goes on in a page that others hold, and the calls behind a shortage leave what it left."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import pages
from hipgraph import Capture
from pages import Fork, Pool, random_sequences
from pages_strict import STRICT, strict_fork, strict_model

pytestmark = pytest.mark.gpu

HD = 64


def _append(ctx, pkg, pool, seqs, width, table, length, rows, seed):
    """A qa_kv_append of `rows` rows for each sequence, over the pool's two planes (K and V of one head of 64)."""
    tokens, ld = rows * seqs, 3 * HD
    r = np.random.default_rng(seed)
    put = ctx.to_device
    qkv, q = put(r.standard_normal((tokens, ld)).astype(np.float16).view(np.uint16)), put(np.zeros((tokens, HD), np.uint16))
    ones = put(np.ones(HD, np.float32))
    cos, sin = put(np.ones((tokens, HD), np.float32)), put(np.zeros((tokens, HD), np.float32))
    start = put((rows * np.arange(seqs + 1)).astype(np.int32))
    kv = pkg.PagedKV(dtype=pkg.F16, page=16, nkvh=1, hd=HD, num_pages=pool.num_pages, k=int(pool.dev[0]), v=int(pool.dev[1]), table=int(table),
                     ldtable=width, seqs=seqs, row_start=int(start), kv_len=int(length), max_rows=rows, max_len=16 * width)
    ctx.kv_append(pkg.KvAppendDesc(dtype=pkg.F16, flags=0, tokens=tokens, nqh=1, eps=1e-6, qkv=int(qkv), ldqkv=ld, qn_w=int(ones), kn_w=int(ones),
                                   cos=int(cos), sin=int(sin), q_out=int(q), ldq=HD, kv=ctypes.pointer(kv)))
    ctx.sync()
    for x in (qkv, q, ones, cos, sin, start):
        x.free()


@pytest.mark.parametrize("length,grow", [(48, 1), (46, 3), (48, 40), (33, 16)])
def test_children_of_a_full_row(ctx, pkg, length, grow):
    """Two children of a parent whose row of the table is full, or has room for less than is to be appended: nothing is shared out,
    and the append behind it leaves the parent's pages as they are.  Full pages below the end of a row are not concerned."""
    pool = Pool(ctx, pkg, 9, (2048, 2048), seed=1)
    refs = np.zeros(9, np.int32)
    table = np.array([[4, 7, 2]], np.int32)
    refs[table[0]] = 1
    call = Fork(ctx, pkg, pool, 16, refs, table, np.array([length], np.int32), [0, 0], np.array([grow, grow], np.int32))
    call.desc.flags |= STRICT
    ctx.upload(call.missing, np.zeros(1, np.int32))
    got = call.run().read()
    short = 2 * (-(-(length + grow) // 16) - 3)
    assert got[3] == short, got
    if short:
        assert (got[0] == -1).all() and (got[1] == 0).all() and np.array_equal(got[2], refs)
        _append(ctx, pkg, pool, 2, 3, call.table, call.len, rows=grow, seed=2)
        pool.check()
    call.free()
    pool.free()


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("seqs,src,width,num_pages", [(6, 5, 6, 64), (300, 200, 12, 3000), (1300, 700, 6, 9000)])
def test_rows_that_do_not_hold_the_growth(ctx, pkg, page, keep, seqs, src, width, num_pages):
    """One launch, two, and more sequences than the block counts in LDS: no growth past a row's end, one row's, many."""
    r = np.random.default_rng(seqs + page)
    pool = Pool(ctx, pkg, num_pages, (64, 4), seed=2)
    table, length, refs = random_sequences(r, src, page, width, num_pages, (width - 2) * page)
    parent = r.integers(-1, src, seqs).astype(np.int32)
    parent[seqs // 2] = 1
    grow = r.integers(0, 2 * page + 1, seqs).astype(np.int32)
    args = (ctx, pkg, pool, page, refs, table, length, parent)
    want = strict_fork(*args, grow, keep=keep, window=40, sinks=3)
    assert want[3] == 0
    grow[seqs // 2] = width * page - length[1] + 1
    assert strict_fork(*args, grow, keep=keep)[3] == 1
    grow[r.integers(0, seqs, seqs // 2)] = 2 ** 31 - 1
    assert strict_fork(*args, grow, keep=keep)[3] > 2 ** 20
    grow[:] = 2 ** 31 - 1
    got = strict_fork(*args, grow, keep=keep)
    assert got[3] == 2 ** 31 - 1 or seqs < 300
    pool.free()


@pytest.mark.parametrize("seed", range(4))
def test_anything(ctx, pkg, seed):
    """Entries, lengths, parents and growths out of every range; rows of no pages."""
    r = np.random.default_rng(200 + seed)
    pool = Pool(ctx, pkg, 64, (64, 4), seed=seed)
    wild = np.array([-2 ** 31, -7, -1, 0, 1, 5, 15, 16, 17, 63, 64, 100, 2 ** 31 - 1], np.int64)
    table = r.choice(np.concatenate([wild, r.integers(0, 60, 30)]), (7, 5)).astype(np.int32)
    length = r.choice(wild, 7).astype(np.int32)
    refs = np.zeros(64, np.int32)
    np.add.at(refs, table[(table >= 0) & (table < 64)], 1)
    parent = r.choice(np.concatenate([wild, np.arange(7), np.arange(7)]), 11).astype(np.int32)
    grow = r.choice(wild, 11).astype(np.int32)
    for keep in (False, True):
        strict_fork(ctx, pkg, pool, 16, refs, table, length, parent, grow, window=int(r.choice([0, 40])), sinks=7, keep=keep)
        strict_fork(ctx, pkg, pool, 32, refs, table, length, parent, np.minimum(grow, 3), keep=keep)
        strict_fork(ctx, pkg, pool, 16, refs, table[:, :0], length, parent, grow, keep=keep)
    pool.free()


def test_captured(ctx, pkg):
    """A call replayed with one row more each time, by the parent's length: the one behind the row's end changes nothing."""
    pool = Pool(ctx, pkg, 20, (64,), seed=3)
    refs = np.zeros(20, np.int32)
    table = np.array([[0, 1, 2, 3]], np.int32)
    refs[:4] = 1
    call = Fork(ctx, pkg, pool, 16, refs, table, np.array([60], np.int32), [0, 0, 0], np.array([1, 1, 1], np.int32), keep=True)
    call.desc.flags |= STRICT
    with Capture(ctx.stream) as cap:
        ctx.pages_fork(call.desc)
    for length in (61, 62, 63, 64, 64, 50):
        ctx.upload(call.missing, np.zeros(1, np.int32))
        ctx.upload(call.refs, refs)
        ctx.upload(call.len0, np.array([length], np.int32))
        cap.replay()
        got = call.read()
        assert got[3] == (3 if length == 64 else 0) and (got[1] == (0 if length == 64 else length + 1)).all()
        assert (got[2] == refs).all() == (length == 64)
    cap.close()
    call.free()
    pool.free()


@pytest.mark.parametrize("before", [1, -1, 2 ** 31 - 1])
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("seqs,src,width,num_pages", [(6, 5, 6, 64), (300, 200, 12, 3000), (1300, 700, 6, 9000), (3, 0, 0, 5), (0, 5, 6, 64)])
def test_behind_a_shortage(ctx, pkg, keep, before, seqs, src, width, num_pages):
    """*missing other than 0: lengths of 0, and nothing else is written."""
    r = np.random.default_rng(seqs + src)
    pool = Pool(ctx, pkg, num_pages, (64, 4), seed=4)
    table, length, refs = random_sequences(r, src, 16, width, num_pages, max(width - 2, 0) * 16)
    length = np.asarray(length, np.int32)
    strict_fork(ctx, pkg, pool, 16, refs, table.reshape(src, width), length, r.integers(-1, max(src, 1), seqs).astype(np.int32), np.ones(seqs, np.int32),
                keep=keep, before=before)
    pool.free()


@pytest.mark.parametrize("first", [0, 1, 2])
@pytest.mark.parametrize("cause", ["pages", "rows"])
@pytest.mark.parametrize("seqs", [6, 300, 1200])
def test_captured_steps_that_take_turns(ctx, pkg, cause, first, seqs):
    """Two forks whose tables take turns, replayed past a shortage in the first step, the second or the third: tables, references and
    pages stay what the last step that went well left, rows appended behind it go nowhere, and a call to no sequences
    gives every page back."""
    width, n = 16, 6 * seqs
    r = np.random.default_rng(seqs + first)
    pool = Pool(ctx, pkg, n, (2048, 2048), seed=5)
    table, length, refs = random_sequences(r, seqs, 16, width, n, 60)
    parent, ones = r.integers(0, seqs, seqs).astype(np.int32), np.ones(seqs, np.int32)
    a = Fork(ctx, pkg, pool, 16, refs, table, length, parent, ones)
    b = Fork(ctx, pkg, pool, 16, refs, table, length, parent, ones)
    b.desc.refs, b.desc.src_table, b.desc.src_len, b.desc.table, b.desc.len = a.desc.refs, a.desc.table, a.desc.len, a.desc.src_table, a.desc.src_len
    b.desc.missing = a.desc.missing
    ctx.upload(a.missing, np.zeros(1, np.int32))
    calls, at = (a, b), ((a.table, a.len), (a.src, a.len0))  # and where each writes
    state, grow = [(np.full((seqs, width), 77, np.int32), None), (table, length)], [ones, ones]
    for x in calls:
        x.desc.flags |= STRICT
    with Capture(ctx.stream) as cap:
        for x in calls:
            ctx.pages_fork(x.desc)
    missing = [0]
    for replay in range(3):
        if first // 2 == replay:  # 7 pages for each, which the pool has not; or more than a row holds for one
            k = first % 2
            grow[k] = 112 * ones if cause == "pages" else np.where(np.arange(seqs) == 1, 16 * width + 1, 1).astype(np.int32)
            ctx.upload(calls[k].grow, grow[k])
        for k in range(2):
            t, le, refs, m, pairs = strict_model(refs, *state[1 - k], parent, grow[k], 16, n, before=missing[-1], table=state[k][0])
            pool.move(pairs)
            state[k] = (t, le)
            missing.append(m)
        cap.replay()
        assert int(pages._back(ctx, a.missing, (1,))[0]) == missing[-1]
        assert np.array_equal(pages._back(ctx, a.refs, refs.shape), refs)
        for k in range(2):
            for buf, want in zip(at[k], state[k]):
                assert np.array_equal(pages._back(ctx, buf, want.shape), want), (replay, k)
        pool.check()
        for k in range(2):
            if (state[k][1] == 0).all():
                _append(ctx, pkg, pool, seqs, width, *at[k], rows=1, seed=replay)
        pool.check()
    assert [m != 0 for m in missing[1:]] == [step >= first for step in range(6)] and len(set(missing[first + 1:])) == 1
    cap.close()
    k = 1 - first % 2  # where the last step that went well left its sequences
    count = np.zeros(n, np.int32)
    np.add.at(count, state[k][0][state[k][0] >= 0], 1)
    assert np.array_equal(count, refs) and refs.sum() > 0
    call = calls[1 - k]  # goes from there
    call.desc.seqs = 0
    ctx.upload(a.missing, np.zeros(1, np.int32))
    ctx.pages_fork(call.desc)
    assert (pages._back(ctx, a.refs, refs.shape) == 0).all() and int(pages._back(ctx, a.missing, (1,))[0]) == 0
    for x in (a, b):
        x.free()
    pool.free()

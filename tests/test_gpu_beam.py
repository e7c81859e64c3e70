"""qa_beam_select on an MI355X against the definition in 64 bits, at vocabularies, ties and logits where it can go wrong.

Tolerances, derived.  parent, token and done are equal wherever the ranks of the definition lie further apart than the sums'
error: log sum exp of f32 sums over at most 8192 terms each (a thread's 32 and six steps of pairs, each rounded: 40 roundings)
of exponentials that are off by (2 |x - max| log2 e + 2) 2^-24 relative, of which those that weigh have |x - max| < 20: below
100 * 2^-24 = 6e-6 in all.  Inputs are drawn so that no two candidates of different beams at the border or in the order are
that near; candidates of one beam are ordered by their logits alone, exactly.  Scores: that and half a step of f32."""
from __future__ import annotations

import numpy as np
import pytest

from hipgraph import Capture
from paged import narrow, widen

pytestmark = pytest.mark.gpu

F16, BF16, F32 = 0, 1, 3
SUM = 100 * 2.0 ** -24


def _stored(x, dtype):
    return x.astype(np.float32) if dtype == F32 else narrow(x, dtype)


def _values(bits, dtype):
    return bits.astype(np.float64) if dtype == F32 else widen(bits, dtype)


def _want(x, score, done, end, groups, beams, width):
    """(parent, token, score, done): sorted by (-total, beam, token)."""
    out = []
    for g in range(groups):
        found = []
        for b in range(g * beams, (g + 1) * beams):
            if not np.isfinite(score[b]):
                continue
            if done is not None and done[b]:
                found.append((-float(score[b]), b, end))
                continue
            row = np.where(x[b] < np.inf, x[b], -np.inf)
            if (row == -np.inf).all():
                continue
            top = row.max()
            lse = top + np.log(np.exp(row - top).sum())
            for t in np.lexsort((np.arange(len(row)), -row))[:width]:
                if row[t] > -np.inf:
                    found.append((-(float(score[b]) + (row[t] - lse)), b, int(t)))
        best = (sorted(found) + [(np.inf, -1, -1)] * width)[:width]
        out += [(b, t, -s, int(b >= 0 and ((done is not None and done[b] != 0) or t == end))) for s, b, t in best]
    p, t, s, d = zip(*out) if out else ((), (), (), ())
    return np.array(p, np.int32), np.array(t, np.int32), np.array(s, np.float64), np.array(d, np.int32)


class Call:
    def __init__(self, ctx, pkg, bits, dtype, vocab, score, done, end, groups, beams, width):
        self.ctx, self.n = ctx, groups * width
        put = ctx.to_device
        self.x, self.s = put(bits), put(np.concatenate([score, [np.nan]]).astype(np.float32))
        self.d = put(np.asarray(done, np.int32)) if done is not None else None
        self.outs = [put(np.full(self.n + 2, 0x5A5A5A5A, np.int32)) for _ in range(4)]
        self.desc = pkg.BeamDesc(dtype=dtype, flags=0, groups=groups, beams=beams, width=width, vocab=vocab, logits=int(self.x), ldl=bits.shape[1],
                                 score=int(self.s), done=int(self.d) if self.d else None, end=end, parent=int(self.outs[0]), token=int(self.outs[1]),
                                 score_out=int(self.outs[2]), done_out=int(self.outs[3]))
        self.size = pkg.beam_select_workspace(self.desc)
        self.ws = put(np.full(self.size + 64, 0xFF, np.uint8))
        self.desc.workspace, self.desc.workspace_bytes = int(self.ws), self.size

    def run(self):
        self.ctx.beam_select(self.desc)
        return self

    def read(self):
        assert (self.ctx.download(self.ws, (self.size + 64,), np.uint8)[self.size:] == 0xFF).all()
        got = [self.ctx.download(o, (self.n + 2,), np.int32) for o in self.outs]
        assert all((o[self.n:] == 0x5A5A5A5A).all() for o in got)
        p, t, s, d = (o[: self.n] for o in got)
        return p, t, s.view(np.float32), d

    def free(self):
        for b in [self.x, self.s, self.d, self.ws] + self.outs:
            if b is not None:
                b.free()


def _check(ctx, pkg, x, dtype, score, done=None, end=-1, groups=1, beams=1, width=1, pad=None):
    """x: [rows, vocab] values that the format holds."""
    vocab = x.shape[1]
    unit = 4 if dtype == F32 else 8
    ld = -(-vocab // unit) * unit + (0 if pad is None else pad * unit)
    bits = np.full((x.shape[0], ld), np.float32(3e4) if dtype == F32 else narrow(np.float32(3e4), dtype))  # the padding would win
    bits[:, :vocab] = _stored(x, dtype)
    call = Call(ctx, pkg, bits, dtype, vocab, np.asarray(score, np.float32), done, end, groups, beams, width).run()
    got = call.read()
    want = _want(_values(bits[:, :vocab], dtype), np.asarray(score, np.float32), done, end, groups, beams, width)
    for a, b, name in ((0, 0, "parent"), (1, 1, "token"), (3, 3, "done")):
        assert np.array_equal(got[a], want[b]), (name, got, want)
    on = want[0] >= 0
    assert (got[2][~on] == -np.inf).all()
    s = want[2][on]
    assert (np.abs(got[2][on] - s) <= SUM + np.spacing(np.abs(s).astype(np.float32)) / 2).all()
    call.free()
    return got


DT = pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])


@DT
@pytest.mark.parametrize("groups,beams,width,vocab", [
    (1, 1, 1, 1), (1, 1, 1, 2), (2, 3, 2, 7), (1, 4, 8, 9), (3, 2, 5, 255), (1, 1, 64, 64), (2, 5, 10, 1000), (1, 8, 16, 2048), (2, 4, 4, 5000), (1, 3, 6, 8191),
    (1, 3, 3, 8192), (1, 2, 4, 8193), (5, 1, 1, 16385), (1, 4, 8, 151936), (3, 8, 8, 30011), (1, 64, 64, 4099), (2, 64, 33, 130), (70, 1, 2, 40)])
def test_select(ctx, pkg, dtype, groups, beams, width, vocab):
    r = np.random.default_rng(vocab + beams)
    x = _values(_stored(2.0 * r.standard_normal((groups * beams, vocab)), dtype), dtype)
    score = -9.0 * r.random(groups * beams)
    _check(ctx, pkg, x, dtype, score, groups=groups, beams=beams, width=width, pad=int(r.integers(0, 3)))


@DT
@pytest.mark.parametrize("vocab", [50, 9001])
def test_select_with_ended_beams(ctx, pkg, dtype, vocab):
    r = np.random.default_rng(vocab)
    x = _values(_stored(r.standard_normal((12, vocab)), dtype), dtype)
    score = -3.0 * r.random(12)
    done = np.array([0, 1, 0, 5, 1, 1, 1, 1, 0, 0, -1, 0], np.int32)
    got = _check(ctx, pkg, x, dtype, score, done, vocab - 3, groups=3, beams=4, width=6)
    assert (got[0][6 + 4: 12] == -1).all()  # the second group has four ended beams and no more
    _check(ctx, pkg, x, dtype, score, None, vocab - 3, groups=3, beams=4, width=6)
    _check(ctx, pkg, x, dtype, score, np.zeros(12, np.int32), 0, groups=3, beams=4, width=6)


@DT
def test_first_step(ctx, pkg, dtype):
    """One sequence in each group: the other scores are none, whatever their logits hold."""
    r = np.random.default_rng(3)
    x = _values(_stored(r.standard_normal((8, 6000)), dtype), dtype)
    x[[1, 2, 3]] = np.nan
    _check(ctx, pkg, x, dtype, [0, -np.inf, np.nan, np.inf] * 2, groups=2, beams=4, width=8)
    got = _check(ctx, pkg, x, dtype, [-np.inf] * 8, groups=2, beams=4, width=8)
    assert (got[0] == -1).all() and (got[1] == -1).all()


@DT
@pytest.mark.parametrize("width", [1, 7, 64])
def test_equal_logits_go_by_their_place(ctx, pkg, dtype, width):
    """All alike, in few values, and alike in every beam: the lowest beam and token first."""
    _check(ctx, pkg, np.zeros((3, 20000)), dtype, [-1.0] * 3, beams=3, width=width)
    r = np.random.default_rng(width)
    few = r.integers(0, 3, (1, 30000)).astype(np.float64)
    _check(ctx, pkg, few, dtype, [0.0], width=width)
    _check(ctx, pkg, np.repeat(few, 2, 0), dtype, [-2.0, -2.0], beams=2, width=width)
    late = np.zeros((1, 17000))
    late[0, [16999, 8191, 8192, 3]] = 4.0
    _check(ctx, pkg, late, dtype, [0.0], width=width)


@DT
def test_zeros_of_either_sign_are_alike(ctx, pkg, dtype):
    x = np.full((2, 9000), -1.0)
    x[:, [7, 100, 2500, 8999]] = [-0.0, 0.0, -0.0, 0.0]
    x[1] = -x[1] - 1.0
    x[1, x[1] == 0] = -0.0
    got = _check(ctx, pkg, x, dtype, [-1.0, -300.0], beams=2, width=6)
    assert list(got[1][:4]) == [7, 100, 2500, 8999]
    _check(ctx, pkg, np.where(np.arange(9000) % 3 == 1, 0.0, -0.0)[None], dtype, [0.0], width=40)


@DT
def test_rising_and_falling_logits(ctx, pkg, dtype):
    """The best are a thread's, a wave's or a chunk's own."""
    for n in (40, 2000, 9000):
        up = np.minimum(np.arange(n) / 4.0, 500.0)[None]
        for x in (up, up[:, ::-1]):
            _check(ctx, pkg, _values(_stored(np.ascontiguousarray(x), dtype), dtype), dtype, [0.0], width=33)
    x = np.full((1, 16384), -30.0)
    x[0, 8192:8192 + 64] = np.arange(64) / 8  # 64 neighbours
    _check(ctx, pkg, x, dtype, [0.0], width=64)


@DT
def test_banned_and_broken_logits(ctx, pkg, dtype):
    """-inf, +inf and NaN are not chosen and not counted; the type's lowest value counts as a number."""
    r = np.random.default_rng(9)
    x = _values(_stored(r.standard_normal((6, 9000)), dtype), dtype)
    x[0, 5:] = -np.inf           # five tokens left
    x[1, :] = -np.inf            # none
    x[2, ::3] = np.nan
    x[3, 100:200] = np.inf
    x[4, :] = np.nan
    low = {F16: -65504.0, BF16: -3.3895313892515355e38, F32: -3.4028234663852886e38}[dtype]
    x[5, :] = low
    x[5, 77] = 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        _check(ctx, pkg, x, dtype, [-1.0] * 6, groups=6, width=8)
        _check(ctx, pkg, x, dtype, [-1.0, -1.1, -1.2, -1.3, -1.4, -1.5], beams=6, width=16)
        _check(ctx, pkg, np.full((1, 300), low), dtype, [0.0], width=3)


@DT
@pytest.mark.parametrize("width", [1, 4, 30, 64])
def test_nan_of_every_kind(ctx, pkg, dtype, width):
    """Quiet and signalling NaN of either sign in places that a thread, a group of lanes or a chunk has for itself."""
    r = np.random.default_rng(width)
    x = r.standard_normal((2, 12000))
    bits = _stored(x, dtype) if dtype != F32 else x.astype(np.float32).view(np.uint32)
    kinds = {F16: [0x7C01, 0xFC01, 0x7E00, 0xFFFF], BF16: [0x7F81, 0xFF81, 0x7FC0, 0xFFFF], F32: [0x7F800001, 0xFF800001, 0x7FC00000, 0xFFFFFFFF]}[dtype]
    for k, kind in enumerate(kinds):
        bits[0, 300 * k: 300 * k + 256] = kind      # groups of lanes in a run
        bits[0, 2048 + k:: 4096] = kind
        bits[1, k:8192:4] = kind                    # a whole chunk
    if dtype == F32:
        bits = bits.view(np.float32)
    with np.errstate(invalid="ignore"):
        score = np.array([-1.0, -1.5], np.float32)
        call = Call(ctx, pkg, bits, dtype, 12000, score, None, -1, 2, 1, width).run()
        got, want = call.read(), _want(_values(bits, dtype), score, None, -1, 2, 1, width)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert (np.abs(got[2] - want[2]) <= SUM + 2.0 ** -21).all()
    call.free()


@DT
def test_large_scores_keep_their_order(ctx, pkg, dtype):
    """Steps of an f32 sum near -4000 are 2.4e-4: logits that differ by less are still told apart."""
    x = np.zeros((1, 3000))
    x[0, [5, 2900, 17]] = [8.0, 8.0 + 2.0 ** -7, 8.0 + 2.0 ** -7] if dtype == F16 else [8.0, 8.0625, 8.0625]
    if dtype == F32:
        x[0, [5, 2900, 17]] = [8.0, 8.0 + 2.0 ** -19, 8.0 + 2.0 ** -20]
    _check(ctx, pkg, x, dtype, [-4000.0], width=4)


def test_far_rows(ctx, pkg):
    """Rows behind the first 4 GB of the logits."""
    vocab, ld, rows = 5000, 1 << 24, 140
    buf = ctx.alloc(2 * ld * rows)
    r = np.random.default_rng(2)
    bits = narrow(r.standard_normal((2, vocab)), F16)
    ctx.upload(buf, bits[0], 0)
    ctx.upload(buf, bits[1], 2 * ld * (rows - 1))
    score = np.full(rows, -np.inf, np.float32)
    score[[0, rows - 1]] = [-1.0, -0.5]
    call = Call(ctx, pkg, np.zeros((1, 8), np.uint16), F16, vocab, score, None, -1, rows, 1, 2)
    call.desc.logits, call.desc.ldl = int(buf), ld
    got = call.run().read()
    want = _want(widen(bits, F16), np.array([-1.0, -0.5]), None, -1, 2, 1, 2)
    assert np.array_equal(got[1][[0, 1, -2, -1]], want[1]) and (got[0][2:-2] == -1).all() and list(got[0][[0, 1, -2, -1]]) == [0, 0, rows - 1, rows - 1]
    call.free()
    buf.free()


def test_captured_and_repeated(ctx, pkg):
    """A captured call, replayed on other logits, and the same bits from equal calls."""
    r = np.random.default_rng(12)
    x = [narrow(r.standard_normal((12, 20000)), F16) for _ in range(3)]
    score = (-5.0 * r.random(12)).astype(np.float32)
    call = Call(ctx, pkg, x[0], F16, 20000, score, None, 7, 3, 4, 8)
    other = Call(ctx, pkg, x[1], F16, 20000, score, None, 7, 3, 4, 8)
    with Capture(ctx.stream) as cap:
        call.run()
    for bits in x + x:
        ctx.upload(call.x, bits)
        cap.replay()
        got = call.read()
        other.run()  # the program's own call between the replays
        ctx.sync()
        want = _want(widen(bits, F16), score, None, 7, 3, 4, 8)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        again = call.run().read()
        assert all(np.array_equal(a, b) for a, b in zip(got, again))
    cap.close()
    call.free()
    other.free()

"""What qa_attention_paged_window, qa_pages_fork, qa_pages_compact, qa_pages_copy and qa_beam_select refuse (before they
look for a device), and their workspaces' sizes; no device is needed."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import pages
from paged import BF16, E4M3, F16

F32 = 3


def _refused(pkg, fn, desc, needle, code=None):
    assert fn(None, ctypes.byref(desc)) == (pkg.QA_EINVAL if code is None else code), pkg.last_error()
    assert needle in pkg.last_error(), pkg.last_error()


def _window(pkg, kv=None, **kw):
    kv = {**dict(dtype=F16, page=16, nkvh=8, hd=128, num_pages=40, k=0x100000, v=0x200000, table=0x300000, ldtable=8, seqs=4, row_start=0x310000,
                 kv_len=0x320000, max_rows=1, max_len=128), **(kv or {})}
    d = dict(dtype=F16, flags=0, tokens=4, nqh=16, q=0x400000, ldq=2048, kv=ctypes.pointer(pkg.PagedKV(**kv)), out=0x500000, ldo=2048, window=64, sinks=4,
             workspace=0x600000, workspace_bytes=1 << 40)
    return pkg.PagedWindowDesc(**{**d, **kw})


@pytest.mark.parametrize("kw,needle", [
    (dict(window=0), "window"), (dict(window=-1), "window"), (dict(window=2 ** 30 + 1), "window"), (dict(sinks=-1), "sinks"), (dict(sinks=2 ** 30 + 1), "sinks"),
    (dict(flags=1), "flags"), (dict(dtype=E4M3), "dtype"), (dict(nqh=12), "multiple"), (dict(ldq=2040), "ldq"), (dict(ldo=2044), "ldo"), (dict(q=None), "null"),
    (dict(out=0x500008), "aligned"), (dict(workspace=0x600004), "aligned"), (dict(kv=dict(hd=96)), "hd=96"), (dict(kv=dict(max_len=129)), "table row"),
    (dict(), "null context")])
def test_window_refusals(pkg, kw, needle):
    d = _window(pkg, kv=kw["kv"]) if kw.get("kv") else _window(pkg, **kw)
    _refused(pkg, pkg.lib().qa_attention_paged_window, d, needle, pkg.QA_EUNSUPPORTED if "hd=" in needle else None)
    d.kv = None
    if "window" not in kw and "sinks" not in kw and "flags" not in kw and "dtype" not in kw:
        _refused(pkg, pkg.lib().qa_attention_paged_window, d, "null kv")


def test_window_workspace(pkg):
    """Bound by the window and the sinks, not by the cache's length; a call without it is refused."""
    def size(max_len, **kw):
        return pkg.attention_paged_window_workspace(_window(pkg, kv=dict(max_len=max_len, ldtable=max_len // 16, seqs=1), tokens=1, **kw))
    assert size(1 << 20, window=300, sinks=4) == 0
    assert 0 < size(1 << 20, window=1500, sinks=4) == size(1 << 16, window=1500, sinks=4) < size(1 << 20, window=1 << 20)
    assert size(1 << 20, window=1 << 30) == pkg.attention_paged_workspace(pkg.PagedAttentionDesc(
        dtype=F16, tokens=1, nqh=16, kv=_window(pkg, kv=dict(max_len=1 << 20, ldtable=1 << 16, seqs=1)).kv))
    d = _window(pkg, kv=dict(max_len=1 << 20, ldtable=1 << 16, seqs=1), tokens=1, window=8192, workspace_bytes=100)
    _refused(pkg, pkg.lib().qa_attention_paged_window, d, "workspace")
    n = ctypes.c_size_t()
    assert pkg.lib().qa_attention_paged_window_workspace(ctypes.byref(_window(pkg, window=0)), ctypes.byref(n)) == pkg.QA_EINVAL


# ------------------------------------------------------------ pages

def _planes(pkg, *sizes, base=0x1000000):
    return (pkg.PagePlane * len(sizes))(*[(base + 0x1000 * i, n) for i, n in enumerate(sizes)])


BAD_PLANES = [((0,), "0 bytes"), ((-16,), "-16 bytes"), ((6,), "6 bytes"), ((4100,), "4100 bytes"), ((4096, 4104), "4104 bytes"), ((2 ** 31,), "bytes")]


def _copy(pkg, sizes=(4096, 32), **kw):
    d = dict(flags=0, nplanes=len(sizes), src=_planes(pkg, *sizes), src_pages=9, dst=_planes(pkg, *sizes), dst_pages=7, pairs=0x300000, npairs=5)
    return pkg.PagesCopyDesc(**{**d, **kw})


def test_copy_refusals(pkg):
    fn = pkg.lib().qa_pages_copy
    for sizes, needle in BAD_PLANES:
        _refused(pkg, fn, _copy(pkg, sizes), needle)
    for kw, needle in ((dict(flags=1), "flags"), (dict(src_pages=0), "pages"), (dict(dst_pages=2 ** 31), "pages"), (dict(nplanes=-1), "nplanes"), (dict(nplanes=65537), "nplanes"),
                       (dict(npairs=-1), "npairs"), (dict(npairs=2 ** 31), "npairs"), (dict(pairs=None), "null"), (dict(pairs=0x300002), "misaligned"),
                       (dict(src=None), "null planes"), (dict(dst=_planes(pkg, 4096, 48)), "48 bytes"), (dict(dst=_planes(pkg, 4096, 32, base=0x1000002)), "aligned"),
                       (dict(dst=_planes(pkg, 8192, 32, base=0x1000008), src=_planes(pkg, 8192, 32)), "aligned"), (dict(dst=_planes(pkg, 4096, 32, base=0x1000004)), "null context"),
                       (dict(dst=_planes(pkg, 4096, 32, base=0)), "null"), (dict(), "null context")):
        _refused(pkg, fn, _copy(pkg, **kw), needle)
    assert fn(None, None) == pkg.QA_EINVAL


def _fork(pkg, **kw):
    d = dict(flags=0, page=16, num_pages=100, planes=_planes(pkg, 4096, 32), nplanes=2, refs=0x100000, src_seqs=4, seqs=6, ldtable=8, src_table=0x200000,
             src_len=0x210000, parent=0x220000, table=0x230000, len=0x240000, grow=0x250000, window=0, sinks=0, missing=0x260000, workspace=0x300000,
             workspace_bytes=1 << 30)
    return pkg.PagesForkDesc(**{**d, **kw})


@pytest.mark.parametrize("kw,needle", [
    (dict(flags=2), "flags"), (dict(page=8), "page=8"), (dict(num_pages=0), "num_pages"), (dict(num_pages=2 ** 31), "num_pages"), (dict(src_seqs=-1), "negative"),
    (dict(seqs=-1), "negative"), (dict(ldtable=-1), "negative"), (dict(seqs=8193), "8192"), (dict(src_seqs=8193), "8192"), (dict(ldtable=2 ** 30), "entries"),
    (dict(window=-1), "window"), (dict(sinks=2 ** 31), "sinks"), (dict(refs=None), "null"), (dict(missing=None), "null"), (dict(src_table=None), "null"), (dict(src_len=None), "null"),
    (dict(parent=None), "null"), (dict(table=None), "null"), (dict(len=None), "null"), (dict(grow=0x250001), "misaligned"), (dict(refs=0x100002), "misaligned"),
    (dict(workspace=0x300008), "misaligned"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=60), "workspace"), (dict(table=0x200000), "sources"),
    (dict(table=0x200000 + 4 * 31), "sources"), (dict(len=0x210000 - 20), "sources"), (dict(len=0x220000), "sources"),
    (dict(missing=0x250008), "sources"), (dict(refs=0x250000 - 396), "sources"), (dict(table=0x220000 - 4 * 47), "sources"), (dict(nplanes=1, planes=None), "null planes"), (dict(), "null context")])
def test_fork_refusals(pkg, kw, needle):
    code = pkg.QA_EUNSUPPORTED if needle in ("page=8", "8192") else None
    _refused(pkg, pkg.lib().qa_pages_fork, _fork(pkg, **kw), needle, code)


def _compact(pkg, **kw):
    d = dict(flags=0, num_pages=100, planes=_planes(pkg, 4096, 32), nplanes=2, refs=0x100000, refs_out=0x110000, seqs=6, ldtable=8, table=0x200000, table_out=0x210000,
             map=0x220000, used=0x230000, workspace=0x300000, workspace_bytes=1 << 30)
    return pkg.PagesCompactDesc(**{**d, **kw})


@pytest.mark.parametrize("kw,needle", [
    (dict(flags=1), "flags"), (dict(num_pages=0), "num_pages"), (dict(seqs=-1), "entries"), (dict(ldtable=2 ** 30), "entries"), (dict(refs=None), "null"),
    (dict(refs_out=None), "null"), (dict(used=None), "null"), (dict(table=None), "null"), (dict(table_out=None), "null"), (dict(map=0x220002), "misaligned"),
    (dict(workspace=0x300004), "misaligned"), (dict(workspace_bytes=100), "workspace"), (dict(refs_out=0x100004), "no part"), (dict(table_out=0x200000 + 4 * 47), "no part"),
    (dict(map=0x100000), "no part"), (dict(map=0x200000 - 396), "no part"), (dict(used=0x200000 + 4 * 47), "no part"), (dict(used=0x100000), "no part"),
    (dict(refs_out=0x200000), "no part"), (dict(table_out=0x100000), "no part"),
    (dict(refs_out=0x100000, table_out=0x200000), "null context"), (dict(), "null context")])
def test_compact_refusals(pkg, kw, needle):
    _refused(pkg, pkg.lib().qa_pages_compact, _compact(pkg, **kw), needle)


def test_page_workspaces(pkg):
    """A few numbers for each page and sequence."""
    assert 0 < pkg.pages_fork_workspace(_fork(pkg)) <= 64 + 8 * 6
    assert pkg.pages_fork_workspace(_fork(pkg, seqs=1024)) <= 64 + 8 * 1024 < pkg.pages_fork_workspace(_fork(pkg, seqs=1025)) <= 64 + 8 * 1025 + 8 * 100
    assert 0 < pkg.pages_compact_workspace(_compact(pkg)) <= 64 + 12 * 100
    n = ctypes.c_size_t()
    assert pkg.lib().qa_pages_fork_workspace(ctypes.byref(_fork(pkg, page=5)), ctypes.byref(n)) == pkg.QA_EUNSUPPORTED
    assert pkg.lib().qa_pages_compact_workspace(None, ctypes.byref(n)) == pkg.QA_EINVAL


def test_the_model_keeps_count():
    """The tests' own model: references are what the tables hold, at every step, and no page is anybody's twice."""
    r = np.random.default_rng(1)
    table, length, refs = pages.random_sequences(r, 8, 16, 12, 300, 150)
    for step in range(30):
        parent = r.integers(-1, len(length), 8).astype(np.int32)
        window = int(r.choice([0, 50]))
        old = table
        table, length, refs, missing, pairs = pages.fork_model(refs, table, length, parent, np.ones(8, np.int32), 16, 300, window=window, sinks=4)
        assert missing == 0
        count = np.zeros(300, np.int32)
        np.add.at(count, table[table >= 0], 1)
        assert np.array_equal(count, refs)
        for i in range(8):  # the page that is written next is its own
            if length[i]:
                assert refs[table[i, (length[i] - 1) // 16]] == 1
        assert not set(d for _, d in pairs) & set(old[old >= 0].tolist()) or all(refs[d] == 1 for _, d in pairs)


# ------------------------------------------------------------ beams

def _beam(pkg, **kw):
    d = dict(dtype=F16, flags=0, groups=2, beams=4, width=8, vocab=1000, logits=0x100000, ldl=1000, score=0x200000, done=0x210000, end=5, parent=0x220000,
             token=0x230000, score_out=0x240000, done_out=0x250000, workspace=0x300000, workspace_bytes=1 << 30)
    return pkg.BeamDesc(**{**d, **kw})


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=E4M3), "dtype"), (dict(dtype=4), "dtype"), (dict(flags=1), "flags"), (dict(groups=-1), "groups"), (dict(beams=0), "beams=0"), (dict(beams=65), "beams=65"),
    (dict(width=0), "width=0"), (dict(width=65), "width=65"), (dict(vocab=0), "vocab"), (dict(vocab=2 ** 31, ldl=2 ** 31), "vocab"), (dict(ldl=992), "ldl"), (dict(ldl=1004), "ldl"),
    (dict(dtype=F32, ldl=1002), "ldl"), (dict(end=1000), "end"), (dict(end=-2), "end"), (dict(end=-1), "end"), (dict(logits=None), "null"), (dict(score=None), "null"),
    (dict(parent=None), "null"), (dict(done_out=None), "null"), (dict(logits=0x100008), "misaligned"), (dict(score=0x200002), "misaligned"), (dict(workspace=0x300004), "misaligned"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=8), "workspace"), (dict(score_out=0x200000), "outputs"), (dict(done_out=0x210000), "outputs"),
    (dict(parent=0x200000 - 60), "outputs"), (dict(token=0x100000 + 15996), "outputs"),
    (dict(score_out=0x100000 + 31996, dtype=F32, ldl=1004), "outputs"), (dict(groups=2 ** 24, vocab=10 ** 6, ldl=10 ** 6, workspace_bytes=2 ** 62), "too large"), (dict(dtype=F32, ldl=1004), "null context"),
    (dict(done=None, end=-1), "null context"), (dict(), "null context")])
def test_beam_refusals(pkg, kw, needle):
    code = pkg.QA_EUNSUPPORTED if needle.startswith(("beams", "width")) else None
    _refused(pkg, pkg.lib().qa_beam_select, _beam(pkg, **kw), needle, code)


def test_beam_workspace(pkg):
    """Grows with the rows' chunks and the width; nothing for no groups."""
    size = [pkg.beam_select_workspace(_beam(pkg, groups=g, vocab=v, ldl=v)) for g, v in ((0, 1000), (1, 1000), (2, 1000), (2, 151936))]
    assert size[0] == 0 < size[1] and size[2] == 2 * size[1] < size[3] <= 8 * 160 * (8 + 8 * 8 + 16)
    assert BF16 == 1 and pkg.lib().qa_beam_select(None, None) == pkg.QA_EINVAL

"""The paged-cache operators on the CPU: what qa_mrope_rows, qa_kv_append and
qa_attention_paged refuse (before they look for a device), the workspace's size,
and the kernels' index arithmetic (csrc/qa_paged.h), compiled for the host, over
tables, row counts and lengths that are out of range."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import paged
from paged import BF16, E4M3, F16


def _kv(pkg, **kw):
    d = dict(dtype=F16, page=16, nkvh=8, hd=128, num_pages=40, k=0x100000, v=0x200000, k_scale=None, v_scale=None, table=0x300000,
             ldtable=8, seqs=4, row_start=0x310000, kv_len=0x320000, max_rows=1, max_len=128)
    return pkg.PagedKV(**{**d, **kw})


def _append(pkg, kv=None, **kw):
    d = dict(dtype=F16, flags=0, tokens=4, nqh=16, eps=1e-6, qkv=0x400000, ldqkv=4096, qn_w=0x500000, kn_w=0x500400, cos=0x600000,
             sin=0x610000, q_out=0x700000, ldq=2048)
    return pkg.KvAppendDesc(**{**d, **kw}, kv=ctypes.pointer(kv) if kv is not None else None)


def _attention(pkg, kv=None, **kw):
    d = dict(dtype=F16, flags=0, tokens=4, nqh=16, q=0x400000, ldq=2048, out=0x500000, ldo=2048, workspace=0x600000,
             workspace_bytes=1 << 40)
    return pkg.PagedAttentionDesc(**{**d, **kw}, kv=ctypes.pointer(kv) if kv is not None else None)


def _mrope(pkg, **kw):
    d = dict(dtype=F16, flags=0, tokens=4, hd=128, axes=3, sec0=24, sec1=20, sec2=20, theta=1e6, pos=0x100000, ldpos=4, cos=0x200000,
             sin=0x300000)
    return pkg.MropeDesc(**{**d, **kw})


def _refused(pkg, fn, desc, code, needle):
    assert fn(None, ctypes.byref(desc)) == code, pkg.last_error()
    assert needle in pkg.last_error(), pkg.last_error()


KV_BAD = [
    (dict(dtype=BF16), "dtype", None), (dict(dtype=7), "dtype", None), (dict(page=8), "page=8", "U"), (dict(page=128), "page=128", "U"),
    (dict(hd=96), "hd=96", "U"), (dict(hd=256), "hd=256", "U"), (dict(nkvh=3), "multiple of nkvh", None), (dict(nkvh=0), "nkvh", None),
    (dict(seqs=-1), "seqs", None), (dict(max_rows=-1), "max_rows", None), (dict(max_len=-1), "max_len", None),
    (dict(max_len=129), "table row", None), (dict(max_len=2 ** 31 - 1, ldtable=2 ** 30), "max_len", None),
    (dict(num_pages=0), "num_pages", None), (dict(num_pages=2 ** 31), "num_pages", None), (dict(ldtable=-1), "table row", None),
    (dict(k=None), "null cache", None), (dict(table=None), "null cache", None), (dict(kv_len=None), "null cache", None),
    (dict(row_start=None), "null cache", None), (dict(v=0x200008), "misaligned", None), (dict(table=0x300002), "misaligned", None),
    (dict(dtype=E4M3, k_scale=0x800000), "null cache", None), (dict(dtype=E4M3, k_scale=0x800000, v_scale=0x900002), "misaligned", None),
]


@pytest.mark.parametrize("kw,needle,code", KV_BAD)
def test_cache_refusals(pkg, kw, needle, code):
    lib, c = pkg.lib(), pkg.QA_EUNSUPPORTED if code else pkg.QA_EINVAL
    _refused(pkg, lib.qa_kv_append, _append(pkg, _kv(pkg, **kw)), c, needle)
    _refused(pkg, lib.qa_attention_paged, _attention(pkg, _kv(pkg, **kw)), c, needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=E4M3), "dtype"), (dict(flags=1), "flags"), (dict(tokens=-1), "tokens"), (dict(tokens=2 ** 31), "tokens"), (dict(nqh=12), "multiple"),
    (dict(ldqkv=4088), "ldqkv"), (dict(ldqkv=4100), "ldqkv"), (dict(ldq=2040), "ldq"), (dict(ldq=2052), "ldq"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(qkv=None), "null"), (dict(q_out=None), "null"), (dict(cos=None), "null"), (dict(sin=0x610004), "aligned"),
    (dict(qkv=0x400002), "aligned"), (dict(qn_w=0x500004), "aligned"),
])
def test_append_refusals(pkg, kw, needle):
    _refused(pkg, pkg.lib().qa_kv_append, _append(pkg, _kv(pkg), **kw), pkg.QA_EINVAL, needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=E4M3), "dtype"), (dict(flags=1), "flags"), (dict(tokens=-1), "tokens"), (dict(nqh=0), "multiple"), (dict(ldq=2040), "ldq"),
    (dict(ldo=2044), "ldo"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(out=0x500008), "aligned"), (dict(workspace=0x600004), "aligned"),
])
def test_attention_refusals(pkg, kw, needle):
    _refused(pkg, pkg.lib().qa_attention_paged, _attention(pkg, _kv(pkg), **kw), pkg.QA_EINVAL, needle)


def test_null_arguments(pkg):
    lib = pkg.lib()
    for fn in (lib.qa_mrope_rows, lib.qa_kv_append, lib.qa_attention_paged):
        assert fn(None, None) == pkg.QA_EINVAL and "null argument" in pkg.last_error()
    _refused(pkg, lib.qa_kv_append, _append(pkg), pkg.QA_EINVAL, "null kv")
    _refused(pkg, lib.qa_attention_paged, _attention(pkg), pkg.QA_EINVAL, "null kv")
    # everything in order but the context
    _refused(pkg, lib.qa_mrope_rows, _mrope(pkg), pkg.QA_EINVAL, "null context")
    _refused(pkg, lib.qa_kv_append, _append(pkg, _kv(pkg)), pkg.QA_EINVAL, "null context")
    _refused(pkg, lib.qa_attention_paged, _attention(pkg, _kv(pkg)), pkg.QA_EINVAL, "null context")
    n = ctypes.c_size_t()
    assert lib.qa_attention_paged_workspace(None, ctypes.byref(n)) == pkg.QA_EINVAL
    assert lib.qa_attention_paged_workspace(ctypes.byref(_attention(pkg, _kv(pkg))), None) == pkg.QA_EINVAL


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=E4M3), "dtype"), (dict(flags=2), "flags"), (dict(hd=124, sec0=22), "multiple of 8"), (dict(hd=264, sec0=92), "up to 256"),
    (dict(hd=0), "multiple of 8"), (dict(axes=0), "axes"), (dict(axes=4), "axes"), (dict(sec0=25), "sections"), (dict(axes=2), "sections"),
    (dict(sec0=65, sec1=-1, sec2=0), "sections"), (dict(axes=1, sec0=44, sec2=0), "sections"), (dict(tokens=5), "ldpos"), (dict(tokens=-1), "tokens"),
    (dict(theta=0.0), "theta"), (dict(theta=0.999), "theta"), (dict(theta=float("nan")), "theta"), (dict(theta=float("inf")), "theta"), (dict(pos=None), "null"),
    (dict(cos=0x200004), "aligned"), (dict(pos=0x100002), "aligned"),
])
def test_mrope_refusals(pkg, kw, needle):
    _refused(pkg, pkg.lib().qa_mrope_rows, _mrope(pkg, **kw), pkg.QA_EINVAL, needle)


def test_batches_past_one_launch_are_refused(pkg):
    wide = _mrope(pkg, tokens=2 ** 28, ldpos=2 ** 28)  # a grid of 2^32 threads
    _refused(pkg, pkg.lib().qa_mrope_rows, wide, pkg.QA_EINVAL, "too large")
    many = _kv(pkg, seqs=1, max_rows=4, max_len=128)
    _refused(pkg, pkg.lib().qa_attention_paged, _attention(pkg, many, tokens=2 ** 30), pkg.QA_EINVAL, "too large")
    _refused(pkg, pkg.lib().qa_kv_append, _append(pkg, many, tokens=2 ** 26), pkg.QA_EINVAL, "too large")
    big = _kv(pkg, seqs=2 ** 23, max_rows=1, max_len=128)
    _refused(pkg, pkg.lib().qa_attention_paged, _attention(pkg, big, workspace_bytes=2 ** 62), pkg.QA_EINVAL, "too large")
    big = _kv(pkg, seqs=2 ** 30, max_rows=4, max_len=128)
    _refused(pkg, pkg.lib().qa_kv_append, _append(pkg, big), pkg.QA_EINVAL, "too large")
    _refused(pkg, pkg.lib().qa_attention_paged, _attention(pkg, big, workspace_bytes=2 ** 62), pkg.QA_EINVAL, "too large")


def test_workspace_is_needed_in_full(pkg):
    """A call with less than qa_attention_paged_workspace's bytes, or with none, is refused."""
    for seqs, tokens, max_len in ((1, 1, 1 << 20), (4, 4, 4096), (3, 700, 2048)):
        kv = _kv(pkg, seqs=seqs, max_rows=tokens, max_len=max_len, ldtable=max_len // 16)
        d = _attention(pkg, kv, tokens=tokens)
        size = pkg.attention_paged_workspace(d)
        assert size % 4 == 0
        if not size:
            continue
        for kw in (dict(workspace_bytes=size - 1), dict(workspace=None)):
            _refused(pkg, pkg.lib().qa_attention_paged, _attention(pkg, kv, tokens=tokens, **kw), pkg.QA_EINVAL, "workspace")


def test_e4m3_restatement():
    """The tests' e4m3: every code survives, midpoints go to even, 448 is the end."""
    codes = np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8)
    v = paged.e4m3_values(codes)
    assert np.array_equal(paged.e4m3_codes(v), codes) and v.max() == 448 and np.abs(v[v != 0]).min() == 2.0 ** -9
    pos = np.sort(v[:127])
    mid = (pos[1:] + pos[:-1]) / 2
    r = paged.e4m3_values(paged.e4m3_codes(mid))
    assert (np.abs(r - mid) == (pos[1:] - pos[:-1]) / 2).all() and (paged.e4m3_codes(mid) & 1 == 0).all()
    assert list(paged.e4m3_codes([np.inf, -1e9, np.nan])) == [0x7E, 0xFE, 0x7F]
    assert [float(paged.scale_for(x)) for x in (448.0, 448.1, 449.0, 224.0, 1.75, 0.0)] == [1.0, 2.0, 2.0, 0.5, 2.0 ** -8, 2.0 ** -110]


INDEX_PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "qa_paged.h"
// every page and slot that an append or an attention of this batch would touch
int main() {
  long long bad = 0, seen = 0;
  const int values[] = {-2147483647 - 1, -5, -1, 0, 1, 2, 7, 15, 16, 17, 40, 1000, 2147483647};
  for (int lp = 4; lp <= 6; ++lp)
    for (int64_t ldt = 0; ldt <= 3; ++ldt)
      for (int a : values) for (int b : values) for (int len : values) for (int entry : values)
        for (int max_rows : {0, 1, 9, 40}) {
          const int64_t tokens = 40;
          int32_t start[2] = {a, b}, lens[1] = {len};
          std::vector<int32_t> table((size_t)ldt + 1, entry);
          qa::PagedParams p{};
          p.table = table.data(); p.row_start = start; p.kv_len = lens;
          p.num_pages = 17; p.ldtable = ldt; p.tokens = tokens; p.seqs = 1;
          p.max_rows = max_rows; p.max_len = (int)(ldt << lp); p.nkvh = 2; p.lp = lp;
          const qa::SeqSpan q = qa::seq_span(p, 0);
          if (q.n < 0 || q.n > max_rows || q.row0 < 0 || q.row0 + q.n > tokens || q.len < 0 || q.len > p.max_len) ++bad;
          if (q.n > 0 && (int64_t)q.pos0 + q.n > q.len) ++bad;  // a row's position is a key's
          // a row that is kept has the position that it has without the bounds
          if (q.n > 0 && a >= 0 && a < b && b < 1 << 30 && q.pos0 != q.len - ((int64_t)b - a)) ++bad;
          const int64_t elems = 17 * 2 * (128LL << lp);
          for (int i = -3; i < q.n + 3; ++i) {
            const int pos = q.pos0 + i;
            const int id = qa::page_at(p, 0, pos);
            ++seen;
            if (id < 0) continue;
            if (pos < 0 || (pos >> lp) >= ldt || id >= 17) ++bad;
            const int64_t at = qa::page_base(p, id, 1, 128) + ((int64_t)(pos & ((1 << lp) - 1))) * 128 + 127;
            if (at < 0 || at >= elems) ++bad;
          }
          // the launch's page slots cover every page the rows touch
          if (q.n > 0 && q.pos0 + q.n > 0) {
            const int first = q.pos0 > 0 ? q.pos0 : 0;
            const int64_t need = ((q.pos0 + q.n - 1) >> lp) - (first >> lp) + 1;
            if (need > qa::pages_touched(max_rows, lp)) ++bad;
          }
        }
  // offsets past 32 bits
  qa::PagedParams p{};
  p.num_pages = 2147483647; p.nkvh = 8; p.lp = 6;
  if (qa::page_base(p, 2147483646, 7, 128) != (2147483646LL * 8 + 7) * 64 * 128) ++bad;
  printf("%lld %lld\n", bad, seen);
}
"""


def test_index_arithmetic_stays_in_range(pkg, tmp_path):
    """seq_span, page_at and page_base over out-of-range row starts, lengths and
    page ids: what they let through lies in the buffers."""
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    src, exe = tmp_path / "i.cpp", tmp_path / "i"
    src.write_text(INDEX_PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", pkg.CSRC, str(src), "-o", str(exe)], check=True)
    bad, seen = map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    assert bad == 0 and seen > 100000


def test_new_descriptor_layouts(pkg, tmp_path):
    """The ctypes mirrors have the C structs' sizes and offsets."""
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    structs = {"qa_mrope_desc": pkg.MropeDesc, "qa_paged_kv": pkg.PagedKV, "qa_kv_append_desc": pkg.KvAppendDesc,
               "qa_paged_attention_desc": pkg.PagedAttentionDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "qa.h"', "int main(void) {"]
    for c, py in structs.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", pkg.INCLUDE_DIR, str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in structs.items():
        assert int(got[c]) == ctypes.sizeof(py), c
        for f, _ in py._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(py, f).offset, (c, f)
    assert os.path.exists(os.path.join(pkg.CSRC, "qa_paged.h"))

"""qa_attention_paged_workspace on the CPU: what a batch's partial results may take."""
from __future__ import annotations

import ctypes

import pytest

from paged import BF16, E4M3, F16

F32 = 4
MOST = 66  # parts of a short sequence's keys: up to 33 are asked for, and rounding them to 256 keys and to an odd number may double that


def _bytes(pkg, *, tokens, seqs, max_rows, max_len, nq=16, nkv=8, hd=128, dtype=F16, cache=None):
    kv = pkg.PagedKV(dtype=dtype if cache is None else cache, page=32, nkvh=nkv, hd=hd, seqs=seqs, max_rows=max_rows, max_len=max_len)
    return pkg.attention_paged_workspace(pkg.PagedAttentionDesc(dtype=dtype, flags=0, tokens=tokens, nqh=nq, kv=ctypes.pointer(kv)))


@pytest.mark.parametrize("max_len,dtype,cache", [(8192, F16, F16), (32768, BF16, E4M3)])
def test_a_prompt_beside_a_single_token(pkg, max_len, dtype, cache):
    """A prompt of 4334 rows, whose keys are not split, and one token behind many keys: only the short sequence's pairs, up
    to 16 for each sequence and kv head, can have partial results.  (For every row they were 577 and 1154 MB.)"""
    size = _bytes(pkg, tokens=4335, seqs=2, max_rows=4334, max_len=max_len, dtype=dtype, cache=cache)
    assert 0 < size <= 2 * 8 * 16 * MOST * (128 + 2) * F32


@pytest.mark.parametrize("seqs,max_len", [(1, 2000), (3, 20000), (64, 8192)])
def test_single_tokens(pkg, seqs, max_len):
    """A token for each sequence: parts for each of its rows and heads."""
    size = _bytes(pkg, tokens=seqs, seqs=seqs, max_rows=1, max_len=max_len)
    each = seqs * 16 * (128 + 2) * F32
    assert size % each == 0 and 2 <= size // each <= MOST


def test_bounds_above_what_the_batch_holds(pkg):
    """64 rows in 64 sequences, any of which may have all of them: 16 pairs for each would be more than the rows have."""
    size = _bytes(pkg, tokens=64, seqs=64, max_rows=64, max_len=32768)
    rows = 64 * 16 * (128 + 2) * F32
    assert 0 < size <= rows * (MOST + 256)
    # and with the longer tiles unsplit
    size = _bytes(pkg, tokens=512, seqs=512, max_rows=512, max_len=32768)
    assert 0 < size <= 8 * rows * MOST


def test_whole_prompts_need_none(pkg):
    assert _bytes(pkg, tokens=4334, seqs=1, max_rows=4334, max_len=4334) == 0
    assert _bytes(pkg, tokens=0, seqs=2, max_rows=1, max_len=4000) == 0

// qa_paged.h -- where a packed batch's rows and a sequence's keys lie: the index
// arithmetic of the paged-cache kernels (qa_paged_append.hip,
// qa_paged_attention.hip), plain C++ so that a host program can run it over any
// table.  Every number that a kernel reads from device memory (row_start,
// kv_len, page ids) is held to its range here, so that none of them can take an
// access outside the buffers the call was given.
#pragma once

#include <stdint.h>

#if defined(__HIP__)
#define QA_HD __host__ __device__ __forceinline__
#else
#define QA_HD inline
#endif

namespace qa {

// The batch and the cache of a call (qa_paged_kv).
struct PagedParams {
  void *k, *v;
  float *k_scale, *v_scale;
  const int32_t *table, *row_start, *kv_len;
  int64_t num_pages, ldtable, tokens;
  int seqs, max_rows, max_len;
  int nkvh, lp;  // page size 1 << lp
};

// A sequence's part of the batch: rows row0 .. row0 + n - 1, the first of them at
// position pos0 (negative where the sequence has fewer keys than rows), len
// keys in all.  Rows that are left out, past max_rows or the batch's end, keep
// their positions: the others' do not move.  seen() keys are seen by any row; those
// behind, of rows that are left out, may be slots that nothing was written to.
struct SeqSpan {
  int64_t row0;
  int n, pos0, len;
  QA_HD int seen() const { return pos0 + n; }
};

QA_HD int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

QA_HD SeqSpan seq_span(const PagedParams& p, int s) {
  const int64_t a = clamp64(p.row_start[s], 0, p.tokens);
  const int64_t last = p.row_start[s + 1] > a ? p.row_start[s + 1] : a, e = last < p.tokens ? last : p.tokens;
  SeqSpan q;
  q.row0 = a;
  q.len = (int)clamp64(p.kv_len[s], 0, p.max_len);
  q.pos0 = (int)clamp64(q.len - (last - a), -(1 << 30), q.len);  // (a batch has at most 2^30 rows)
  q.n = (int)clamp64(e - a, 0, p.max_rows);
  return q;
}

// The page that holds position pos of sequence s, or -1: pos is at or past the
// table's end, or the table's entry names no page.
QA_HD int page_at(const PagedParams& p, int s, int pos) {
  const int64_t i = (int64_t)(pos >> p.lp);
  if (pos < 0 || i >= p.ldtable) return -1;
  const int32_t id = p.table[(int64_t)s * p.ldtable + i];
  return id >= 0 && id < p.num_pages ? id : -1;
}

// First element of kv head h of page id, with hd elements for each of the
// page's tokens (K [page][hd], V [hd][page]).
QA_HD int64_t page_base(const PagedParams& p, int id, int h, int hd) {
  return ((int64_t)id * p.nkvh + h) * ((int64_t)hd << p.lp);
}

// Pages that up to `rows` consecutive positions touch, wherever they begin.
QA_HD int64_t pages_touched(int64_t rows, int lp) {
  return rows <= 0 ? 0 : (rows + (2LL << lp) - 2) >> lp;
}

}  // namespace qa

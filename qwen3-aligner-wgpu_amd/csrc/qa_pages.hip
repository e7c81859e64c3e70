// qa_pages.hip -- a pool's pages: copied, shared and taken for the next step's sequences,
// moved to the front.
//
// Page numbers are planned on the device by one block, in whole numbers and in one
// order, so that equal calls give equal tables; the pages' bytes follow in a launch over all
// planes.  Plans are bound by trips to memory and the instructions of one CU's sixteen
// waves: parents and lengths, tables, references, the search for free pages, what
// is written: 4.8 us for 4 sequences, and 2.5 to 8 us for a pool
// of 90 to 4096 pages.  Free pages are looked for from the front, 4096 a round, and twice where the
// first does not have enough: 192 new ones behind 1061 others take the block 5.0 us, behind
// 5157 7.8, 17445 16.5, 132133 92.  Copies are bound by the pages' bytes, twice: 1900 pages of 524 KB
// 404 us, 4.9 TB/s, where a large copy reaches 5.1.
#include "qa_internal.h"

namespace qa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- pages from one place to another ----
//
// blockIdx.y is the plane.  A wave takes 4 KB of a page at a time, four 16-byte loads
// in flight for each lane; short pages (scales), and those that are not in 16 bytes, go
// by words, a lane each.  The next pair is read in front of a piece's loads, the first along
// with the number of pairs, which may turn out to be without it (84 pages' copies 3.1 us for
// 3.4, 21 pages of 28 layers 15.0 for 15.4).
constexpr int kPiece = 4096;
// Number u, u + step .. of the units of the pairs' pages, `each` to a page.
struct Unit {
  uint32_t pair, part, pairs, parts, each;
  __device__ __forceinline__ Unit(uint32_t u, uint32_t step, uint32_t n)
      : pair(u / n), part(u - u / n * n), pairs(step / n), parts(step - step / n * n), each(n) {}
  __device__ __forceinline__ void next() {
    part += parts;
    const uint32_t over = part >= each;
    part -= over * each;
    pair += pairs + over;
  }
};
__global__ void __launch_bounds__(256) page_copy_kernel(const PagePlanes planes, const PagesCopyParams p) {
  const auto pl = planes.at[blockIdx.y];
  asm volatile("" ::"s"(pl.src), "s"(pl.dst), "s"(pl.bytes), "s"(p.count), "s"(p.dst_pages));  // in one trip to memory
  __builtin_amdgcn_sched_barrier(0);
  const int64_t bytes = pl.bytes;
  const uint32_t held = (uint32_t)p.npairs;
  auto at = [&](uint32_t pair) { return p.pairs + 2 * (int64_t)(pair < held ? pair : 0); };
  auto count = [&] { return p.count ? (uint32_t)clamp64(*p.count, 0, p.npairs) : held; };
  auto is_pair = [&](int32_t a, int32_t b) { return a >= 0 && a < p.src_pages && b >= 0 && b < p.dst_pages; };
  if (((uint64_t)pl.src | (uint64_t)pl.dst | (uint64_t)bytes) % 16 || bytes < 1024) {
    Unit u(blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, (uint32_t)bytes / 4);
    int32_t a = at(u.pair)[0], b = at(u.pair)[1];
    for (const uint32_t n = count(); u.pair < n;) {
      if (is_pair(a, b))
        *reinterpret_cast<uint32_t*>(pl.dst + b * bytes + 4 * u.part) = *reinterpret_cast<const uint32_t*>(pl.src + a * bytes + 4 * u.part);
      u.next();
      a = at(u.pair)[0];
      b = at(u.pair)[1];
    }
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  Unit u(blockIdx.x * 4 + wave, gridDim.x * 4, ((uint32_t)bytes + kPiece - 1) / kPiece);
  int32_t a = at(u.pair)[0], b = at(u.pair)[1];
  for (const uint32_t n = count(); u.pair < n;) {
    const int64_t off = (int64_t)u.part * kPiece + lane * 16;
    const unsigned char* from = pl.src + a * bytes + off;
    unsigned char* to = pl.dst + b * bytes + off;
    const bool on = is_pair(a, b);
    u.next();
    a = at(u.pair)[0];
    b = at(u.pair)[1];
    if (!on) continue;
    u32x4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (off + e * 1024 < bytes) x[e] = *reinterpret_cast<const u32x4*>(from + e * 1024);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (off + e * 1024 < bytes) *reinterpret_cast<u32x4*>(to + e * 1024) = x[e];
  }
}

// ---- the next step's sequences ----

__device__ __forceinline__ int64_t capacity(const PagesForkParams& p) {
  const int64_t c = p.ldtable << p.lp;
  return c < (1 << 30) ? c : 1 << 30;
}
__device__ __forceinline__ int src_length(const PagesForkParams& p, int s) { return (int)clamp64(p.src_len[s], 0, capacity(p)); }
__device__ __forceinline__ int pages_of(const PagesForkParams& p, int keys) { return (int)(((int64_t)keys + (1 << p.lp) - 1) >> p.lp); }
__device__ __forceinline__ bool is_source(const PagesForkParams& p, int q) { return q >= 0 && q < p.src_seqs; }
// The pages with which a sequence of `keys` keys goes on: those below `pages` that are
// below sink_pages() or from `near` on.
__device__ __forceinline__ int sink_pages(const PagesForkParams& p) { return p.window > 0 ? (int)((p.sinks + (1 << p.lp) - 1) >> p.lp) : 0; }
struct Reach {
  int pages, near;
  __device__ __forceinline__ bool goes_on(int sinks, int64_t k) const { return k < pages && (k < sinks || k >= near); }
};
__device__ __forceinline__ Reach reach_of(const PagesForkParams& p, int keys) {
  const int64_t seen = keys - p.window + 1;  // the first key of the next row's window
  return {pages_of(p, keys), p.window > 0 && seen > 0 ? (int)(seen >> p.lp) : 0};
}
__device__ __forceinline__ int page_id(const PagesForkParams& p, int32_t id) { return id >= 0 && id < p.num_pages ? id : -1; }

// What a source's entry k adds to its page's references: its children hold it, and the
// source does no longer.
__device__ __forceinline__ int change_of(const PagesForkParams& p, Reach r, int sinks, int children, int64_t k) {
  return (r.goes_on(sinks, k) ? children : 0) - (p.keep ? 0 : 1);
}

// STRICT: growth behind the end of a row is a shortage, and a call behind one leaves all but the
// lengths as it is.  Not 0 then; read first and looked at in front of the first write, so that it is no
// trip to memory of its own.  Kernels of their own, as a flag among the arguments is one in calls
// without it (192 sequences 55.2 us, with such a flag 55.8; strict 55.6).
template <bool STRICT>
__device__ __forceinline__ int32_t shortage(const PagesForkParams& p) {
  if constexpr (STRICT) return *p.missing;
  else return 0;
}

// Blocks of sources: references; blocks of sequences: their rows of the table, up to
// the last page that they share.
template <bool STRICT>
__global__ void __launch_bounds__(256) fork_share_kernel(const PagesForkParams p) {
  const int b = blockIdx.x, sinks = sink_pages(p), held = shortage<STRICT>(p);
  if (b >= p.src_seqs) {
    const int i = b - p.src_seqs, q = p.parent[i];
    const Reach r = is_source(p, q) ? reach_of(p, src_length(p, q)) : Reach{0, 0};
    if (held) return;
    for (int64_t k = threadIdx.x; k < p.ldtable; k += 256)
      p.table[i * p.ldtable + k] = r.goes_on(sinks, k) ? page_id(p, p.src_table[q * p.ldtable + k]) : -1;
    return;
  }
  __shared__ int children;
  if (threadIdx.x == 0) children = 0;
  __syncthreads();
  int mine = 0;
  for (int i = threadIdx.x; i < p.seqs; i += 256) mine += p.parent[i] == b;
  if (mine) atomicAdd(&children, mine);
  __syncthreads();
  const Reach r = reach_of(p, src_length(p, b));
  const int all = children;
  if (held) return;
  for (int64_t k = threadIdx.x; k < p.ldtable; k += 256) {
    const int by = change_of(p, r, sinks, all, k);
    const int id = by ? page_id(p, p.src_table[b * p.ldtable + k]) : -1;
    if (id >= 0) atomicAdd(p.refs + id, by);
  }
}

// The workspace: the number of copies, the pairs to copy, and for pages that several
// sequences may be about to write on, how many those are and which is the first.
__device__ __forceinline__ int32_t* ws_pairs(const PagesForkParams& p) { return p.ws + 4; }
__device__ __forceinline__ int32_t* ws_writers(const PagesForkParams& p) { return p.ws + 4 + 2 * p.seqs; }
__device__ __forceinline__ int32_t* ws_first(const PagesForkParams& p) { return ws_writers(p) + p.num_pages; }

// What one block writes and reads again, past its L1.
__device__ __forceinline__ int32_t peek(const int32_t* x) { return __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void poke(int32_t* x, int32_t v) { __hip_atomic_store(x, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// ... behind everything that it wrote so far.
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
}

// Inclusive sum over a wave by lane moves: within rows of 16, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ int plus_moved(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_upto(int v) {
  v = plus_moved<0x111, 0xF>(v);  // from 1, 2, 4, 8 lanes below
  v = plus_moved<0x112, 0xF>(v);
  v = plus_moved<0x114, 0xF>(v);
  v = plus_moved<0x118, 0xF>(v);
  v = plus_moved<0x142, 0xA>(v);  // the sum of the row below, to rows 1 and 3
  return plus_moved<0x143, 0xC>(v);  // of the lower half, to the upper
}
// ... and over a block of 1024: the first wave sums up to N * 16 waves' sums, in LDS.
template <int N>
struct WaveSums {
  int sum[N * 16], total;
  __device__ __forceinline__ void put(int n, int v) { sum[n * 16 + (threadIdx.x >> 6)] = v; }  // by one lane
  // Then, for all: before(n), the sum of what was put before the wave's n-th.
  __device__ __forceinline__ void add_up() {
    __syncthreads();
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x, v = lane < N * 16 ? sum[lane] : 0, upto = wave_upto(v);
      if (lane < N * 16) sum[lane] = upto - v;
      if (lane == 63) total = upto;
    }
    __syncthreads();
  }
  __device__ __forceinline__ int before(int n) const { return sum[n * 16 + (threadIdx.x >> 6)]; }
};

// One block: who copies its last page, how many pages each sequence takes, the lowest
// free pages, dealt out in order.  SHARE: what fork_share_kernel does, too, which saves a
// launch where there is little of it.
// Sequences with the same last page are counted in an LDS table of pages, for up to kTake
// of them, and in the workspace beyond (three trips to memory: 2 us).
constexpr int kTake = 1024, kRound = 4, kSlots = 2048;
template <bool SHARE, bool STRICT>
__global__ void __launch_bounds__(kTake) fork_take_kernel(const PagesForkParams p) {
  __shared__ int start[kForkSeqs];  // pages taken before sequence i; bit 31: its first is a copy
  __shared__ int held[kForkSeqs];   // its parent's keys
  __shared__ int lasts[kForkSeqs];  // the page that it goes on writing, or -1
  __shared__ int source[SHARE ? 2 * kTake : 1];  // SHARE: a source's keys, its children
  __shared__ int slots[3 * kSlots];              // a page, how many write on it, the first of them
  __shared__ WaveSums<kRound> sums;
  __shared__ int copies;
  __shared__ unsigned long long past;  // STRICT: pages behind the ends of rows
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, part = (1 << p.lp) - 1;
  const bool few = p.seqs <= kTake;
  const int before = shortage<STRICT>(p);
  auto hold = [&] {
    for (int i = t; i < p.seqs; i += kTake) p.len[i] = 0;
    if (t == 0) p.ws[0] = 0;
  };
  if (t == 0) {
    copies = 0;
    if constexpr (STRICT) past = 0;
  }
  if (few)
    for (int i = t; i < kSlots; i += kTake) {
      slots[i] = -1;
      slots[kSlots + i] = 0;
      slots[2 * kSlots + i] = p.seqs;
    }
  int own_parent = -1, own_grow = 0;
  if constexpr (SHARE) {  // (a source and a sequence at most to a thread)
    if (t < p.seqs) {
      own_parent = p.parent[t];
      own_grow = p.grow ? p.grow[t] : 0;
    }
    const bool on = is_source(p, own_parent);
    source[t] = t < p.src_seqs ? src_length(p, t) : 0;
    source[kTake + t] = 0;
    __syncthreads();
    if (on) atomicAdd(&source[kTake + own_parent], 1);
    if (t < p.seqs) {
      held[t] = on ? source[own_parent] : 0;
      start[t] = own_parent;  // for now
      lasts[t] = -1;
    }
    __syncthreads();
    if (before) return hold();
    const int width = (int)p.ldtable, entries = p.seqs * width, sources = p.src_seqs * width, sinks = sink_pages(p);
    const int most = entries > sources ? entries : sources;
    constexpr int B = 4;  // entries of either table under way
    for (int w0 = wave * 64; w0 < most; w0 += B * kTake) {
      int id[B], gone[B], by[B];
#pragma unroll
      for (int e = 0; e < B; ++e) {
        id[e] = gone[e] = -1;
        if (w0 + e * kTake >= most) break;  // (the wave as one)
        const int at = w0 + e * kTake + lane, row = fastdiv(at, p.by_width), k = at - row * width;
        if (at < entries && reach_of(p, held[row]).goes_on(sinks, k)) id[e] = p.src_table[start[row] * width + k];
        by[e] = at < sources ? change_of(p, reach_of(p, source[row]), sinks, source[kTake + row], k) : 0;
        if (by[e]) gone[e] = p.src_table[at];
      }
#pragma unroll
      for (int e = 0; e < B; ++e) {
        if (w0 + e * kTake >= most) break;
        const int at = w0 + e * kTake + lane;
        if (at < entries) {
          const int row = fastdiv(at, p.by_width), page = page_id(p, id[e]);
          p.table[at] = page;
          if (at - row * width == held[row] >> p.lp && (held[row] & part)) lasts[row] = page;
        }
        gone[e] = page_id(p, gone[e]);
        if (gone[e] >= 0) atomicAdd(p.refs + gone[e], by[e]);
      }
    }
    settle();
  }
  if (!SHARE && before) return hold();
  int64_t behind = 0;  // STRICT: pages behind the ends of the thread's rows
  // every sequence's growth; start[i]: the pages behind its last
  for (int i = t; i < p.seqs; i += kTake) {
    const int q = SHARE ? own_parent : p.parent[i], more = !is_source(p, q) ? 0 : SHARE ? own_grow : p.grow ? p.grow[i] : 0;
    int have;
    if constexpr (SHARE) have = held[i];
    else held[i] = have = is_source(p, q) ? src_length(p, q) : 0;
    const int64_t want = (int64_t)have + (more > 0 ? more : 0);
    const int now = (int)clamp64(want, 0, capacity(p));
    if (STRICT && want > now) behind += ((want + part) >> p.lp) - pages_of(p, now);
    if (now == have) lasts[i] = -1;
    else if constexpr (!SHARE) lasts[i] = have & part ? p.table[i * p.ldtable + (have >> p.lp)] : -1;
    start[i] = pages_of(p, now) - pages_of(p, have);
    p.len[i] = now;
  }
  int32_t *pairs = ws_pairs(p), *writers = ws_writers(p), *first = ws_first(p);
  uint32_t slot = 0;
  if (few) {
    if constexpr (!SHARE) __syncthreads();  // the slots are clear
    const int last = t < p.seqs ? lasts[t] : -1;
    if (last >= 0) {
      slot = (uint32_t)last * 2654435761u >> 21;
      for (;; slot = (slot + 1) & (kSlots - 1)) {  // (twice as many as sequences)
        const int who = atomicCAS(&slots[slot], -1, last);
        if (who == -1 || who == last) break;
      }
      atomicAdd(&slots[kSlots + slot], 1);
      atomicMin(&slots[2 * kSlots + slot], t);
    }
  } else {
    for (int i = t; i < p.seqs; i += kTake)
      if (lasts[i] >= 0) {
        poke(writers + lasts[i], 0);
        poke(first + lasts[i], p.seqs);
      }
    settle();
    for (int i = t; i < p.seqs; i += kTake)
      if (lasts[i] >= 0) {
        atomicAdd(writers + lasts[i], 1);
        atomicMin(first + lasts[i], i);
      }
    settle();
  }
  if (STRICT && behind > 0) atomicAdd(&past, (unsigned long long)behind);
  const int mine0 = t < p.seqs && lasts[t] >= 0 ? peek(p.refs + lasts[t]) : 1;  // of the thread's first sequence
  // A round of the search for free pages; the first one's loads go out here.
  uint64_t free[kRound];
  auto look = [&](int64_t p0) {
    bool is[kRound];
#pragma unroll
    for (int e = 0; e < kRound; ++e) {
      const int64_t at = p0 + e * kTake + t;
      is[e] = at < p.num_pages && peek(p.refs + at) <= 0;
    }
#pragma unroll
    for (int e = 0; e < kRound; ++e) free[e] = __builtin_amdgcn_ballot_w64(is[e]);
  };
  look(0);
  __syncthreads();
  int need = 0;
  for (int i0 = 0; i0 < p.seqs; i0 += kTake) {
    const int i = i0 + t;
    int mine = 0;
    bool copy = false;
    if (i < p.seqs) {
      const int last = lasts[i];
      if (last >= 0) {
        const int refs = i0 == 0 ? mine0 : peek(p.refs + last);
        const int n = few ? slots[kSlots + slot] : peek(writers + last), least = few ? slots[2 * kSlots + slot] : peek(first + last);
        copy = !(refs == n && least == i);
      }
      mine = start[i] + copy;
    }
    const int upto = wave_upto(mine);
    if (lane == 63) sums.put(0, upto);
    if (lane < kRound - 1) sums.put(lane + 1, 0);
    sums.add_up();
    if (i < p.seqs) start[i] = (need + sums.before(0) + upto - mine) | (copy ? 1 << 31 : 0);
    need += sums.total;
    __syncthreads();
  }
  // the k-th page taken: its sequence is the last that starts at or before k
  auto take = [&](int k, int page) {
    int lo = 0, hi = p.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((start[mid] & 0x7fffffff) <= k) lo = mid;
      else hi = mid;
    }
    const int j = k - (start[lo] & 0x7fffffff);
    const bool partial = start[lo] < 0;
    p.table[lo * p.ldtable + (partial ? held[lo] >> p.lp : pages_of(p, held[lo])) + j] = page;
    p.refs[page] = 1;
    if (partial && j == 0) {
      const int c = atomicAdd(&copies, 1);
      pairs[2 * c] = lasts[lo];
      pairs[2 * c + 1] = page;
      atomicAdd(p.refs + lasts[lo], -1);
    }
  };
  // what a round finds: before which page of the wave's n-th 64 how many lie, and how many there are
  auto add_up = [&] {
    if (lane == 0)
#pragma unroll
      for (int e = 0; e < kRound; ++e) sums.put(e, __popcll(free[e]));
    sums.add_up();
  };
  auto give = [&](int64_t p0, int found) {
#pragma unroll
    for (int e = 0; e < kRound; ++e) {
      const int k = found + sums.before(e) + __popcll(free[e] & ((1ull << lane) - 1));
      if ((free[e] >> lane & 1) && k < need) take(k, (int)(p0 + e * kTake + t));
    }
  };
  // Nothing is given out before there is enough, so that a call without changes nothing:
  // what is needed lies in the first round, mostly, or is looked for twice.
  int found = 0;
  int64_t p0 = 0;
  while (need > 0) {
    add_up();
    found += sums.total;
    if (found >= need || p0 + kRound * kTake >= p.num_pages) break;
    p0 += kRound * kTake;
    look(p0);
    __syncthreads();
  }
  if (found < need || (STRICT && past)) {  // nothing is taken, and what the sources held is theirs again
    for (int64_t k = t; k < p.seqs * p.ldtable; k += kTake) p.table[k] = -1;
    for (int i = t; i < p.seqs; i += kTake) p.len[i] = 0;
    for (int q = wave; q < p.src_seqs; q += kTake / 64) {
      int children = 0;
      for (int i0 = 0; i0 < p.seqs; i0 += 64) children += __popcll(__builtin_amdgcn_ballot_w64(i0 + lane < p.seqs && p.parent[i0 + lane] == q));
      const Reach r = reach_of(p, src_length(p, q));
      for (int64_t k = lane; k < p.ldtable; k += 64) {
        const int by = change_of(p, r, sink_pages(p), children, k);
        const int id = by ? page_id(p, p.src_table[q * p.ldtable + k]) : -1;
        if (id >= 0) atomicAdd(p.refs + id, -by);
      }
    }
  } else if (need > 0 && p0 == 0) {
    give(0, 0);
  } else if (need > 0) {
    const int64_t last = p0;
    int upto = 0;
    for (p0 = 0; p0 <= last; p0 += kRound * kTake) {
      __syncthreads();
      look(p0);
      add_up();
      give(p0, upto);
      upto += sums.total;
    }
  }
  __syncthreads();
  if (t == 0) {
    const int lacking = found < need ? need - found : 0;
    if constexpr (STRICT) *p.missing = (int)clamp64(lacking + (int64_t)past, 0, INT32_MAX);
    else *p.missing = lacking;
    p.ws[0] = copies;
  }
}

// ---- used pages to the front ----
//
// The workspace: the number of moves, the used pages of each chunk, the pairs to move,
// their references, and for each page its new number, -1, or -2 - r where it is the
// r-th that moves.
constexpr int kChunk = 4096;
__host__ __device__ __forceinline__ int64_t chunks_of(const PagesCompactParams& p) { return (p.num_pages + kChunk - 1) / kChunk; }
__device__ __forceinline__ int32_t* ws_counts(const PagesCompactParams& p) { return p.ws + 4; }
__device__ __forceinline__ int32_t* ws_moves(const PagesCompactParams& p) { return p.ws + 4 + ((chunks_of(p) + 1) & ~1LL); }
__device__ __forceinline__ int32_t* ws_held(const PagesCompactParams& p) { return ws_moves(p) + (p.num_pages & ~1LL); }
__device__ __forceinline__ int32_t* ws_new(const PagesCompactParams& p) { return ws_held(p) + p.num_pages / 2; }

// All of it in one block, the pages' new numbers in LDS, for a small pool and tables: a
// launch in the place of three.
constexpr int kSmallPool = 4 * 1024, kSmallTable = 16 * 1024;
__global__ void __launch_bounds__(1024) compact_small_kernel(const PagesCompactParams p) {
  constexpr int N = kSmallPool / 1024;
  __shared__ int name[kSmallPool], gaps[kSmallPool / 2];
  __shared__ WaveSums<N> sums;
  const int t = threadIdx.x, lane = t & 63, pages = (int)p.num_pages;
  int32_t* moves = ws_moves(p);
  int refs[N], rank[N];
#pragma unroll
  for (int e = 0; e < N; ++e) refs[e] = e * 1024 + t < pages ? p.refs[e * 1024 + t] : 0;
  uint64_t on[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    on[e] = __builtin_amdgcn_ballot_w64(refs[e] > 0);
    if (lane == 0) sums.put(e, __popcll(on[e]));
  }
  sums.add_up();
  const int used = sums.total;
#pragma unroll
  for (int e = 0; e < N; ++e) rank[e] = sums.before(e) + __popcll(on[e] & ((1ull << lane) - 1));  // used pages in front
  __syncthreads();
  // of those that stay: the used pages among the first `used`
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const uint64_t stay = __builtin_amdgcn_ballot_w64(e * 1024 + t < used && refs[e] > 0);
    if (lane == 0) sums.put(e, __popcll(stay));
    if (e * 1024 + t < used && refs[e] <= 0) gaps[e * 1024 + t - rank[e]] = e * 1024 + t;
  }
  sums.add_up();
  const int front = sums.total;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int at = e * 1024 + t;
    if (at >= pages) continue;
    const bool moved = at >= used && refs[e] > 0;
    const int to = moved ? gaps[rank[e] - front] : refs[e] > 0 ? at : -1;
    name[at] = to;
    if (p.map) p.map[at] = to;
    if (refs[e] > 0) p.refs_out[to] = refs[e];
    if (at >= used) p.refs_out[at] = 0;  // (no page goes there)
    if (moved) {
      moves[2 * (rank[e] - front)] = at;
      moves[2 * (rank[e] - front) + 1] = to;
    }
  }
  __syncthreads();
  for (int i = t; i < (int)p.entries; i += 1024) {
    const int id = p.table[i];
    p.table_out[i] = id >= 0 && id < pages ? name[id] : -1;
  }
  if (t == 0) {
    p.ws[0] = used - front;
    *p.used = used;
  }
}

// Inclusive sum over a block of 1024 (wave sums in LDS).
__device__ __forceinline__ int block_sum(int v, int* waves, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_upto(v);
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const int x = waves[w];
    before += w < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + v;
}

// Used pages among [from, to), by a block of 1024.
__device__ __forceinline__ int count_used(const PagesCompactParams& p, int64_t from, int64_t to, int* waves) {
  int n = 0, all;
  for (int64_t at = from + threadIdx.x; at < to; at += 1024) n += p.refs[at] > 0;
  block_sum(n, waves, &all);
  return all;
}
__global__ void __launch_bounds__(1024) compact_count_kernel(const PagesCompactParams p) {
  __shared__ int waves[16];
  const int64_t from = (int64_t)blockIdx.x * kChunk, to = from + kChunk < p.num_pages ? from + kChunk : p.num_pages;
  const int n = count_used(p, from, to, waves);
  if (threadIdx.x == 0) ws_counts(p)[blockIdx.x] = n;
}
__global__ void __launch_bounds__(1024) compact_plan_kernel(const PagesCompactParams p) {
  __shared__ int waves[16];
  const int64_t chunks = chunks_of(p);
  const int32_t* counts = ws_counts(p);
  auto sum_of = [&](int64_t to) {  // used pages of the first `to` chunks
    int n = 0, all;
    for (int64_t c = threadIdx.x; c < to; c += 1024) n += counts[c];
    block_sum(n, waves, &all);
    return all;
  };
  const int used = sum_of(chunks);
  const int64_t cut = used / kChunk;
  const int front = sum_of(cut) + count_used(p, cut * kChunk, used, waves);  // used pages that stay
  int before = sum_of(blockIdx.x);
  int32_t *moves = ws_moves(p), *held = ws_held(p), *to = ws_new(p);
  for (int e = 0; e < kChunk / 1024; ++e) {
    const int64_t at = (int64_t)blockIdx.x * kChunk + e * 1024 + threadIdx.x;
    const int refs = at < p.num_pages ? p.refs[at] : 0, on = refs > 0;
    int all;
    const int rank = before + block_sum(on, waves, &all) - on;  // used pages in front of it
    before += all;
    if (at >= p.num_pages) continue;
    if (at < used) {
      to[at] = on ? (int32_t)at : -1;
      if (!on) moves[2 * (at - rank) + 1] = (int32_t)at;
    } else {
      to[at] = on ? -2 - (rank - front) : -1;
      if (on) {
        moves[2 * (rank - front)] = (int32_t)at;
        held[rank - front] = refs;
      }
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.ws[0] = used - front;
    p.ws[1] = used;
    *p.used = used;
  }
}
__global__ void __launch_bounds__(256) compact_rename_kernel(const PagesCompactParams p) {
  const int moved = p.ws[0], used = p.ws[1];
  const int32_t *moves = ws_moves(p), *held = ws_held(p), *to = ws_new(p);
  auto name = [&](int64_t id) {
    if (id < 0 || id >= p.num_pages) return -1;
    const int n = to[id];
    return n <= -2 ? moves[2 * (-2 - n) + 1] : n;
  };
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = first; i < p.num_pages; i += step) {
    if (p.map) p.map[i] = name(i);
    if (i >= used) p.refs_out[i] = 0;
    else if (to[i] >= 0) p.refs_out[i] = p.refs[i];
  }
  for (int64_t i = first; i < moved; i += step) p.refs_out[moves[2 * i + 1]] = held[i];
  for (int64_t i = first; i < p.entries; i += step) p.table_out[i] = name(p.table[i]);
}

template <bool STRICT>
void launch_fork(PagesForkParams p, hipStream_t s) {
  // one launch up to 4096 entries, which are under way at once (8.4 us for 200, 13.2 in two
  // launches); 11136 take 57.5 with the copies, 55.5 in two
  const bool little = p.seqs <= kTake && p.src_seqs <= kTake && (p.seqs + p.src_seqs) * p.ldtable <= 4 * kTake;
  if (little) {
    p.by_width = fastdiv_make((uint32_t)(p.ldtable > 0 ? p.ldtable : 1));
    hipLaunchKernelGGL((fork_take_kernel<true, STRICT>), dim3(1), dim3(kTake), 0, s, p);
  } else {
    hipLaunchKernelGGL((fork_share_kernel<STRICT>), dim3(p.src_seqs + p.seqs), dim3(256), 0, s, p);
    hipLaunchKernelGGL((fork_take_kernel<false, STRICT>), dim3(1), dim3(kTake), 0, s, p);
  }
}

}  // namespace

size_t pages_fork_workspace(const PagesForkParams& p) {
  return (4 + 2 * (size_t)p.seqs + (p.seqs > kTake ? 2 * (size_t)p.num_pages : 0)) * 4;
}
size_t pages_compact_workspace(const PagesCompactParams& p) {
  return (size_t)(4 + ((chunks_of(p) + 1) & ~1LL) + (p.num_pages & ~1LL) + p.num_pages / 2 + p.num_pages) * 4;
}

hipError_t launch_pages_copy(const PagePlanes& planes, const PagesCopyParams& p, hipStream_t s) {
  if (planes.n == 0 || p.npairs == 0) return hipSuccess;
  int64_t most = 1;
  for (int i = 0; i < planes.n; ++i) most = most > planes.at[i].bytes ? most : planes.at[i].bytes;
  const double units = (double)p.npairs * (double)((most + kPiece - 1) / kPiece) / 4;
  const double room = 4096.0 / planes.n > 16 ? 4096.0 / planes.n : 16;
  const unsigned x = (unsigned)(units < room ? units + 1 : room);
  hipLaunchKernelGGL(page_copy_kernel, dim3(x, planes.n), dim3(256), 0, s, planes, p);
  return hipGetLastError();
}

hipError_t launch_pages_fork(const PagesForkParams& p, PagesCopyParams* moves, hipStream_t s) {
  if (p.strict) launch_fork<true>(p, s);
  else launch_fork<false>(p, s);
  *moves = {p.ws + 4, p.seqs, p.ws, p.num_pages, p.num_pages};
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesCompactParams& p, PagesCopyParams* moves, hipStream_t s) {
  *moves = {p.ws + 4 + ((chunks_of(p) + 1) & ~1LL), p.num_pages / 2, p.ws, p.num_pages, p.num_pages};
  if (p.num_pages <= kSmallPool && p.entries <= kSmallTable) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(1024), 0, s, p);
    return hipGetLastError();
  }
  const unsigned chunks = (unsigned)chunks_of(p);
  hipLaunchKernelGGL(compact_count_kernel, dim3(chunks), dim3(1024), 0, s, p);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(chunks), dim3(1024), 0, s, p);
  const int64_t most = p.num_pages > p.entries ? p.num_pages : p.entries;
  hipLaunchKernelGGL(compact_rename_kernel, dim3((unsigned)(most / 256 < 1024 ? most / 256 + 1 : 1024)), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace qa

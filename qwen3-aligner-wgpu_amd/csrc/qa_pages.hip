// qa_pages.hip -- a pool's pages: copied, shared and taken for the next step's sequences,
// moved to the front.
#include "qa_internal.h"

namespace qa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- pages from one place to another ----
//
// blockIdx.y is the plane.  A wave takes 4 KB of a page at a time, four 16-byte loads
// in flight for each lane; pages that are no multiple of 16 bytes, and short ones (scales), go
// by words, a lane each.
constexpr int kPiece = 4096;
__global__ void __launch_bounds__(256) page_copy_kernel(const PagePlanes planes, const PagesCopyParams p) {
  const auto& pl = planes.at[blockIdx.y];
  const int64_t count = p.count ? clamp64(*p.count, 0, p.npairs) : p.npairs;
  const int64_t bytes = pl.bytes;
  if (bytes % 16 || bytes < 1024) {
    const int64_t words = bytes / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count * words; i += (int64_t)gridDim.x * 256) {
      const int64_t pair = i / words, w = i - pair * words;
      const int32_t a = p.pairs[2 * pair], b = p.pairs[2 * pair + 1];
      if (a < 0 || a >= p.src_pages || b < 0 || b >= p.dst_pages) continue;
      *reinterpret_cast<uint32_t*>(pl.dst + b * bytes + 4 * w) = *reinterpret_cast<const uint32_t*>(pl.src + a * bytes + 4 * w);
    }
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t pieces = (bytes + kPiece - 1) / kPiece;
  for (int64_t u = (int64_t)blockIdx.x * 4 + wave; u < count * pieces; u += (int64_t)gridDim.x * 4) {
    const int64_t pair = u / pieces;
    const int64_t off = (u - pair * pieces) * kPiece + lane * 16;
    const int32_t a = p.pairs[2 * pair], b = p.pairs[2 * pair + 1];
    if (a < 0 || a >= p.src_pages || b < 0 || b >= p.dst_pages) continue;
    const unsigned char* from = pl.src + a * bytes + off;
    unsigned char* to = pl.dst + b * bytes + off;
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
// Whether a sequence of `keys` keys goes on with page number k of its source.
__device__ __forceinline__ bool goes_on(const PagesForkParams& p, int keys, int64_t k) {
  if (k << p.lp >= keys) return false;
  return p.window <= 0 || k << p.lp < p.sinks || ((k + 1) << p.lp) > keys - p.window + 1;
}
__device__ __forceinline__ int page_id(const PagesForkParams& p, int32_t id) { return id >= 0 && id < p.num_pages ? id : -1; }

// What source s's entry k adds to its page's references: its children hold it, and the
// source does no longer.
__device__ __forceinline__ int change_of(const PagesForkParams& p, int keys, int children, int64_t k) {
  return (goes_on(p, keys, k) ? children : 0) - (p.keep ? 0 : 1);
}

// Blocks of sources: references; blocks of sequences: their rows of the table, up to
// the last page that they share.
__global__ void __launch_bounds__(256) fork_share_kernel(const PagesForkParams p) {
  const int b = blockIdx.x;
  if (b >= p.src_seqs) {
    const int i = b - p.src_seqs, q = p.parent[i];
    const bool on = is_source(p, q);
    const int keys = on ? src_length(p, q) : 0;
    for (int64_t k = threadIdx.x; k < p.ldtable; k += 256)
      p.table[i * p.ldtable + k] = on && goes_on(p, keys, k) ? page_id(p, p.src_table[q * p.ldtable + k]) : -1;
    return;
  }
  __shared__ int children;
  if (threadIdx.x == 0) children = 0;
  __syncthreads();
  int mine = 0;
  for (int i = threadIdx.x; i < p.seqs; i += 256) mine += p.parent[i] == b;
  if (mine) atomicAdd(&children, mine);
  __syncthreads();
  const int keys = src_length(p, b), all = children;
  for (int64_t k = threadIdx.x; k < p.ldtable; k += 256) {
    const int by = change_of(p, keys, all, k);
    const int id = page_id(p, p.src_table[b * p.ldtable + k]);
    if (by && id >= 0) atomicAdd(p.refs + id, by);
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

struct Growth {
  int have, now, last;  // keys before and behind; the page that is written on, or -1
};
__device__ __forceinline__ Growth growth(const PagesForkParams& p, int i) {
  const int q = p.parent[i];
  Growth g = {0, 0, -1};
  if (!is_source(p, q)) return g;
  g.have = src_length(p, q);
  const int more = p.grow ? p.grow[i] : 0;
  g.now = (int)clamp64((int64_t)g.have + (more > 0 ? more : 0), 0, capacity(p));
  if ((g.have & ((1 << p.lp) - 1)) && g.now > g.have) g.last = p.table[i * p.ldtable + (g.have >> p.lp)];
  return g;
}

// Inclusive sum over a block of 1024 (wave sums in LDS).
__device__ __forceinline__ int block_sum(int v, int* waves, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int e = 1; e < 64; e <<= 1) {
    const int x = __shfl_up(v, e, 64);
    v += lane >= e ? x : 0;
  }
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

// One block: who copies its last page, how many pages each sequence takes, the lowest
// free pages, dealt out in order.
constexpr int kTake = 1024, kRound = 4;
__global__ void __launch_bounds__(kTake) fork_take_kernel(const PagesForkParams p) {
  __shared__ int start[kForkSeqs + 1];  // pages taken before sequence i; bit 31: its first is a copy
  __shared__ int waves[kRound * 16];
  int32_t *pairs = ws_pairs(p), *writers = ws_writers(p), *first = ws_first(p);
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int i = t; i < p.seqs; i += kTake) {
    const Growth g = growth(p, i);
    if (g.last < 0) continue;
    poke(writers + g.last, 0);
    poke(first + g.last, p.seqs);
  }
  __syncthreads();
  for (int i = t; i < p.seqs; i += kTake) {
    const Growth g = growth(p, i);
    if (g.last < 0) continue;
    atomicAdd(writers + g.last, 1);
    atomicMin(first + g.last, i);
  }
  __syncthreads();
  int need = 0, copies = 0;  // so far, of all
  for (int i0 = 0; i0 < p.seqs; i0 += kTake) {
    const int i = i0 + t;
    int mine = 0;
    bool copy = false;
    if (i < p.seqs) {
      const Growth g = growth(p, i);
      copy = g.last >= 0 && !(p.refs[g.last] == peek(writers + g.last) && peek(first + g.last) == i);
      mine = pages_of(p, g.now) - pages_of(p, g.have) + copy;
      p.len[i] = g.now;
    }
    int all, each;
    const int upto = block_sum(mine, waves, &all), number = block_sum(copy, waves, &each);
    if (i < p.seqs) start[i] = (need + upto - mine) | (copy ? 1 << 31 : 0);
    if (copy) {  // the page and, for now, the sequence
      const int c = copies + number - 1;
      pairs[2 * c] = p.table[i * p.ldtable + (src_length(p, p.parent[i]) >> p.lp)];
      pairs[2 * c + 1] = i;
    }
    need += all;
    copies += each;
  }
  __syncthreads();
  auto place = [&](int k) {  // the entry of the k-th page taken: its sequence is the last that starts at or before k
    int lo = 0, hi = p.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((start[mid] & 0x7fffffff) <= k) lo = mid;
      else hi = mid;
    }
    const int have = src_length(p, p.parent[lo]), j = k - (start[lo] & 0x7fffffff);
    return lo * p.ldtable + (start[lo] < 0 ? have >> p.lp : pages_of(p, have)) + j;
  };
  int found = 0;
  for (int64_t p0 = 0; p0 < p.num_pages && found < need; p0 += kRound * kTake) {
    uint64_t free[kRound];
#pragma unroll
    for (int e = 0; e < kRound; ++e) {
      const int64_t at = p0 + e * kTake + t;
      free[e] = __builtin_amdgcn_ballot_w64(at < p.num_pages && p.refs[at] <= 0);
      if (lane == 0) waves[e * 16 + wave] = __popcll(free[e]);
    }
    __syncthreads();
    int all = found;
#pragma unroll
    for (int e = 0; e < kRound; ++e) {
      int k = all + __popcll(free[e] & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const int x = waves[e * 16 + w];
        k += w < wave ? x : 0;
        all += x;
      }
      if ((free[e] >> lane & 1) && k < need) p.table[place(k)] = (int32_t)(p0 + e * kTake + t);
    }
    found = all;
    __syncthreads();
  }
  if (found < need) {  // nothing is taken, and what the sources held is theirs again
    for (int64_t k = t; k < p.seqs * p.ldtable; k += kTake) p.table[k] = -1;
    for (int i = t; i < p.seqs; i += kTake) p.len[i] = 0;
    for (int q = wave; q < p.src_seqs; q += kTake / 64) {
      int children = 0;
      for (int i0 = 0; i0 < p.seqs; i0 += 64) children += __popcll(__builtin_amdgcn_ballot_w64(i0 + lane < p.seqs && p.parent[i0 + lane] == q));
      const int keys = src_length(p, q);
      for (int64_t k = lane; k < p.ldtable; k += 64) {
        const int by = change_of(p, keys, children, k);
        const int id = page_id(p, p.src_table[q * p.ldtable + k]);
        if (by && id >= 0) atomicAdd(p.refs + id, -by);
      }
    }
  } else {
    for (int k = t; k < need; k += kTake) p.refs[p.table[place(k)]] = 1;
    for (int c = t; c < copies; c += kTake) {
      const int old = pairs[2 * c], i = pairs[2 * c + 1];
      atomicAdd(p.refs + old, -1);
      pairs[2 * c + 1] = p.table[i * p.ldtable + (src_length(p, p.parent[i]) >> p.lp)];
    }
  }
  if (t == 0) {
    *p.missing = found < need ? need - found : 0;
    p.ws[0] = found < need ? 0 : copies;
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

}  // namespace

size_t pages_fork_workspace(const PagesForkParams& p) { return (4 + 2 * (size_t)p.seqs + 2 * (size_t)p.num_pages) * 4; }
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
  if (p.src_seqs + p.seqs > 0) hipLaunchKernelGGL(fork_share_kernel, dim3(p.src_seqs + p.seqs), dim3(256), 0, s, p);
  hipLaunchKernelGGL(fork_take_kernel, dim3(1), dim3(kTake), 0, s, p);
  *moves = {p.ws + 4, p.seqs, p.ws, p.num_pages, p.num_pages};
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesCompactParams& p, PagesCopyParams* moves, hipStream_t s) {
  const unsigned chunks = (unsigned)chunks_of(p);
  hipLaunchKernelGGL(compact_count_kernel, dim3(chunks), dim3(1024), 0, s, p);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(chunks), dim3(1024), 0, s, p);
  const int64_t most = p.num_pages > p.entries ? p.num_pages : p.entries;
  hipLaunchKernelGGL(compact_rename_kernel, dim3((unsigned)(most / 256 < 1024 ? most / 256 + 1 : 1024)), dim3(256), 0, s, p);
  *moves = {p.ws + 4 + ((chunks_of(p) + 1) & ~1LL), p.num_pages / 2, p.ws, p.num_pages, p.num_pages};
  return hipGetLastError();
}

}  // namespace qa

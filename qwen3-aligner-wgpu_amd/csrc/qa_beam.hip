// qa_beam.hip -- the step of a beam search: for each group the `width` best of
// score[b] + x[b][t] - log sum_t' exp x[b][t'] over its beams b and the vocabulary t.
//
// Within a row the order is that of the logits, so a first launch needs each logit
// once: a block takes a chunk of a row, and leaves its maximum, its sum of exponentials and
// its `width` largest logits in the workspace.  A second one, a block for each group,
// joins the sums in f64 and ranks the chunks' candidates, in f64 too: an f32 sum of
// a score near -50 and a log-probability has steps of 4e-6, and candidates that differ
// by less would change places.  What is left of that is the chunks' f32 sums, at most 6e-6 of a
// row's logarithm: it moves a beam's candidates together, so that those of one beam keep
// their order, and only those of two that are as close can change places.  Equal ones go by
// (beam, token), so every comparison is of (value, index) pairs of which no two are alike:
// results do not depend on timing.
//
// 192 rows of 151936 f16 logits, the best 8 of 8 beams: 20.7 us, the chunks 15.6 (58 MB at 3.7
// TB/s: loads and maxima alone take 11.4, the exponentials 2 more, the lists and their
// ranks the rest), the join 4.7; in f32 29.4, 117 MB.  4 rows: 9.9 us, two launches and 5 trips to
// memory.
#include "qa_internal.h"

namespace qa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kThreads = 256;

// A candidate as one number: the larger logit first, then the lower token; 0 is behind all.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 is 0
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

// The workspace: each chunk's maximum and sum of exponentials (0 where it has none), then
// the keys of each chunk's candidates, best first, 0 behind the last.
struct Stat {
  float top, sum;
};
// A barrier for what waves exchange through LDS: loads and stores of memory go on across
// it, where __syncthreads() waits for them.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4) | (0x0 << 8));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Logits of a thread, by how many there are in all: 8 below 0.5 M, 16 below 3 M, 32 beyond.  Small
// chunks are more blocks and longer lists to merge (us with 8 / 16 / 32: 8 rows of 60000 9.8 / 9.8 /
// 10.3, 64 of 12000 9.7 / 10.2 / 11.3, 4 of 151936 11.0 / 10.2 / 10.2, 12 of them 13.4 / 11.6 / 11.7,
// 24 14.4 / 11.9 / 11.3, 192 39.7 / 27.9 / 22.8; 192 of 12000 10.8 / 10.8 / 11.6, of 32000 15.0 / 13.2 / 12.5;
// with the ranks and the join as they were, what was 22.8 is 20.7 now).
int each_of(const BeamParams& p) {
  const int64_t all = p.groups * p.beams * p.vocab;
  return all < 500000 ? 8 : all < 3000000 ? 16 : 32;
}
int64_t chunks_of(const BeamParams& p) { return (p.vocab + kThreads * each_of(p) - 1) / (kThreads * each_of(p)); }
int chunk_of(const BeamParams& p) { return (int)(((p.vocab + chunks_of(p) - 1) / chunks_of(p) + 7) & ~7LL); }
__device__ __forceinline__ Stat* stats(const BeamParams& p) { return (Stat*)p.ws; }
__device__ __forceinline__ uint64_t* cands(const BeamParams& p, int64_t chunks) { return (uint64_t*)(stats(p) + p.groups * p.beams * chunks); }

// A beam that has no continuations of its own: none, or ended.
__device__ __forceinline__ bool is_none(float score) { return !(score > -INFINITY && score < INFINITY); }

template <class V, class I>
__device__ __forceinline__ bool before(V v, I i, V w, I j) {
  return v > w || (v == w && i < j);
}

// f over the lanes whose numbers have the lowest bits of `apart`, a power of two from 1
// (all of them) to 64, in common; by lane moves.
template <int CTRL>
__device__ __forceinline__ float moved(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <class F>
__device__ __forceinline__ float over_lanes(float x, int apart, F f) {
  if (apart <= 1) x = f(x, moved<0x121>(x));  // a row of 16 turned by 1, by 2 ..
  if (apart <= 2) x = f(x, moved<0x122>(x));
  if (apart <= 4) x = f(x, moved<0x124>(x));
  if (apart <= 8) x = f(x, moved<0x128>(x));
  if (apart <= 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (apart <= 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return x;
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }

// A thread's logits of a chunk: kEach / N runs of N, a run of 16 bytes.
template <int DT>
constexpr int kRun = DT == QA_F32 ? 4 : 8;
template <int DT>
__device__ __forceinline__ float logit(const void* row, int64_t t) {
  if constexpr (DT == QA_F32) return ((const float*)row)[t];
  else if constexpr (DT == QA_F16) return (float)((const _Float16*)row)[t];
  else return __uint_as_float((uint32_t)((const uint16_t*)row)[t] << 16);
}
template <int DT>
__device__ __forceinline__ void unpack(u32x4 w, float* x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == QA_F32) {
      x[e] = __uint_as_float(w[e]);
    } else if constexpr (DT == QA_F16) {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      const uint32_t word = w[e];  // (a bit cast of the vector's element itself reads its first)
      const h2 h = __builtin_bit_cast(h2, word);
      x[2 * e] = (float)h[0];
      x[2 * e + 1] = (float)h[1];
    } else {
      x[2 * e] = __uint_as_float(w[e] << 16);
      x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
}

// The best `width` of a block's logits: the threads are taken as 4 to 64 groups, at least
// `width` of them (every 4th to every 64th thread, so that a short chunk's have logits in
// all), and what is below the least of the groups' best cannot be among them.  The
// others, about width * log width, are listed in LDS, each wave's apart (a shared counter
// is a trip to the LDS for each of them), and each one's rank is the number of those
// before it.  More than a wave's list holds, which many equal numbers can be, go by rounds
// of the block.
constexpr int kList = 256;
__device__ __forceinline__ int groups_of(int width) { return width <= 4 ? 4 : width <= 8 ? 8 : width <= 16 ? 16 : width <= 32 ? 32 : 64; }

template <int DT, int EACH>
__global__ void __launch_bounds__(kThreads) beam_chunk_kernel(const BeamParams p, int chunks, int chunk_len) {
  constexpr int N = kRun<DT>, RUNS = EACH / N, ES = DT == QA_F32 ? 4 : 2;
  constexpr float kLowest = -3.402823466e38f;
  __shared__ float best[kThreads / 64][64], vs[kThreads / 64];
  __shared__ int is[kThreads / 64], ranks[kThreads / 64][64], lengths[kThreads / 64];
  __shared__ __attribute__((aligned(16))) uint64_t lists[kThreads / 64][kList + 8];
  asm volatile("" ::"s"(p.logits), "s"(p.width), "s"(chunks));  // the arguments in one trip to memory
  __builtin_amdgcn_sched_barrier(0);
  const int t = threadIdx.x, lane = t & 63, groups = groups_of(p.width);
  const int row = blockIdx.x / (uint32_t)chunks;
  const int64_t first = (int64_t)(blockIdx.x - row * chunks) * chunk_len;
  const int t0 = (int)(first < p.vocab ? first : p.vocab), len = (int)(p.vocab - t0 < chunk_len ? p.vocab - t0 : chunk_len);
  const char* src = (const char*)p.logits + (row * p.ldl + t0) * ES;
  const float score = p.score[row];
  const int over = (p.done ? p.done : (const int32_t*)p.score)[row];  // (no branch in front of the loads)
  // all loads first, of the chunk's first run where a thread has none
  u32x4 raw[RUNS] = {};
  if (len >= N)
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      const int at = (r * kThreads + t) * N;
      raw[r] = *reinterpret_cast<const u32x4*>(src + (uint32_t)(at + N <= len ? at * ES : 0));
    }
  if (is_none(score) || (p.done && over)) return;
  float x[EACH];
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    unpack<DT>(raw[r], x + r * N);
    const int at = (r * kThreads + t) * N;
    if (at + N > len)
#pragma unroll
      for (int e = 0; e < N; ++e) x[r * N + e] = at + e < len ? logit<DT>(src, at + e) : -INFINITY;
  }
  auto token = [&](int j) { return t0 + (j / N * kThreads + t) * N + j % N; };
  float own, top, least, sum;
  for (;;) {
    own = -INFINITY;
#pragma unroll
    for (int j = 0; j < EACH; ++j) own = fmaxf(own, x[j]);  // NaN is not the larger
    best[t >> 6][lane] = over_lanes(own, groups, larger);
    lds_barrier();
    const float m = fmaxf(fmaxf(best[0][lane], best[1][lane]), fmaxf(best[2][lane], best[3][lane]));
    top = over_lanes(m, 1, larger);
    least = fmaxf(over_lanes(m, 1, smaller), kLowest);
    const float off = top == -INFINITY ? 0.f : top;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < EACH; ++j) part[j & 3] += __builtin_amdgcn_exp2f((x[j] - off) * kLog2e);
    sum = over_lanes((part[0] + part[1]) + (part[2] + part[3]), 1, sum_of);
    if (lane == 0) vs[t >> 6] = sum;
    lds_barrier();
    sum = (vs[0] + vs[1]) + (vs[2] + vs[3]);
    if (sum < INFINITY) break;
    // a NaN, or an infinity, from which it is NaN: again without
#pragma unroll
    for (int j = 0; j < EACH; ++j) x[j] = x[j] < INFINITY ? x[j] : -INFINITY;
  }
  if (t == 0) stats(p)[blockIdx.x] = {top, sum};
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int mine_n = 0;  // the wave as one
#pragma unroll
  for (int j0 = 0; j0 < EACH; j0 += 4)
    if (__builtin_amdgcn_ballot_w64(fmaxf(fmaxf(x[j0], x[j0 + 1]), fmaxf(x[j0 + 2], x[j0 + 3])) >= least))
#pragma unroll
      for (int j = j0; j < j0 + 4; ++j)
        if (const uint64_t who = __builtin_amdgcn_ballot_w64(x[j] >= least)) {
          const int at = mine_n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
          if (x[j] >= least && at < kList) lists[wave][at] = key_of(x[j], token(j));
          mine_n += __popcll(who);
        }
  if (lane < 8 && mine_n <= kList) lists[wave][mine_n + lane] = 0;  // behind the last
  if (lane == 0) lengths[wave] = mine_n;
  lds_barrier();
  uint64_t* out = cands(p, chunks) + (int64_t)blockIdx.x * p.width;
  int ends[kThreads / 64], longest = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const int n = __builtin_amdgcn_readfirstlane(lengths[w]);
    longest = n > longest ? n : longest;
    ends[w] = n + (w ? ends[w - 1] : 0);
  }
  const int n = ends[kThreads / 64 - 1];
  // candidate number c of all
  auto listed = [&](int c) {
    int w = 0, first = 0;
#pragma unroll
    for (int v = 1; v < kThreads / 64; ++v)
      if (c >= ends[v - 1]) {
        w = v;
        first = ends[v - 1];
      }
    return lists[w][c - first];
  };
  if (n <= 64) {  // a lane for each, compared with a quarter of the others by each wave
    const uint64_t mine = lane < n ? listed(lane) : 0;
    int rank = 0;
    for (int k = wave; k < n; k += kThreads / 64) {
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), k) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, k);
      rank += other > mine;
    }
    ranks[wave][lane] = rank;
    lds_barrier();
    if (t < 64) {
      rank = lane < n ? (ranks[0][lane] + ranks[1][lane]) + (ranks[2][lane] + ranks[3][lane]) : lane;
      if (rank < p.width) out[rank] = mine;
    }
  } else if (longest <= kList) {  // a thread for each, eight of the others at once
    for (int c = t; c < n; c += kThreads) {
      const uint64_t mine = listed(c);
      int rank = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w)
        for (int k = 0; k < ends[w] - (w ? ends[w - 1] : 0); k += 8) {
          u64x2 other[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) other[e] = *reinterpret_cast<const u64x2*>(lists[w] + k + 2 * e);
#pragma unroll
          for (int e = 0; e < 4; ++e) rank += (other[e][0] > mine) + (other[e][1] > mine);
        }
      if (rank < p.width) out[rank] = mine;
    }
  } else {
    // the thread's best that comes behind (v, i); read again: held until here, the logits
    // would take registers of which the CU's other blocks live
    auto next = [&](float v, int i, float* bv, int* bi) {
      *bv = -INFINITY;
      *bi = INT32_MAX;
      for (int k = t; k < len; k += kThreads) {
        const float y = logit<DT>(src, k);
        if (y < INFINITY && before(v, i, y, t0 + k) && y > *bv) {
          *bv = y;
          *bi = t0 + k;
        }
      }
    };
    int at;
    next(INFINITY, -1, &own, &at);
    for (int k = 0; k < p.width; ++k) {
      float v = own;
      int i = at;
#pragma unroll
      for (int e = 32; e > 0; e >>= 1) {
        const float w = __shfl_xor(v, e, 64);
        const int j = __shfl_xor(i, e, 64);
        if (before(w, j, v, i)) {
          v = w;
          i = j;
        }
      }
      lds_barrier();
      if (lane == 0) {
        vs[t >> 6] = v;
        is[t >> 6] = i;
      }
      lds_barrier();
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w)
        if (before(vs[w], is[w], v, i)) {
          v = vs[w];
          i = is[w];
        }
      if (t == 0) out[k] = key_of(v, i);
      if (at == i) next(v, i, &own, &at);
    }
  }
}

// What lane ^ D holds, by lane moves: rows of 16 turned or mirrored, fours permuted, rows and
// halves swapped.
template <int D>
__device__ __forceinline__ uint32_t from_lane(uint32_t x) {
  constexpr int HI = D >> 2 & 3, LO = (D ^ (HI & 1 ? 3 : 0)) & 3;  // mirrors of 8 and of 16 turn fours round
  constexpr int ROW = HI == 1 ? 0x141 : HI == 2 ? 0x128 : 0x140;
  constexpr int FOUR = (LO ^ 0) | (LO ^ 1) << 2 | (LO ^ 2) << 4 | (LO ^ 3) << 6;
  if constexpr (HI != 0) x = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, ROW, 0xF, 0xF, true);
  if constexpr (LO != 0) x = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, FOUR, 0xF, 0xF, true);
  if constexpr ((D & 16) != 0) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = threadIdx.x & 16 ? r[0] : r[1];
  }
  if constexpr ((D & 32) != 0) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = threadIdx.x & 32 ? r[0] : r[1];
  }
  return x;
}
template <int D>
__device__ __forceinline__ uint64_t from_lane(uint64_t x) {
  return (uint64_t)from_lane<D>((uint32_t)(x >> 32)) << 32 | from_lane<D>((uint32_t)x);
}
template <int D>
__device__ __forceinline__ double from_lane(double x) {
  return __builtin_bit_cast(double, from_lane<D>(__builtin_bit_cast(uint64_t, x)));
}
// A continuation of a group: its value, and its beam and rank there as one number, the lower first.
struct Total {
  double v;
  uint32_t at;
};
template <int D>
__device__ __forceinline__ Total from_lane(Total x) {
  return {from_lane<D>(x.v), from_lane<D>(x.at)};
}
__device__ __forceinline__ bool better(uint64_t a, uint64_t b) { return a > b; }
__device__ __forceinline__ bool better(Total a, Total b) { return a.v > b.v || (a.v == b.v && a.at < b.at); }

// Sorted runs of 2^LW numbers, one in each run's lanes, the best first, merged: the better
// of one and the other turned round, lane by lane, are the better half of both, rising
// and falling, which LW steps sort (Batcher's bitonic merge).  `turned`: that.
template <int D, class T>
__device__ __forceinline__ T sorted_steps(T x) {
  if constexpr (D > 0) {
    const T y = from_lane<D>(x);
    if (better(y, x) != ((threadIdx.x & D) != 0)) x = y;
    x = sorted_steps<D / 2>(x);
  }
  return x;
}
template <int LW, class T>
__device__ __forceinline__ T merged(T run, T turned) {
  return sorted_steps<(1 << LW) / 2>(better(turned, run) ? turned : run);
}
// All of a wave's runs as one, in every run's lanes.
template <int LW, int D, class T>
__device__ __forceinline__ T wave_run(T run) {
  if constexpr (D < 64) run = wave_run<LW, 2 * D>(merged<LW>(run, from_lane<(D | ((1 << LW) - 1))>(run)));
  return run;
}
template <int D>
__device__ __forceinline__ double wave_sum(double x) {
  if constexpr (D > 0) x = wave_sum<D / 2>(x + from_lane<D>(x));
  return x;
}

// A block for each group, whose waves take the beams by turns, or, where one's lists are many
// runs (kLong), several a part of them each: lists are merged by logit, the chunks' sums
// joined by the first.  Then one wave merges the beams' by value.
constexpr int kRankWaves = 16, kLong = 16;
template <int LW>
__global__ void __launch_bounds__(64 * kRankWaves) beam_rank_kernel(const BeamParams p, int chunks, int of_beam) {
  constexpr int W = 1 << LW, RUNS = 64 >> LW;
  __shared__ double add[64];  // score - log sum of each beam
  __shared__ uint64_t best[64 * W], parts[kRankWaves][W];
  const int64_t row0 = (int64_t)blockIdx.x * p.beams;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int k = lane & (W - 1), run = lane >> LW;
  const int part = wave % of_beam, teams = (int)(blockDim.x >> 6) / of_beam;
  for (int b0 = 0; b0 < p.beams; b0 += teams) {  // (the same number of rounds for all waves)
    const int b = b0 + wave / of_beam;
    const int64_t row = row0 + b;
    const float score = b < p.beams ? p.score[row] : -INFINITY;
    const bool over = b < p.beams && p.done && p.done[row], live = !is_none(score) && !over;
    const Stat* st = stats(p) + row * chunks;
    Stat first = {-INFINITY, 0.f};
    uint64_t acc = 0;
    if (live) {
      const uint64_t* cd = cands(p, chunks) + row * chunks * p.width;
      const int step = RUNS * of_beam;
      auto load = [&](int c) { return c < chunks && k < p.width ? cd[(int64_t)c * p.width + k] : 0; };
      if (part == 0 && lane < chunks) first = st[lane];
      for (int c0 = part * RUNS; c0 < chunks; c0 += 4 * step) {
        uint64_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = load(c0 + e * step + run);
        if (c0 == part * RUNS) acc = x[0];
        else acc = merged<LW>(acc, from_lane<W - 1>(x[0]));
#pragma unroll
        for (int e = 1; e < 4; ++e)
          if (c0 + e * step < chunks) acc = merged<LW>(acc, from_lane<W - 1>(x[e]));
      }
      acc = wave_run<LW, W>(acc);
    }
    for (int n = of_beam / 2; n > 0; n /= 2) {  // the parts in pairs
      if (lane < W) parts[wave][lane] = acc;
      lds_barrier();
      if (part < n) acc = merged<LW>(acc, parts[wave + n][W - 1 - k]);
      lds_barrier();
    }
    if (part > 0 || b >= p.beams) continue;
    if (live) {
      float top = first.top;
      for (int c = lane + 64; c < chunks; c += 64) top = fmaxf(top, st[c].top);
      top = over_lanes(top, 1, larger);
      double sum = first.sum == 0.f ? 0.0 : first.sum * exp((double)first.top - (double)top);
      for (int c = lane + 64; c < chunks; c += 64)
        if (st[c].sum != 0.f) sum += st[c].sum * exp((double)st[c].top - (double)top);
      sum = wave_sum<32>(sum);
      if (lane == 0) add[b] = (double)score - ((double)top + log(sum));
    } else {
      acc = k == 0 && !is_none(score) ? key_of(0.f, p.end) : 0;
      if (lane == 0) add[b] = score;
    }
    if (lane < W) best[b * W + lane] = acc;
  }
  lds_barrier();
  if (wave > 0) return;
  auto load = [&](int b) {
    const uint64_t x = b < p.beams ? best[b * W + k] : 0;
    return x ? Total{add[b] + (double)logit_of(x), (uint32_t)(b * W + k)} : Total{-INFINITY, ~0u};
  };
  Total all = load(run);
  for (int b0 = RUNS; b0 < p.beams; b0 += RUNS) all = merged<LW>(all, from_lane<W - 1>(load(b0 + run)));
  all = wave_run<LW, W>(all);
  if (lane >= p.width) return;
  const bool on = all.at != ~0u;
  const int64_t row = row0 + (on ? all.at >> LW : 0), o = (int64_t)blockIdx.x * p.width + lane;
  const int token = on ? token_of(best[all.at]) : -1;
  p.parent[o] = on ? (int)row : -1;
  p.token[o] = token;
  p.score_out[o] = on ? (float)all.v : -INFINITY;
  p.done_out[o] = on && (token == p.end || (p.done && p.done[row]));
}

template <int DT>
void launch_chunks(const BeamParams& p, hipStream_t s) {
  const int chunks = (int)chunks_of(p);
  const dim3 grid((unsigned)(p.groups * p.beams * chunks));
  const int each = each_of(p);
  if (each == 8) hipLaunchKernelGGL((beam_chunk_kernel<DT, 8>), grid, dim3(kThreads), 0, s, p, chunks, chunk_of(p));
  else if (each == 16) hipLaunchKernelGGL((beam_chunk_kernel<DT, 16>), grid, dim3(kThreads), 0, s, p, chunks, chunk_of(p));
  else hipLaunchKernelGGL((beam_chunk_kernel<DT, 32>), grid, dim3(kThreads), 0, s, p, chunks, chunk_of(p));
}
template <int LW>
void launch_rank(const BeamParams& p, hipStream_t s) {
  const int chunks = (int)chunks_of(p);
  int of_beam = 1;
  if (chunks > kLong * (64 >> LW))
    while (2 * of_beam * p.beams <= kRankWaves) of_beam *= 2;
  const int teams = p.beams < kRankWaves / of_beam ? p.beams : kRankWaves / of_beam;
  hipLaunchKernelGGL((beam_rank_kernel<LW>), dim3((unsigned)p.groups), dim3(64 * of_beam * teams), 0, s, p, chunks, of_beam);
}

}  // namespace

int64_t beam_select_blocks(int, const BeamParams& p) {
  const double n = (double)p.groups * p.beams * (double)chunks_of(p);
  return n > 9e18 ? INT64_MAX : (int64_t)n;
}
size_t beam_select_workspace(int, const BeamParams& p) {
  return (size_t)(p.groups * p.beams * chunks_of(p)) * (sizeof(Stat) + p.width * sizeof(uint64_t));
}
hipError_t launch_beam_select(int dtype, const BeamParams& p, hipStream_t s) {
  if (dtype == QA_F32) launch_chunks<QA_F32>(p, s);
  else if (dtype == QA_BF16) launch_chunks<QA_BF16>(p, s);
  else launch_chunks<QA_F16>(p, s);
  if (p.width <= 4) launch_rank<2>(p, s);
  else if (p.width <= 8) launch_rank<3>(p, s);
  else if (p.width <= 16) launch_rank<4>(p, s);
  else if (p.width <= 32) launch_rank<5>(p, s);
  else launch_rank<6>(p, s);
  return hipGetLastError();
}

}  // namespace qa

// qa_beam.hip -- the step of a beam search: for each group the `width` best of
// score[b] + x[b][t] - log sum_t' exp x[b][t'] over its beams b and the vocabulary t.
//
// Within a row the order is that of the logits, so a first launch needs each logit
// once: a block takes a chunk of a row, and leaves its maximum, its sum of exponentials and
// its `width` largest logits in the workspace.  A second one, a block for each group,
// joins the sums in f64 and ranks the chunks' candidates, in f64 too: an f32 sum of
// a score near -50 and a log-probability has steps of 4e-6, and candidates that differ
// by less would change places.  Equal ones go by (beam, token), so every comparison is
// of (value, index) pairs of which no two are alike: results do not depend on timing.
#include "qa_internal.h"

namespace qa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kThreads = 256, kChunk = 8192, kEach = kChunk / kThreads;

// The workspace: each chunk's maximum and sum, then each chunk's candidates (logit,
// token), best first, token -1 behind the last.
struct Stat {
  float top, sum;
};
struct Cand {
  float x;
  int token;
};
__host__ __device__ __forceinline__ int64_t chunks_of(const BeamParams& p) { return (p.vocab + kChunk - 1) / kChunk; }
__device__ __forceinline__ Stat* stats(const BeamParams& p) { return (Stat*)p.ws; }
__device__ __forceinline__ Cand* cands(const BeamParams& p) { return (Cand*)(stats(p) + p.groups * p.beams * chunks_of(p)); }

// A beam that has no continuations of its own: none, or ended.
__device__ __forceinline__ bool is_none(float score) { return !(score > -INFINITY && score < INFINITY); }

template <class V, class I>
__device__ __forceinline__ bool before(V v, I i, V w, I j) {
  return v > w || (v == w && i < j);
}
template <class V, class I>
__device__ __forceinline__ void wave_best(V& v, I& i) {
#pragma unroll
  for (int e = 32; e > 0; e >>= 1) {
    const V w = __shfl_xor(v, e, 64);
    const I j = __shfl_xor(i, e, 64);
    if (before(w, j, v, i)) {
      v = w;
      i = j;
    }
  }
}
template <class V, class I>
__device__ __forceinline__ void block_best(V& v, I& i, V* vs, I* is) {
  wave_best(v, i);
  if ((threadIdx.x & 63) == 0) {
    vs[threadIdx.x >> 6] = v;
    is[threadIdx.x >> 6] = i;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w)
    if (before(vs[w], is[w], v, i)) {
      v = vs[w];
      i = is[w];
    }
  __syncthreads();
}

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

template <int DT>
__global__ void __launch_bounds__(kThreads) beam_chunk_kernel(const BeamParams p) {
  constexpr int N = kRun<DT>, RUNS = kEach / N;
  __shared__ float vs[kThreads / 64];
  __shared__ int is[kThreads / 64];
  const int64_t chunks = chunks_of(p), row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
  if (is_none(p.score[row]) || (p.done && p.done[row])) return;
  const int t = threadIdx.x;
  const int64_t t0 = chunk * kChunk;
  const char* src = (const char*)p.logits + row * p.ldl * (DT == QA_F32 ? 4 : 2);
  float x[kEach];
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    const int64_t at = t0 + (r * kThreads + t) * N;
    if (at + N <= p.vocab) {
      unpack<DT>(*reinterpret_cast<const u32x4*>(src + at * (DT == QA_F32 ? 4 : 2)), x + r * N);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[r * N + e] = at + e < p.vocab ? logit<DT>(src, at + e) : -INFINITY;
    }
  }
  auto token = [&](int j) { return (int)(t0 + (j / N * kThreads + t) * N + j % N); };
#pragma unroll
  for (int j = 0; j < kEach; ++j) x[j] = x[j] < INFINITY ? x[j] : -INFINITY;  // NaN too
  // its best that comes behind (v, i)
  auto next = [&](float v, int i, float* bv, int* bi) {
    *bv = -INFINITY;
    *bi = INT32_MAX;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (before(v, i, x[j], token(j)) && x[j] > *bv) {
        *bv = x[j];
        *bi = token(j);
      }
  };
  float mine;
  int at;
  next(INFINITY, -1, &mine, &at);
  float v = mine;
  int i = at;
  block_best(v, i, vs, is);
  const float top = v;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < kEach; ++j) sum += top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x[j] - top) * kLog2e);
#pragma unroll
  for (int e = 32; e > 0; e >>= 1) sum += __shfl_xor(sum, e, 64);
  if ((t & 63) == 0) vs[t >> 6] = sum;
  __syncthreads();
  if (t == 0) stats(p)[blockIdx.x] = {top, (vs[0] + vs[1]) + (vs[2] + vs[3])};
  __syncthreads();
  Cand* out = cands(p) + (int64_t)blockIdx.x * p.width;
  for (int k = 0;; ) {
    if (t == 0) out[k] = {v, v == -INFINITY ? -1 : i};
    if (++k == p.width) break;
    if (at == i) next(v, i, &mine, &at);
    v = mine;
    i = at;
    block_best(v, i, vs, is);
  }
}

template <int DT>
__global__ void __launch_bounds__(kThreads) beam_rank_kernel(const BeamParams p) {
  __shared__ double vs[kThreads / 64], add[64];  // score - log sum of each beam
  __shared__ int64_t is[kThreads / 64];
  const int64_t chunks = chunks_of(p), g = blockIdx.x, row0 = g * p.beams;
  const int t = threadIdx.x, lane = t & 63;
  for (int b = t >> 6; b < p.beams; b += kThreads / 64) {
    const float score = p.score[row0 + b];
    if (is_none(score) || (p.done && p.done[row0 + b])) continue;
    const Stat* st = stats(p) + (row0 + b) * chunks;
    float top = -INFINITY;
    for (int64_t c = lane; c < chunks; c += 64) top = fmaxf(top, st[c].top);
#pragma unroll
    for (int e = 32; e > 0; e >>= 1) top = fmaxf(top, __shfl_xor(top, e, 64));
    double sum = 0.0;
    for (int64_t c = lane; c < chunks; c += 64)
      if (st[c].top > -INFINITY) sum += (double)st[c].sum * exp((double)st[c].top - (double)top);
#pragma unroll
    for (int e = 32; e > 0; e >>= 1) sum += __shfl_xor(sum, e, 64);
    if (lane == 0) add[b] = (double)score - ((double)top + log(sum));
  }
  __syncthreads();
  const int64_t each = chunks * p.width, n = p.beams * each;
  // candidate number c: its value and its (beam, token) as one index; false if it is none
  auto candidate = [&](int64_t c, double* v, int64_t* i) {
    const int64_t b = c / each;
    const float score = p.score[row0 + b];
    if (is_none(score)) return false;
    if (p.done && p.done[row0 + b]) {
      *v = score;
      *i = b * p.vocab + p.end;
      return c == b * each;
    }
    const Cand k = cands(p)[row0 * each + c];
    *v = add[b] + (double)k.x;
    *i = b * p.vocab + k.token;
    return k.token >= 0;
  };
  auto next = [&](double v, int64_t i, double* bv, int64_t* bi) {
    *bv = -INFINITY;
    *bi = INT64_MAX;
    for (int64_t c = t; c < n; c += kThreads) {
      double w;
      int64_t j;
      if (candidate(c, &w, &j) && before(v, i, w, j) && before(w, j, *bv, *bi)) {
        *bv = w;
        *bi = j;
      }
    }
  };
  double mine;
  int64_t at;
  next(INFINITY, -1, &mine, &at);
  for (int k = 0; k < p.width; ++k) {
    double v = mine;
    int64_t i = at;
    block_best(v, i, vs, is);
    if (t == 0) {
      const bool on = i != INT64_MAX;
      const int64_t b = on ? i / p.vocab : 0, o = g * p.width + k;
      p.parent[o] = on ? (int)(row0 + b) : -1;
      p.token[o] = on ? (int)(i - b * p.vocab) : -1;
      p.score_out[o] = on ? (float)v : -INFINITY;
      p.done_out[o] = on && ((p.done && p.done[row0 + b]) || i - b * p.vocab == p.end);
    }
    if (at == i) next(v, i, &mine, &at);
  }
}

template <int DT>
hipError_t launch(const BeamParams& p, hipStream_t s) {
  hipLaunchKernelGGL((beam_chunk_kernel<DT>), dim3((unsigned)(p.groups * p.beams * chunks_of(p))), dim3(kThreads), 0, s, p);
  hipLaunchKernelGGL((beam_rank_kernel<DT>), dim3((unsigned)p.groups), dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

}  // namespace

int64_t beam_select_blocks(int, const BeamParams& p) {
  const double n = (double)p.groups * p.beams * (double)chunks_of(p);
  return n > 9e18 ? INT64_MAX : (int64_t)n;
}
size_t beam_select_workspace(int, const BeamParams& p) {
  return (size_t)(p.groups * p.beams * chunks_of(p)) * (sizeof(Stat) + p.width * sizeof(Cand));
}
hipError_t launch_beam_select(int dtype, const BeamParams& p, hipStream_t s) {
  return dtype == QA_F32 ? launch<QA_F32>(p, s) : dtype == QA_BF16 ? launch<QA_BF16>(p, s) : launch<QA_F16>(p, s);
}

}  // namespace qa

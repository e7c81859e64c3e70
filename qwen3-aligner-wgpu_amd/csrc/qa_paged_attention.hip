// qa_paged_attention.hip -- causal attention of a packed batch over the paged
// cache (16-bit or e4m3 pages).
//
// Row i of a sequence with n rows and len keys sees keys 0 .. len - n + i:
// out = sum_t p_t v_t / sum_t p_t, p_t = exp(q.k_t / sqrt(hd) - max).  One wave to a
// (row, q head), 64 keys at a time: lane = key for the scores, lane = d for P.V.
#include "qa_internal.h"

namespace qa {
namespace {

template <int DT>
__device__ __forceinline__ float widen16(uint32_t h) {
  if constexpr (DT == QA_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
  return __uint_as_float(h << 16);
}
template <int DT>
__device__ __forceinline__ uint16_t narrow16(float v) {
  if constexpr (DT == QA_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <int DT, bool F8>
__device__ __forceinline__ float element(const void* x, int64_t i) {
  if constexpr (F8) return __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t*>(x)[i], 0);
  return widen16<DT>(static_cast<const uint16_t*>(x)[i]);
}

template <int DT, bool F8, int HD>
__global__ void __launch_bounds__(64) paged_attention_kernel(const PagedAttnParams p) {
  __shared__ float qs[HD], ps[64];
  const PagedParams& kv = p.kv;
  const int lane = threadIdx.x, head = (int)(blockIdx.x % p.nqh), h = head / p.rep;
  const int64_t b = blockIdx.x / p.nqh;
  const int s = (int)(b / kv.max_rows), i = (int)(b % kv.max_rows);
  const SeqSpan sq = seq_span(kv, s);
  if (i >= sq.n) return;
  const int64_t t = sq.row0 + i;
  for (int d = lane; d < HD; d += 64) qs[d] = widen16<DT>(p.q[t * p.ldq + (int64_t)head * HD + d]);
  __syncthreads();
  const int keys = sq.pos0 + i + 1;  // not above len; may be zero or less
  float o[HD / 64] = {}, m = -INFINITY, l = 0.f;
  for (int k0 = 0; k0 < keys; k0 += 64) {
    const int id = k0 + lane < keys ? page_at(kv, s, k0 + lane) : -1;
    const int slot = (k0 + lane) & ((1 << kv.lp) - 1);
    float x = -INFINITY;
    if (id >= 0) {
      const int64_t at = page_base(kv, id, h, HD) + (int64_t)slot * HD;
      float a = 0.f;
      for (int d = 0; d < HD; ++d) a += qs[d] * element<DT, F8>(kv.k, at + d);
      if constexpr (F8) a *= kv.k_scale[(int64_t)id * kv.nkvh + h];
      x = a * p.scale;
    }
    float top = x;
    for (int e = 32; e > 0; e >>= 1) top = fmaxf(top, __shfl_xor(top, e, 64));
    const float m2 = fmaxf(m, top);
    if (m2 == -INFINITY) continue;
    const float al = expf(m - m2), w = expf(x - m2);
    m = m2;
    l = l * al + w;
    __syncthreads();
    ps[lane] = w;
    __syncthreads();
    for (int j = 0; j < HD / 64; ++j) o[j] *= al;
    for (int e = 0; e < 64 && k0 + e < keys; ++e) {
      const int pid = __shfl(id, e, 64);
      if (pid < 0) continue;
      const float ww = F8 ? ps[e] * kv.v_scale[(int64_t)pid * kv.nkvh + h] : ps[e];
      for (int j = 0; j < HD / 64; ++j)
        o[j] += ww * element<DT, F8>(kv.v, page_base(kv, pid, h, HD) + ((int64_t)(lane + 64 * j) << kv.lp) +
                                               ((k0 + e) & ((1 << kv.lp) - 1)));
    }
  }
  for (int e = 32; e > 0; e >>= 1) l += __shfl_xor(l, e, 64);
  const float inv = m == -INFINITY ? 0.f : 1.0f / l;  // no key: zeros
  for (int j = 0; j < HD / 64; ++j) p.out[t * p.ldo + (int64_t)head * HD + lane + 64 * j] = narrow16<DT>(o[j] * inv);
}

template <int DT, bool F8, int HD>
hipError_t launch_one(const PagedAttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.kv.seqs * p.kv.max_rows * p.nqh));
  hipLaunchKernelGGL((paged_attention_kernel<DT, F8, HD>), grid, dim3(64), 0, s, p);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(bool e4m3, int hd, const PagedAttnParams& p, hipStream_t s) {
  if (hd == 64) return e4m3 ? launch_one<DT, true, 64>(p, s) : launch_one<DT, false, 64>(p, s);
  return e4m3 ? launch_one<DT, true, 128>(p, s) : launch_one<DT, false, 128>(p, s);
}

}  // namespace

size_t paged_attention_workspace(int, const PagedAttnParams&) { return 0; }

hipError_t launch_attention_paged(int dtype, bool e4m3, int hd, const PagedAttnParams& p, hipStream_t s) {
  return dtype == QA_BF16 ? launch_dt<QA_BF16>(e4m3, hd, p, s) : launch_dt<QA_F16>(e4m3, hd, p, s);
}

}  // namespace qa

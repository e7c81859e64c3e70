// qa_paged_append.hip -- a step's new rows into the paged cache: q / k head
// RMSNorm and rotation as in qk_norm_rope_kernel, q to its rows, K and V to the
// slots of their sequences' pages, in the 16-bit format or in e4m3.
//
// One grid.  The first blocks take the q heads, HD / 16 lanes to a head, each
// lane with the 8-element chunk c and its rotation partners, chunk c + HD / 16.
// Each other block takes one (sequence, page, kv head): the rows of this call
// that fall into that page, K and V.  A page is one block's because an e4m3 page
// has one scale: its block finds the largest new value, raises the scale if it
// must, rounds what the page held again, and stores the rows, with no other
// block to wait for.  The V page is [hd][page], so V goes through an LDS tile.
//
// e4m3 scales are powers of two, the least 2^e with amax <= 448 * 2^e: dividing by
// one is exact, so a value is rounded once however often its page's scale
// grows, but for what falls below e4m3's normal range (2^-6 of the scale).
#include "qa_internal.h"

namespace qa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ f32x2 widen2(uint32_t h) {
  if constexpr (DT == QA_F16) return __builtin_convertvector(__builtin_bit_cast(f16x2, h), f32x2);
  return (f32x2){__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)};
}
template <int DT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (DT == QA_F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// Values within +-448 (infinities come down to it, NaN stays) as four e4m3.
__device__ __forceinline__ float hold448(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(hold448(a), hold448(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hold448(c), hold448(d), w, true);
}

// The least power of two p with amax <= 448 p (448 = 1.75 * 2^8), held to
// [2^-110, 2^120] so that p and 1 / p are normal.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
  return __uint_as_float((uint32_t)(min(max(e, -110), 120) + 127) << 23);
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // NaN too
}

// The normed and rotated chunks c and c + HD / 16 of a q or k head, for the
// HD / 16 lanes that share it (all of them call, `on` or not).
template <int DT, int HD>
__device__ __forceinline__ void norm_rope(const uint16_t* raw, const float* nw, const float* cs, const float* sn,
                                          int c, float eps, bool on, float* xa, float* xb) {
  constexpr int L = HD / 16, half = HD / 2;
  u32x4 va = {0, 0, 0, 0}, vb = {0, 0, 0, 0};
  f32x4 t[12] = {};
  if (on) {
    va = *reinterpret_cast<const u32x4*>(raw + 8 * c);
    vb = *reinterpret_cast<const u32x4*>(raw + half + 8 * c);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      t[h] = *reinterpret_cast<const f32x4*>(nw + 8 * c + 4 * h);
      t[2 + h] = *reinterpret_cast<const f32x4*>(nw + half + 8 * c + 4 * h);
      t[4 + h] = *reinterpret_cast<const f32x4*>(cs + 8 * c + 4 * h);
      t[6 + h] = *reinterpret_cast<const f32x4*>(cs + half + 8 * c + 4 * h);
      t[8 + h] = *reinterpret_cast<const f32x4*>(sn + 8 * c + 4 * h);
      t[10 + h] = *reinterpret_cast<const f32x4*>(sn + half + 8 * c + 4 * h);
    }
  }
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x2 a = widen2<DT>(va[e]), b = widen2<DT>(vb[e]);
    xa[2 * e] = a[0];
    xa[2 * e + 1] = a[1];
    xb[2 * e] = b[0];
    xb[2 * e + 1] = b[1];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    s += xa[e] * xa[e];
    s += xb[e] * xb[e];
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o, 64);
  const float inv = 1.0f / sqrtf(s / (float)HD + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int h = e >> 2, i = e & 3;
    const float a = xa[e] * inv * t[h][i], b = xb[e] * inv * t[2 + h][i];
    xa[e] = a * t[4 + h][i] - b * t[8 + h][i];
    xb[e] = b * t[6 + h][i] + a * t[10 + h][i];
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack8(const float* x) {
  return u32x4{narrow2<DT>(x[0], x[1]), narrow2<DT>(x[2], x[3]), narrow2<DT>(x[4], x[5]), narrow2<DT>(x[6], x[7])};
}

template <int DT, int HD>
__device__ __forceinline__ void q_part(const AppendParams& p, int64_t bx) {
  constexpr int L = HD / 16, hpw = 64 / L;
  const int lane = threadIdx.x & 63;
  const int groups = (p.nqh + hpw - 1) / hpw;
  const int64_t item = bx * 4 + (threadIdx.x >> 6);
  const int64_t t = item / groups;
  // rows of no sequence keep what they hold
  const int64_t t0 = p.kv.row_start[0], t1 = p.kv.row_start[p.kv.seqs];
  if (t >= p.kv.tokens || t < t0 || t >= t1) return;
  const int head = (int)(item % groups) * hpw + lane / L, c = lane % L;
  const bool on = head < p.nqh;
  float xa[8], xb[8];
  norm_rope<DT, HD>(p.qkv + t * p.ldqkv + (int64_t)(on ? head : 0) * HD, p.qn, p.cos + t * HD, p.sin + t * HD, c, p.eps, on,
                    xa, xb);
  if (!on) return;
  uint16_t* dst = p.q_out + t * p.ldq + (int64_t)head * HD + 8 * c;
  *reinterpret_cast<u32x4*>(dst) = pack8<DT>(xa);
  *reinterpret_cast<u32x4*>(dst + HD / 2) = pack8<DT>(xb);
}

// A page's 8-bit values rounded again to a scale 1 / ratio times the old one.
__device__ __forceinline__ void rescale(uint8_t* page, int bytes, float ratio) {
  for (int i = threadIdx.x * 16; i < bytes; i += 256 * 16) {
    u32x4 w = *reinterpret_cast<const u32x4*>(page + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[e], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[e], true);
      w[e] = e4m3x4(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
    }
    *reinterpret_cast<u32x4*>(page + i) = w;
  }
}

template <int DT, bool F8, int HD>
__device__ __forceinline__ void kv_part(const AppendParams& p, int64_t b, int slots) {
  constexpr int L = HD / 16;          // lanes to a row
  constexpr int RP = 256 / L;         // rows in a pass
  constexpr int NP = (64 + RP - 1) / RP;  // passes over the largest page
  __shared__ uint16_t tile[64][HD + 2];
  __shared__ float top[2][4];
  const PagedParams& kv = p.kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = (int)(b % kv.nkvh);
  const int64_t sp = b / kv.nkvh;
  const int s = (int)(sp / slots);
  const SeqSpan sq = seq_span(kv, s);
  const int page = 1 << kv.lp;
  // this block's page of the sequence, and the positions of it that are new
  const int first = sq.pos0 > 0 ? sq.pos0 : 0;
  const int64_t pi = (int64_t)(first >> kv.lp) + sp % slots;
  const int64_t lo64 = pi << kv.lp, end = (int64_t)sq.pos0 + sq.n;
  const int64_t to = end < lo64 + page ? end : lo64 + page;
  const int64_t from = lo64 > first ? lo64 : first;
  if (from >= to) return;
  const int id = page_at(kv, s, (int)from);
  if (id < 0) return;
  const int slot0 = (int)(from - lo64), nr = (int)(to - from);
  const int64_t t0 = sq.row0 + (from - sq.pos0);
  const uint16_t* src = p.qkv + t0 * p.ldqkv + (int64_t)p.nqh * HD + (int64_t)h * HD;
  const int64_t base = page_base(kv, id, h, HD);

  float xa[NP][8], xb[NP][8];
  float ka = 0.f, va = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RP + tid / L, c = tid % L;
    const bool on = r < nr;
    const uint16_t* row = src + (int64_t)(on ? r : 0) * p.ldqkv;
    const float* cs = p.cos + (t0 + (on ? r : 0)) * HD;
    const float* sn = p.sin + (t0 + (on ? r : 0)) * HD;
    if (on) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + (int64_t)kv.nkvh * HD + 16 * c + 8 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          *reinterpret_cast<uint32_t*>(&tile[r][16 * c + 8 * u + 2 * e]) = w[e];
          if constexpr (F8) {
            const f32x2 f = widen2<DT>(w[e]);
            va = fmaxf(va, fmaxf(finite_abs(f[0]), finite_abs(f[1])));
          }
        }
      }
    }
    norm_rope<DT, HD>(row, p.kn, cs, sn, c, p.eps, on, xa[i], xb[i]);
    if constexpr (F8) {
      if (on) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ka = fmaxf(ka, fmaxf(finite_abs(xa[i][e]), finite_abs(xb[i][e])));
      }
    }
  }
  float kinv = 1.f, vinv = 1.f;
  if constexpr (F8) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      ka = fmaxf(ka, __shfl_xor(ka, o, 64));
      va = fmaxf(va, __shfl_xor(va, o, 64));
    }
    if (lane == 0) {
      top[0][wave] = ka;
      top[1][wave] = va;
    }
    float* sc[2] = {kv.k_scale + (int64_t)id * kv.nkvh + h, kv.v_scale + (int64_t)id * kv.nkvh + h};
    float old[2] = {0.f, 0.f};
    if (slot0 > 0) {  // a scale that is no positive number stands for a page of nothing
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        old[i] = *sc[i];
        old[i] = old[i] > 0.f && old[i] < INFINITY ? old[i] : 0.f;
      }
    }
    __syncthreads();  // every thread has the old scales
    float now[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      now[i] = fmaxf(old[i], scale_for(fmaxf(fmaxf(top[i][0], top[i][1]), fmaxf(top[i][2], top[i][3]))));
    if (tid < 2) *sc[tid] = tid ? now[1] : now[0];
    if (slot0 > 0) {
      if (now[0] != old[0]) rescale((uint8_t*)kv.k + base, page * HD, old[0] / now[0]);
      if (now[1] != old[1]) rescale((uint8_t*)kv.v + base, page * HD, old[1] / now[1]);
    }
    kinv = 1.0f / now[0];
    vinv = 1.0f / now[1];
  }
  __syncthreads();  // the V tile; the page as it was is rounded again before the new rows go in

#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RP + tid / L, c = tid % L;
    if (r >= nr) continue;
    const int64_t at = base + (int64_t)(slot0 + r) * HD + 8 * c;
    if constexpr (F8) {
      uint8_t* dst = (uint8_t*)kv.k + at;
      uint32_t wa[2], wb[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        wa[e] = e4m3x4(xa[i][4 * e] * kinv, xa[i][4 * e + 1] * kinv, xa[i][4 * e + 2] * kinv, xa[i][4 * e + 3] * kinv);
        wb[e] = e4m3x4(xb[i][4 * e] * kinv, xb[i][4 * e + 1] * kinv, xb[i][4 * e + 2] * kinv, xb[i][4 * e + 3] * kinv);
      }
      *reinterpret_cast<uint64_t*>(dst) = wa[0] | (uint64_t)wa[1] << 32;
      *reinterpret_cast<uint64_t*>(dst + HD / 2) = wb[0] | (uint64_t)wb[1] << 32;
    } else {
      uint16_t* dst = (uint16_t*)kv.k + at;
      *reinterpret_cast<u32x4*>(dst) = pack8<DT>(xa[i]);
      *reinterpret_cast<u32x4*>(dst + HD / 2) = pack8<DT>(xb[i]);
    }
  }
  // V^T: CH slots of one d to a thread, 16 bytes where all of them are new
  constexpr int CH = F8 ? 16 : 8;
  const int nch = page / CH;  // chunks of a V row
  const int c0 = slot0 / CH, c1 = (slot0 + nr + CH - 1) / CH;
  const int per = c1 - c0;
  for (int u = tid; u < HD * per; u += 256) {
    const int d = u / per, ch = c0 + u % per, f = ch * CH - slot0;  // f: the chunk's first row of the tile
    const int64_t at = base + ((int64_t)d * nch + ch) * CH;
    if constexpr (F8) {
      uint8_t* dst = (uint8_t*)kv.v + at;
      auto val = [&](int r) { return widen2<DT>(tile[r][d])[0] * vinv; };
      if (f >= 0 && f + CH <= nr) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = e4m3x4(val(f + 4 * e), val(f + 4 * e + 1), val(f + 4 * e + 2), val(f + 4 * e + 3));
        *reinterpret_cast<u32x4*>(dst) = w;
      } else {
        for (int e = max(0, -f); e < CH && f + e < nr; ++e) dst[e] = (uint8_t)e4m3x4(val(f + e), 0.f, 0.f, 0.f);
      }
    } else {
      uint16_t* dst = (uint16_t*)kv.v + at;
      if (f >= 0 && f + CH <= nr) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (uint32_t)tile[f + 2 * e][d] | (uint32_t)tile[f + 2 * e + 1][d] << 16;
        *reinterpret_cast<u32x4*>(dst) = w;
      } else {
        for (int e = max(0, -f); e < CH && f + e < nr; ++e) dst[e] = tile[f + e][d];
      }
    }
  }
}

template <int DT, bool F8, int HD>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p, int64_t qblocks, int slots) {
  if ((int64_t)blockIdx.x < qblocks) q_part<DT, HD>(p, blockIdx.x);
  else kv_part<DT, F8, HD>(p, blockIdx.x - qblocks, slots);
}

template <int DT, bool F8, int HD>
hipError_t launch_one(const AppendParams& p, hipStream_t s) {
  const int64_t hpw = 1024 / HD, items = p.kv.tokens * ((p.nqh + hpw - 1) / hpw), qb = (items + 3) / 4;
  const int64_t slots = pages_touched(p.kv.max_rows, p.kv.lp);
  hipLaunchKernelGGL((kv_append_kernel<DT, F8, HD>), dim3((unsigned)(qb + slots * p.kv.seqs * p.kv.nkvh)), dim3(256), 0, s, p,
                     qb, (int)slots);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(bool e4m3, int hd, const AppendParams& p, hipStream_t s) {
  if (hd == 64) return e4m3 ? launch_one<DT, true, 64>(p, s) : launch_one<DT, false, 64>(p, s);
  return e4m3 ? launch_one<DT, true, 128>(p, s) : launch_one<DT, false, 128>(p, s);
}

}  // namespace

hipError_t launch_kv_append(int dtype, bool e4m3, int hd, const AppendParams& p, hipStream_t s) {
  return dtype == QA_BF16 ? launch_dt<QA_BF16>(e4m3, hd, p, s) : launch_dt<QA_F16>(e4m3, hd, p, s);
}

}  // namespace qa

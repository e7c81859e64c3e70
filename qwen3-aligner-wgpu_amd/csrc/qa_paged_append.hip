// qa_paged_append.hip -- a step's new rows into the paged cache: q / k head
// RMSNorm and rotation as in qk_norm_rope_kernel, q to its rows, K and V to the
// slots of their sequences' pages, in the 16-bit format or in e4m3.
//
// One grid.  Its first blocks take one (sequence, page, kv head) each: the rows of
// this call that fall into that page, K and V.  A page is one block's because an
// e4m3 page has one scale: its block finds the largest new value, raises the scale
// if it must, rounds what the page held again, and stores the rows, with no other
// block to wait for.  The V page is [hd][page], so V goes through an LDS tile.
// The other blocks take the q heads, a wave to a row, HD / 16 lanes to a head, each
// lane with the 8-element chunk c and its rotation partners, chunk c + HD / 16; the
// row's cosines and sines and the norm's weights stay in registers from head to
// head.  (The pages' blocks are the longer ones, with two barriers and V's turn:
// behind the rows' instead of before them, 18.4 us for 15.7 at 4334 rows.)
//
// Bound by the bytes: 4334 rows of 16 q and 8 kv heads of 128 into empty e4m3 pages, 67
// MB, 15.7 us (4.2 TB/s), into 16-bit pages, 75 MB, 15.0; a step's few rows by the
// launch and a chain of loads, row_start, the table, the row: 32 single rows 4.2 us.
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

// What a lane needs for its chunk c of every head: the norm's weights of both chunks,
// and the row's cosines and sines (whose second half repeats the first).
struct Turn {
  float wa[8], wb[8], co[8], si[8];
};
__device__ __forceinline__ void load8(float* to, const float* from) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(from + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[4 * h + e] = v[e];
  }
}
template <int HD>
__device__ __forceinline__ Turn load_turn(const float* nw, const float* cs, const float* sn, int c) {
  Turn t;
  load8(t.wa, nw + 8 * c);
  load8(t.wb, nw + HD / 2 + 8 * c);
  load8(t.co, cs + 8 * c);
  load8(t.si, sn + 8 * c);
  return t;
}
// The sum over the 4 or 8 lanes that share a head, by moves within a row of lanes:
// each lane's neighbour, the neighbouring pair, and (8) the mirrored lane.
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int HD, class T>
__device__ __forceinline__ T head_sum(T s) {
  s += moved<0xB1>(s);                              // quad_perm [1, 0, 3, 2]
  s += moved<0x4E>(s);                              // quad_perm [2, 3, 0, 1]
  if constexpr (HD == 128) s += moved<0x141>(s);    // row_half_mirror
  return s;
}
// The normed and rotated chunks of a q or k head from its raw ones, for the HD / 16
// lanes that share it (all of them call).
template <int DT, int HD>
__device__ __forceinline__ void norm_rope(u32x4 va, u32x4 vb, const Turn& t, float eps, float* xa, float* xb) {
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
  const float inv = 1.0f / sqrtf(head_sum<HD>(s) / (float)HD + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = xa[e] * inv * t.wa[e], b = xb[e] * inv * t.wb[e];
    xa[e] = a * t.co[e] - b * t.si[e];
    xb[e] = b * t.co[e] + a * t.si[e];
  }
}

// x to f32 so that a further rounding, to fewer bits, gives what rounding x itself
// to those would: towards zero, with the last bit set where anything was lost.
__device__ __forceinline__ float to_odd(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)u, lost = (lo & 0x1fffffffu) + 0x1fffffffu;  // bit 29: some of the 29 bits is set
  return (float)__builtin_bit_cast(double, (u & ~0xffffffffull) | ((lo | lost) & 0xe0000000u));
}
// The same for a k head that goes to e4m3, whose steps are 2^20 times f32's: in f32 a
// few values of a long prompt end up on the other side of a step's middle than
// their definition.  In f64 none does (4334 rows 15.5 -> 15.7 us).
template <int DT, int HD>
__device__ __forceinline__ void norm_rope_exact(u32x4 va, u32x4 vb, const Turn& t, float eps, float* xa, float* xb) {
  float fa[8], fb[8];
  double q[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x2 a = widen2<DT>(va[e]), b = widen2<DT>(vb[e]);
    fa[2 * e] = a[0];
    fa[2 * e + 1] = a[1];
    fb[2 * e] = b[0];
    fb[2 * e + 1] = b[1];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e & 3] = fma((double)fa[e], (double)fa[e], fma((double)fb[e], (double)fb[e], q[e & 3]));
  const double v = head_sum<HD>((q[0] + q[1]) + (q[2] + q[3])) * (1.0 / HD) + (double)eps, y = __builtin_amdgcn_rsq(v);  // y to 2^-23: one step of Newton's
  const double inv = v < (double)INFINITY ? y * fma(-0.5 * v * y, y, 1.5) : v == v ? 0.0 : v;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double a = (double)fa[e] * (double)t.wa[e] * inv, b = (double)fb[e] * (double)t.wb[e] * inv;
    xa[e] = to_odd(fma(a, (double)t.co[e], -b * (double)t.si[e]));
    xb[e] = to_odd(fma(b, (double)t.co[e], a * (double)t.si[e]));
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack8(const float* x) {
  return u32x4{narrow2<DT>(x[0], x[1]), narrow2<DT>(x[2], x[3]), narrow2<DT>(x[4], x[5]), narrow2<DT>(x[6], x[7])};
}

// Row t's place in its sequence, for the whole wave: row_start rises, and each step looks
// at 64 of what is left of it, so that 64 sequences take one load, which does not wait
// for the others of q_part.  row_start[0] <= t < row_start[seqs].
__device__ __forceinline__ int64_t row_in_sequence(const PagedParams& kv, int64_t t) {
  const int lane = threadIdx.x & 63;
  for (int lo = 0, n = kv.seqs;;) {  // the last start <= t is one of lo .. lo + n - 1
    const int step = (n - 1) / 64 + 1;
    const int start = lane * (int64_t)step < n ? kv.row_start[lo + lane * step] : 0x7fffffff;
    const uint64_t upto = __builtin_amdgcn_ballot_w64(start <= t);
    const int at = upto ? 63 - __builtin_clzll(upto) : 0;
    if (step == 1) return t - max(__builtin_amdgcn_readlane(start, at), 0);
    lo += at * step;
    n = min(step, n - at * step);
  }
}

template <int DT, int HD>
__device__ __forceinline__ void q_part(const AppendParams& p, int64_t bx) {
  constexpr int L = HD / 16, hpw = 64 / L;  // lanes to a head, heads at once
  const int lane = threadIdx.x & 63, c = lane % L, sub = lane / L;
  const int64_t t = bx * 4 + (threadIdx.x >> 6);
  // rows of no sequence keep what they hold
  const int64_t t0 = p.kv.row_start[0], t1 = p.kv.row_start[p.kv.seqs];
  if (t >= p.kv.tokens || t < t0 || t >= t1) return;
  const Turn turn = load_turn<HD>(p.qn, p.cos + t * HD, p.sin + t * HD, c);
  const uint16_t* src = p.qkv + t * p.ldqkv + 8 * c;
  uint16_t* dst = p.q_out + t * p.ldq + 8 * c;
  auto load = [&](int head, u32x4* a, u32x4* b) {  // past the last head: the last again
    const uint16_t* raw = src + (int64_t)min(head, p.nqh - 1) * HD;
    *a = *reinterpret_cast<const u32x4*>(raw);
    *b = *reinterpret_cast<const u32x4*>(raw + HD / 2);
  };
  u32x4 va, vb, na, nb;
  load(sub, &va, &vb);
  // ... and so do those past max_rows, which only a batch of more rows can have; the first
  // loads are under way by now (8 prompts of 771 rows 16.2 us, 16.1 without this, 16.6 with it before them)
  if (p.kv.max_rows < p.kv.tokens && row_in_sequence(p.kv, t) >= p.kv.max_rows) return;
  for (int h0 = 0; h0 < p.nqh; h0 += hpw) {
    load(h0 + hpw + sub, &na, &nb);  // the next heads, while these are at work
    float xa[8], xb[8];
    norm_rope<DT, HD>(va, vb, turn, p.eps, xa, xb);
    if (h0 + sub < p.nqh) {
      *reinterpret_cast<u32x4*>(dst + (int64_t)(h0 + sub) * HD) = pack8<DT>(xa);
      *reinterpret_cast<u32x4*>(dst + (int64_t)(h0 + sub) * HD + HD / 2) = pack8<DT>(xb);
    }
    va = na;
    vb = nb;
  }
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

template <int DT, bool F8, int HD, int NP>
__device__ __forceinline__ void kv_part(const AppendParams& p, int64_t b, int slots) {
  constexpr int L = HD / 16;   // lanes to a row
  constexpr int RP = 256 / L;  // rows in a pass; NP: passes over a page
  __shared__ uint16_t tile[NP * RP][HD + 2];
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
    if (i * RP >= nr) break;
    const int r = i * RP + tid / L, c = tid % L;
    const bool on = r < nr;
    const int at = on ? r : nr - 1;  // lanes past the last row do it again, and store nothing
    const uint16_t* row = src + (int64_t)at * p.ldqkv;
    const u32x4 wk[2] = {*reinterpret_cast<const u32x4*>(row + 8 * c), *reinterpret_cast<const u32x4*>(row + HD / 2 + 8 * c)};
    const Turn turn = load_turn<HD>(p.kn, p.cos + (t0 + at) * HD, p.sin + (t0 + at) * HD, c);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(row + (int64_t)kv.nkvh * HD + 16 * c + 8 * u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (on) *reinterpret_cast<uint32_t*>(&tile[r][16 * c + 8 * u + 2 * e]) = w[e];
        if constexpr (F8) {
          const f32x2 f = widen2<DT>(w[e]);
          va = fmaxf(va, fmaxf(finite_abs(f[0]), finite_abs(f[1])));
        }
      }
    }
    if constexpr (F8) norm_rope_exact<DT, HD>(wk[0], wk[1], turn, p.eps, xa[i], xb[i]);
    else norm_rope<DT, HD>(wk[0], wk[1], turn, p.eps, xa[i], xb[i]);
    if constexpr (F8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) ka = fmaxf(ka, fmaxf(finite_abs(xa[i][e]), finite_abs(xb[i][e])));
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

template <int DT, bool F8, int HD, int NP>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p, int64_t pages, int slots) {
  if ((int64_t)blockIdx.x < pages) kv_part<DT, F8, HD, NP>(p, blockIdx.x, slots);
  else q_part<DT, HD>(p, blockIdx.x - pages);
}

template <int DT, bool F8, int HD>
hipError_t launch_one(const AppendParams& p, hipStream_t s) {
  const int64_t slots = pages_touched(p.kv.max_rows, p.kv.lp), pages = slots * p.kv.seqs * p.kv.nkvh;
  const dim3 grid((unsigned)(pages + (p.kv.tokens + 3) / 4));
  if (HD == 128 && p.kv.lp == 6) hipLaunchKernelGGL((kv_append_kernel<DT, F8, HD, HD / 64>), grid, dim3(256), 0, s, p, pages, (int)slots);
  else hipLaunchKernelGGL((kv_append_kernel<DT, F8, HD, 1>), grid, dim3(256), 0, s, p, pages, (int)slots);
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

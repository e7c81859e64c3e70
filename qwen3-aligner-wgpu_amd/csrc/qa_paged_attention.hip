// qa_paged_attention.hip -- causal attention of a packed batch over the paged
// cache (16-bit or e4m3 pages), hd 64 or 128, any number of q heads to a kv head.
//
// Row i of a sequence with n rows and len keys sees keys 0 .. len - n + i:
// out = sum_t p_t v_t / sum_t p_t, p_t = exp(q.k_t / sqrt(hd) - max).  The q heads of a
// kv head and the rows of a sequence are one list, R = i * rep + head: a tile takes
// 16 of them to each of RT column groups, so a step of one token fills the matrix
// cores' columns with the q heads of its kv head, and a prompt with its rows.
//
// A wave takes 64 keys a step, K and V straight from the pages into fragments:
//  * S = K.Q^T on v_mfma_f32_16x16x32 (A = 16 keys x 32 d, B = the tile's q).  A lane
//    (c = lane & 15, g = lane >> 4) gets rows 4 g .. 4 g + 3 of each of four products;
//    row m of product t is given key 16 (m / 4) + 4 t + m % 4, so that the lane ends
//    up with keys 16 g .. 16 g + 15 of column c, all of them in one page.
//  * online softmax in the log2 domain; a lane has its column's statistics, joined
//    over g; the maximum moves only when it grows by more than 2^8.
//  * O^T += V^T.P^T: lane (d = c, g) reads keys 16 g .. of the page's V row d, 16 or 32
//    bytes in a run, in the order in which P lies in its registers.
// Probabilities go into the product as two 16-bit terms (value and rounding
// residue).  Over an e4m3 cache K is widened to the call's format (exactly), its
// scale goes into the score's factor, and V's into p in f32; P and V are
// multiplied as bf16 there, whose range takes any scale.
//
// Keys are split: a block's waves take turns at its 64-key blocks (WK) and join
// through LDS; beyond `chunk` keys further blocks take the next chunk, write
// (O, max, sum) to the workspace, and paged_join_kernel joins them.
#include "qa_internal.h"

namespace qa {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLazy = 8.f;  // the running maximum lags by up to this (log2)

template <int DT>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == QA_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == QA_F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
template <int DT>
__device__ __forceinline__ f32x2 unpack2(uint32_t h) {
  if constexpr (DT == QA_F16) return __builtin_convertvector(__builtin_bit_cast(f16x2, h), f32x2);
  else return (f32x2){__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)};
}
// Eight e4m3 values (two words) as a 16-bit fragment; exact in both formats.
template <int DT>
__device__ __forceinline__ u32x4 widen_e4m3(uint32_t a, uint32_t b) {
  if constexpr (DT == QA_F16)
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true))};
  else
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true))};
}

// Maximum and sum over the four lanes that share a column (lane ^ 16, lane ^ 32).
__device__ __forceinline__ float column_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// How a sequence's rows and keys are divided among blocks of 256 threads: tiles
// of WQ x RT x 16 rows (few rows: one column group, all waves on the keys), chunks
// of keys.  Both kernels and the host go by it.
constexpr int kFewRows = 16;
struct Split {
  int few_chunk, few_chunks;    // sequences of at most kFewRows (row, head) pairs
  int many_chunk, many_chunks;  // the others
  int tiles;                    // tiles of the longest of those, 0: there are none
  int units;                    // blocks per sequence and kv head
  int parts;                    // partial results per row, 1: no workspace
};
constexpr int kManyRT = 2, kManyWQ = 4;

Split split_of(const PagedAttnParams& p) {
  Split s{};
  const int64_t rows = (int64_t)p.kv.max_rows * p.rep, len = p.kv.max_len > 1 ? p.kv.max_len : 1;
  const bool many = rows > kFewRows;
  const int64_t heads = (int64_t)p.kv.seqs * p.kv.nkvh;
  auto divide = [&](int64_t blocks, int64_t want, int64_t least, int* chunk, int* chunks) {
    int64_t parts = blocks > 0 ? (want + blocks - 1) / blocks : 1;
    int64_t c = (len + parts - 1) / parts;
    c = (c < least ? least : c) + 255 & ~(int64_t)255;
    *chunk = (int)c;
    *chunks = (int)((len + c - 1) / c);
  };
  divide(heads, 1024, 512, &s.few_chunk, &s.few_chunks);
  if (many) {
    constexpr int tr = 16 * kManyRT * kManyWQ;
    s.tiles = (int)((rows + tr - 1) / tr);
    divide(heads * s.tiles, 512, 512, &s.many_chunk, &s.many_chunks);
  }
  s.units = s.tiles * s.many_chunks > s.few_chunks ? s.tiles * s.many_chunks : s.few_chunks;
  s.parts = s.many_chunks > s.few_chunks ? s.many_chunks : s.few_chunks;
  return s;
}

// Partial results in the workspace: O of (row, head, part), then its max and sum.
__device__ __forceinline__ int64_t part_index(const PagedAttnParams& p, const Split& sp, int64_t t, int head, int part) {
  return (t * p.nqh + head) * sp.parts + part;
}
__device__ __forceinline__ float* part_stats(const PagedAttnParams& p, const Split& sp, int hd) {
  return p.ws + p.kv.tokens * p.nqh * sp.parts * hd;
}

// One tile over the keys of one chunk.
template <int DT, bool F8, int HD, int RT, int WQ, int WK>
__device__ __forceinline__ void tile_body(const PagedAttnParams& p, const Split& sp, const SeqSpan& sq, int s, int h, int tile,
                                          int part, int chunk, unsigned char* smem) {
  constexpr int PV = F8 ? (int)QA_BF16 : DT;  // format of the P.V product
  constexpr float kBias = PV == QA_F16 ? 7.f : 0.f;  // f16 p scaled by 2^7: normal down to 2^-21
  constexpr int ES = F8 ? 1 : 2, E16 = 16 / ES;  // element size, elements of 16 bytes
  constexpr int KS = HD * ES / 64;               // 64-byte slices of a K row
  constexpr int QS = HD / 32;                    // products over d
  constexpr int ND = HD / 16;                    // d tiles
  constexpr int VS = F8 ? 1 : 2;                 // 16-byte loads of a V row's 16 keys
  const PagedParams& kv = p.kv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int wq = wave / WK, wk = wave % WK;
  const int R0 = (tile * WQ + wq) * RT * 16, NR = sq.n * p.rep;

  // rows of this lane's columns; columns past the last repeat it and store nothing
  int pos[RT], head[RT];
  int64_t tok[RT];
  u32x4 q[RT][QS];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int R = min(R0 + r * 16 + c, NR - 1);
    const int i = R / p.rep;
    head[r] = h * p.rep + R % p.rep;
    tok[r] = sq.row0 + i;
    pos[r] = sq.pos0 + i;
    const uint16_t* src = p.q + tok[r] * p.ldq + (int64_t)head[r] * HD;
#pragma unroll
    for (int e = 0; e < QS; ++e)
      q[r][e] = *reinterpret_cast<const u32x4*>(src + (F8 ? (e >> 1) * 64 + g * 16 + (e & 1) * 8 : e * 32 + g * 8));
  }
  const int top = sq.pos0 + (min(R0 + RT * 16, NR) - 1) / p.rep + 1;  // keys that the wave's last row sees
  const int k0 = part * chunk, k1 = min(k0 + chunk, top);
  const int nb = R0 < NR && k1 > k0 ? (k1 - k0 + 63) / 64 : 0;
  const int steps = (nb - wk + WK - 1) / WK;

  f32x4 o[RT][ND] = {};
  float m[RT], l[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  const int pmask = (1 << kv.lp) - 1;
  const int gk = c >> 2;  // the 16-key group that this lane's K rows are in
  auto key_of = [&](int it) { return k0 + (wk + it * WK) * 64; };
  auto id_of = [&](int pos) { return pos < sq.len ? page_at(kv, s, pos) : -1; };
  u32x4 kr[4][KS], vr[ND][VS];
  float ks = 1.f, vs = 0.f;
  auto load_k = [&](int it, int id) {
    const int64_t at = page_base(kv, max(id, 0), h, HD) + (int64_t)(((key_of(it) + 16 * gk) & pmask) + (c & 3)) * HD + g * E16;
    const unsigned char* src = (const unsigned char*)kv.k + at * ES;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < KS; ++e) kr[t][e] = *reinterpret_cast<const u32x4*>(src + 4 * t * HD * ES + e * 64);
  };
  auto load_v = [&](int it, int id) {
    const int64_t at = page_base(kv, max(id, 0), h, HD) + ((int64_t)c << kv.lp) + ((key_of(it) + 16 * g) & pmask);
    const unsigned char* src = (const unsigned char*)kv.v + at * ES;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < VS; ++e) vr[d][e] = *reinterpret_cast<const u32x4*>(src + (((int64_t)d * 16 << kv.lp) * ES + e * 16));
  };
  auto load_scales = [&](int id, float* a, float* b) {
    if constexpr (F8) {
      const int64_t at = (int64_t)max(id, 0) * kv.nkvh + h;
      const float x = kv.k_scale[at], y = kv.v_scale[at];
      *a = id < 0 ? 1.f : x;
      *b = id < 0 ? 0.f : y;
    }
  };

  int idk = -1, idv = -1, idk1 = -1, idv1 = -1;
  float ks1 = 1.f, vs1 = 0.f;
  if (steps > 0) {
    idk = id_of(key_of(0) + 16 * gk);
    idv = id_of(key_of(0) + 16 * g);
    if (steps > 1) {
      idk1 = id_of(key_of(1) + 16 * gk);
      idv1 = id_of(key_of(1) + 16 * g);
    }
    load_k(0, idk);
    load_v(0, idv);
    load_scales(idv, &ks, &vs);
  }
  for (int it = 0; it < steps; ++it) {
    const int kg = key_of(it) + 16 * g;  // the lane's first key
    // S = K.Q^T
    f32x4 sc[RT][4] = {};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < QS; ++e) {
        u32x4 a;
        if constexpr (F8) a = widen_e4m3<DT>(kr[t][e >> 1][2 * (e & 1)], kr[t][e >> 1][2 * (e & 1) + 1]);
        else a = kr[t][e];
#pragma unroll
        for (int r = 0; r < RT; ++r) sc[r][t] = mfma<DT>(a, q[r][e], sc[r][t]);
      }
    // the next block's K, and the page ids of the one after
    const int idv_now = idv;
    if (it + 1 < steps) {
      load_k(it + 1, idk1);
      load_scales(idv1, &ks1, &vs1);
      idk = idk1;
      idv = idv1;
      if (it + 2 < steps) {
        idk1 = id_of(key_of(it + 2) + 16 * gk);
        idv1 = id_of(key_of(it + 2) + 16 * g);
      }
    }
    // keys of the lane that the sequence has; what lies behind them, or on no
    // page, may hold anything, NaN too, and 0 * NaN is not 0
    const int have = idv_now < 0 ? 0 : sq.len - kg;
    const float f = p.scale * kLog2e * ks;
    u32x4 ph[RT][2], pl[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int see = min(have, pos[r] + 1 - kg);
      if (__builtin_amdgcn_ballot_w64(see < 16)) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * t + e >= see) sc[r][t][e] = -INFINITY;
      }
      float x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] = fmaxf(fmaxf(sc[r][t][0], sc[r][t][1]), fmaxf(sc[r][t][2], sc[r][t][3]));
      const float bm = column_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * f);
      if (__builtin_amdgcn_ballot_w64(bm > m[r] + kLazy)) {
        const float mn = fmaxf(m[r], bm);
        const float al = __builtin_amdgcn_exp2f(m[r] - (mn == -INFINITY ? 0.f : mn));
        l[r] *= al;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[r][d] *= al;
        m[r] = mn;
      }
      const float mb = (m[r] == -INFINITY ? 0.f : m[r]) - kBias;
      float sum[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][t][e], f, -mb));
        sum[t] = (w[0] + w[1]) + (w[2] + w[3]);
        if constexpr (F8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] *= vs;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t hi = pack2<PV>(w[2 * e], w[2 * e + 1]);
          const f32x2 b = unpack2<PV>(hi);
          ph[r][t >> 1][2 * (t & 1) + e] = hi;
          pl[r][t >> 1][2 * (t & 1) + e] = pack2<PV>(w[2 * e] - b[0], w[2 * e + 1] - b[1]);
        }
      }
      l[r] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    if (__builtin_amdgcn_ballot_w64(have < 16)) {
#pragma unroll
      for (int w = 0; w < VS * 4; ++w) {
        const int n = have - w * (4 / ES);  // elements of word w that are keys
        const uint32_t mask = n >= 4 / ES ? ~0u : n <= 0 ? 0u : (1u << (8 * ES * n)) - 1;
#pragma unroll
        for (int d = 0; d < ND; ++d) vr[d][w >> 2][w & 3] &= mask;
      }
    }
    // O^T += V^T.P^T
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u32x4 a;
        if constexpr (F8) a = widen_e4m3<QA_BF16>(vr[d][0][2 * j], vr[d][0][2 * j + 1]);
        else a = vr[d][j];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          o[r][d] = mfma<PV>(a, ph[r][j], o[r][d]);
          o[r][d] = mfma<PV>(a, pl[r][j], o[r][d]);
        }
      }
    if (it + 1 < steps) load_v(it + 1, idv);
    ks = ks1;
    vs = vs1;
  }

#pragma unroll
  for (int r = 0; r < RT; ++r) l[r] = column_sum(l[r]);
  // this wave's d tiles of the block's result, joined over the WK waves in order
  constexpr int NM = ND / WK;
  f32x4 w[RT][NM];
  if constexpr (WK > 1) {
    f32x4* xo = reinterpret_cast<f32x4*>(smem);                                         // [wave][RT][ND][64]
    float* xs = reinterpret_cast<float*>(smem + (size_t)WQ * WK * RT * ND * 64 * 16);   // [wave][RT][2][64]
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int d = 0; d < ND; ++d) xo[((wave * RT + r) * ND + d) * 64 + lane] = o[r][d];
      xs[((wave * RT + r) * 2) * 64 + lane] = m[r];
      xs[((wave * RT + r) * 2 + 1) * 64 + lane] = l[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float mm = -INFINITY;
      for (int a = 0; a < WK; ++a) mm = fmaxf(mm, xs[(((wq * WK + a) * RT + r) * 2) * 64 + lane]);
      const float mu = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
#pragma unroll
      for (int d = 0; d < NM; ++d) w[r][d] = f32x4{0, 0, 0, 0};
      for (int a = 0; a < WK; ++a) {
        const int at = (wq * WK + a) * RT + r;
        const float al = __builtin_amdgcn_exp2f(xs[at * 2 * 64 + lane] - mu);
        ll += xs[(at * 2 + 1) * 64 + lane] * al;
#pragma unroll
        for (int d = 0; d < NM; ++d) w[r][d] += xo[(at * ND + wk * NM + d) * 64 + lane] * al;
      }
      m[r] = mm;
      l[r] = ll;
    }
  } else {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int d = 0; d < NM; ++d) w[r][d] = o[r][d];
  }
  // the tile's keys are one chunk: the result; else its part of it
  const int last = min((tile + 1) * WQ * RT * 16, NR) - 1;
  const bool whole = sq.pos0 + last / p.rep + 1 <= chunk;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (R0 + r * 16 + c >= NR) continue;
    if (whole) {
      const float inv = l[r] == 0.f ? 0.f : 1.0f / l[r];  // no key: zeros
      uint16_t* dst = p.out + tok[r] * p.ldo + (int64_t)head[r] * HD + 4 * g;
#pragma unroll
      for (int d = 0; d < NM; ++d) {
        const f32x4 y = w[r][d] * inv;
        *reinterpret_cast<u32x2*>(dst + (wk * NM + d) * 16) = u32x2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
      }
    } else {
      const int64_t at = part_index(p, sp, tok[r], head[r], part);
      float* dst = p.ws + at * HD + 4 * g;
#pragma unroll
      for (int d = 0; d < NM; ++d) *reinterpret_cast<f32x4*>(dst + (wk * NM + d) * 16) = w[r][d];
      if (wk == 0 && g == 0) {
        float* st = part_stats(p, sp, HD) + at * 2;
        st[0] = m[r];
        st[1] = l[r];
      }
    }
  }
}

template <int HD, int RT, int WQ, int WK>
constexpr int body_lds() {
  return WK > 1 ? WQ * WK * RT * 64 * (HD / 16 * 16 + 8) : 16;
}

// Block -> kv head fastest (with 8 of them a head's blocks share an XCD's L2), then
// unit, then sequence.  A sequence's units are its chunks, or its tiles times
// their chunks, the last tiles (the longest) first.
template <int DT, bool F8, int HD, bool MANY>
__global__ void __launch_bounds__(256, MANY ? 1 : 2) paged_attention_kernel(const PagedAttnParams p, const Split sp) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[body_lds<HD, 1, 1, 4>()];
  const int h = (int)(blockIdx.x % p.kv.nkvh);
  const int u = (int)(blockIdx.x / p.kv.nkvh % sp.units), s = (int)(blockIdx.x / p.kv.nkvh / sp.units);
  const SeqSpan sq = seq_span(p.kv, s);
  if (sq.n == 0) return;
  const int NR = sq.n * p.rep;
  if (!MANY || NR <= kFewRows) {
    if (u >= sp.few_chunks || (u > 0 && u * sp.few_chunk >= sq.pos0 + sq.n)) return;
    tile_body<DT, F8, HD, 1, 1, 4>(p, sp, sq, s, h, 0, u, sp.few_chunk, smem);
  } else {
    constexpr int tr = 16 * kManyRT * kManyWQ;
    const int tiles = (NR + tr - 1) / tr;
    const int tile = tiles - 1 - u % sp.tiles, part = u / sp.tiles;
    if (tile < 0 || part >= sp.many_chunks) return;
    const int last = min((tile + 1) * tr, NR) - 1;
    if (part > 0 && part * sp.many_chunk >= sq.pos0 + last / p.rep + 1) return;
    tile_body<DT, F8, HD, kManyRT, kManyWQ, 1>(p, sp, sq, s, h, tile, part, sp.many_chunk, smem);
  }
}

// The parts of a row and head joined: one wave each, HD / 64 elements a lane.
template <int DT, int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttnParams p, const Split sp) {
  const int lane = threadIdx.x & 63;
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int head = (int)(b % p.nqh);
  const int64_t si = b / p.nqh;
  const int s = (int)(si / p.kv.max_rows), i = (int)(si % p.kv.max_rows);
  if (s >= p.kv.seqs) return;
  const SeqSpan sq = seq_span(p.kv, s);
  if (i >= sq.n) return;
  const int NR = sq.n * p.rep, R = i * p.rep + head % p.rep;
  const bool few = NR <= kFewRows;
  constexpr int tr = 16 * kManyRT * kManyWQ;
  const int last = few ? NR - 1 : min((R / tr + 1) * tr, NR) - 1;
  const int chunk = few ? sp.few_chunk : sp.many_chunk, keys = sq.pos0 + last / p.rep + 1;
  if (keys <= chunk) return;  // its tile has written the result
  const int parts = (keys + chunk - 1) / chunk;
  const int64_t t = sq.row0 + i, at = part_index(p, sp, t, head, 0);
  const float* st = part_stats(p, sp, HD) + at * 2;
  float mm = -INFINITY;
  for (int a = lane; a < parts; a += 64) mm = fmaxf(mm, st[2 * a]);
#pragma unroll
  for (int e = 32; e > 0; e >>= 1) mm = fmaxf(mm, __shfl_xor(mm, e, 64));
  const float mu = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, y[HD / 64] = {};
  const float* src = p.ws + at * HD + lane * (HD / 64);
  for (int a = 0; a < parts; ++a) {
    const float al = __builtin_amdgcn_exp2f(st[2 * a] - mu);
    ll += st[2 * a + 1] * al;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) y[e] += src[(int64_t)a * HD + e] * al;
  }
  const float inv = ll == 0.f ? 0.f : 1.0f / ll;
  uint16_t* dst = p.out + t * p.ldo + (int64_t)head * HD + lane * (HD / 64);
  if constexpr (HD == 128) *reinterpret_cast<uint32_t*>(dst) = pack2<DT>(y[0] * inv, y[1] * inv);
  else *dst = (uint16_t)pack2<DT>(y[0] * inv, 0.f);
}

template <int DT, bool F8, int HD>
hipError_t launch_one(const PagedAttnParams& p, hipStream_t s) {
  const Split sp = split_of(p);
  const dim3 grid((unsigned)((int64_t)p.kv.seqs * p.kv.nkvh * sp.units));
  if (sp.tiles) hipLaunchKernelGGL((paged_attention_kernel<DT, F8, HD, true>), grid, dim3(256), 0, s, p, sp);
  else hipLaunchKernelGGL((paged_attention_kernel<DT, F8, HD, false>), grid, dim3(256), 0, s, p, sp);
  if (sp.parts > 1) {
    const int64_t rows = (int64_t)p.kv.seqs * p.kv.max_rows * p.nqh;
    hipLaunchKernelGGL((paged_join_kernel<DT, HD>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p, sp);
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(bool e4m3, int hd, const PagedAttnParams& p, hipStream_t s) {
  if (hd == 64) return e4m3 ? launch_one<DT, true, 64>(p, s) : launch_one<DT, false, 64>(p, s);
  return e4m3 ? launch_one<DT, true, 128>(p, s) : launch_one<DT, false, 128>(p, s);
}

}  // namespace

int64_t paged_attention_blocks(const PagedAttnParams& p) {
  const Split sp = split_of(p);
  const int64_t rows = (int64_t)p.kv.seqs * p.kv.max_rows, blocks = (int64_t)p.kv.seqs * p.kv.nkvh;
  // saturating: the caller compares with a bound far below
  const double most = (double)rows * p.nqh > (double)blocks * sp.units ? (double)rows * p.nqh : (double)blocks * sp.units;
  return most > 9e18 ? INT64_MAX : (int64_t)most;
}

size_t paged_attention_workspace(int hd, const PagedAttnParams& p) {
  const Split sp = split_of(p);
  return sp.parts > 1 ? (size_t)p.kv.tokens * p.nqh * sp.parts * (hd + 2) * sizeof(float) : 0;
}

hipError_t launch_attention_paged(int dtype, bool e4m3, int hd, const PagedAttnParams& p, hipStream_t s) {
  return dtype == QA_BF16 ? launch_dt<QA_BF16>(e4m3, hd, p, s) : launch_dt<QA_F16>(e4m3, hd, p, s);
}

}  // namespace qa

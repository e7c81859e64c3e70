// qa_paged_attention.hip -- causal attention of a packed batch over the paged
// cache (16-bit or e4m3 pages), hd 64 or 128, any number of q heads to a kv head.
//
// Row i of a sequence with n rows and len keys sees keys 0 .. len - n + i:
// out = sum_t p_t v_t / sum_t p_t, p_t = exp(q.k_t / sqrt(hd) - max).  The q heads of a
// kv head and the rows of a sequence are one list, R = i * rep + head, and a tile
// takes 16, 64 or 128 of its pairs as the columns of the products S = K.Q^T and
// O^T += V^T.P^T: a step of one token fills columns with the q heads of its kv head, a
// prompt with its rows, and every key is read once for all of them.
//
// K and V go to LDS in blocks of 64 keys by DMA (buffer_load ... lds), page by page, a
// page's resource being its own bytes, so that a hole in the table comes as
// zeros.  (Straight from the pages into fragments, a load instruction touches 16
// rows, and the address unit bounds the kernel: 90 us where the tiles take 33.)  Chunks of
// 16 bytes lie within their row in an order that leaves fragment reads without
// bank conflicts (0.3 % of LDS cycles; 28 % in plain order).  The rows of a product
// are given those keys that leave a lane with 16 consecutive keys of its column, in the
// order in which its fragment of V has them: P goes from one product into the
// other in registers.
//
// Online softmax in the log2 domain; the maximum moves only when it grows by more
// than 2^8, so nearly every step leaves O as it is.  Over an e4m3 cache K is widened
// to the call's format (exactly), its scale goes into the score's factor, and V's into
// p in f32; P and V are multiplied as bf16 there, whose range takes any scale.
// Probabilities go into the product as a sum of 16-bit terms, a value and the rounding
// of what it leaves: two of f16 (scaled by 2^7, so that small ones stay normal),
// which hold 22 bits of p, or three of bf16, which hold all 24.  (Two of bf16 hold 16:
// 2.3e-6 of the result, which moved 0.24 % of bf16 outputs to the neighbouring value
// where three move 0.06 %, as many as a sum in another order; 64 sequences over e4m3
// 127.4 us with two, 127.9 with three.)  Two of bf16 are left in the longer tiles over
// bf16 pages, as in qa_attention_prefill's default, where a third product costs most: 771
// rows behind 1536 keys 33.5 us with two, 38.7 with three (e4m3 pages 37.5 and 42.3).
//
// Sequences of up to 16 pairs (single tokens): paged_few_kernel.  Bound by the
// cache's bytes: 32 sequences of up to 4353 keys, 8 kv heads of 128, 342 MB in f16: 69 us,
// 4.9 TB/s (a large copy: 5.1); 64 of up to 8193 in e4m3, 598 MB: 127 us, 4.7 TB/s.  The
// smallest calls by latency: one sequence of 323 keys 8.4 us, of which launching is 4.
// Longer ones: paged_many_kernel, bound by the two phases of a step, of which the
// softmax is as long as the products: 771 rows behind 1536 keys, 16 heads of 128:
// 33 us, 367 TFLOP/s, 550 with the products of the residues.
// Keys of long sequences are split among blocks, which leave (O, max, sum) in the
// workspace for paged_join_kernel.
#include <utility>

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
// (a, b) minus the 16-bit values h = pack2(a, b), exact in f32, rounded
// to two 16-bit values again.  f16: as products with a 1 that the compiler does
// not see, which become one v_fma_mix each, h's half read and the result's
// written as they lie.
template <int DT>
__device__ __forceinline__ uint32_t residue2(uint32_t h, float a, float b) {
  if constexpr (DT == QA_F16) {
    const f16x2 v = __builtin_bit_cast(f16x2, h);
    float one = 1.f;
    asm("" : "+s"(one));
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)__builtin_fmaf(-(float)v[0], one, a), (_Float16)__builtin_fmaf(-(float)v[1], one, b)});
  } else {
    return pack2<DT>(a - __uint_as_float(h << 16), b - __uint_as_float(h & 0xffff0000u));
  }
}
// What a second term leaves, of bf16.
__device__ __forceinline__ uint32_t residue2(uint32_t h, uint32_t l, float a, float b) {
  a -= __uint_as_float(h << 16);
  b -= __uint_as_float(h & 0xffff0000u);
  return residue2<QA_BF16>(l, a, b);
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

#define QA_LDS __attribute__((address_space(3)))

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// Every LDS read so far has its data: what it read may be overwritten.
__device__ __forceinline__ void wait_lds() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4) | (0x0 << 8));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A value that all of a wave's lanes have, as a scalar.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// m = max(m, a, b, c, d) in two instructions: the maximum of a product's elements
// alone would take each of them through an instruction of its own first.
__device__ __forceinline__ void max4(float& m, float a, float b, float c, float d) {
  m = fmaxf(fmaxf(m, a), b);
  m = fmaxf(fmaxf(m, c), d);
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

// Sizes that a call's formats give.
template <int DT, bool F8, int HD>
struct Cfg {
  static constexpr int PV = F8 ? (int)QA_BF16 : DT;              // format of the P.V product
  static constexpr int NT = PV == QA_F16 ? 2 : 3;                // 16-bit terms of a probability
  static constexpr int NL = F8 ? 3 : 2;                          // in the longer tiles
  static constexpr float kBias = PV == QA_F16 ? 7.f : 0.f;       // f16 p scaled by 2^7: normal down to 2^-21
  static constexpr int ES = F8 ? 1 : 2;                          // bytes of a cache element
  static constexpr int CR = HD * ES / 16;                        // 16-byte chunks of a K row
  static constexpr int LCR = CR == 16 ? 4 : CR == 8 ? 3 : 2;
  static constexpr int KS = CR / 4;                              // 64-byte slices of a K row
  static constexpr int QS = HD / 32;                             // products over d
  static constexpr int ND = HD / 16;                             // d tiles
  static constexpr int VS = F8 ? 1 : 2;                          // chunks of a V row's 16 keys
  static constexpr int LI = CR;                                  // DMA instructions of a tile, K's and V's alike
  static constexpr int TILE = 64 * HD * ES;                      // bytes of a K or V tile
};

// How a call's rows and keys are divided among blocks, from its sizes alone (lengths
// are on the device), so that the workspace is known without one.
//  * few: a sequence of at most kFewRows (row, head) pairs is one column group; a
//    block's four waves take turns at a part of its keys, each with tiles of its own.
//    Bound by the cache's bytes, so a sequence is cut where its block alone would be
//    at work after the others, or CUs have none: a join costs about 5 us.  Unsplit up to
//    20 keys for each sequence and kv head of the batch (us, unsplit / the best split;
//    f16, hd 128: 64 of them behind up to 700 keys 10.8 / 11.0, 1500 15.5 / 13.4; 128
//    behind 1500 17.1 / 19.2, 4300 49.1 / 39.3; 256 behind 4300 70.5 / 73.3), and up to
//    4096 keys past 256 of them (512 behind 3300 93.7 / 93.9, e4m3 4352 73.2 / 67.5).
//    That line is good at full rounds of blocks; where the last round has few, the best
//    split wins earlier (all as long, f16, hd 128: 264 behind 1000 32.3 / 34.7, 2000 58.4 /
//    49.8, 4096 127.5 / 105.0; 320 behind 1000 32.8 / 36.6, 2000 66.5 / 62.4, 4096 133.1 /
//    122.6; 384 behind 4096 140.6 / 142.6; 576 behind 4096 222.4 / 210.8; e4m3 264 behind
//    4096 63.0 / 51.4, 320 71.6 / 63.2, 384 81.3 / 78.0).
//    Else into parts that give every CU its blocks (one, or two of e4m3 or hd 64, by
//    their LDS), and with more sequences into more, down to about 1024 keys, as their
//    joins are one launch (e4m3, 512 behind 8192, in 1, 3, 5, 9 parts: 133.6, 124.7, 122.8,
//    121.1; f16, 64 behind 8192 in 5 and 9: 26.5, 28.8).  The number is odd: blocks go to
//    CUs in turns, and with an even one the same CUs get all the first, full parts
//    (512 behind 4352, f16, in 3, 4, 5: 118.6, 148.9, 122).  A part is a multiple of 256
//    keys, a block of 64 for each wave.
//  * many: tiles of 64 or 128 pairs.  Of 64 up to 600 tiles: 128-row blocks load each
//    tile for twice the rows, but are half as many, each with twice the steps (8 kv
//    heads of 128, no past, 64 / 128, us: 1500 rows 28.1 / 37.9, 2500 62.6 / 59.8, 3500
//    101.7 / 86.2, 4334 153 / 141; prompts of 323 rows, 4 of them 20.9 / 16.2, which the
//    line misses, 8 32.2 / 29.3, 16 60.5 / 45.2; of 771, 2 24.0 / 24.5, 4 43.7 / 39.2; 2 of
//    1500 55.2 / 44.2; one of 4334 and 4 of 771 188 / 167, in either order; e4m3: 4 of 323
//    23.0 / 19.3, 8 35.5 / 34.9, 2 of 771 27.2 / 31.9, 4 51.6 / 49.3).
//    Their keys are split while the CUs take the parts at once, down to 256: 64 rows
//    behind 16000 keys 166 us whole, 28.8 in 32 parts; 200 behind 700 18.1 whole, 16.3 in
//    four; 8 prompts of up to 100 rows behind 1500 (4 of 64) 24.2 whole, 20.4 in the two
//    that this gives, 19.7 in three; but 771 behind 1536 (200 blocks) 32 whole, 43 in two,
//    as half the CUs' parts have to wait.  Up to 640 keys there is no gain (600 and none
//    before, 4 kv heads of 64: 12.4 whole, 13.5 in three).
//  * kCus is a whole device's: the workspace has to be known without a device, so that
//    on a partition of one the parts are more than its CUs need.
constexpr int kFewRows = 16, kFewWaves = 4;
constexpr int kManyWaves = 8;
constexpr int kCus = 256;
struct Split {
  int few, many;                // which of the two kinds the batch may hold
  int few_chunk, few_chunks;    // keys of a part, parts of the longest sequence
  int many_chunk, many_chunks;
  int many_rows;                // pairs of a tile
  int tiles;                    // tiles that all sequences of `many` can have together
  int few_pairs;                // pairs that a sequence of `few` can have
  int by_seq;                   // where partial results of `few` lie, see part_index()
  int64_t few_parts, many_parts;  // partial results of either kind in the workspace
};

Split split_of(const PagedAttnParams& p, bool e4m3, int hd) {
  Split s{};
  const int64_t rows = (int64_t)p.kv.max_rows * p.rep, len = p.kv.max_len > 1 ? p.kv.max_len : 1;
  const int64_t heads = (int64_t)p.kv.seqs * p.kv.nkvh;
  auto divide = [&](int64_t parts, int64_t least, int* chunk, int* chunks) {
    int64_t c = (len + parts - 1) / parts;
    c = ((c < least ? least : c) + 255) & ~(int64_t)255;
    *chunk = (int)c;
    *chunks = (int)((len + c - 1) / c);
  };
  s.many = rows > kFewRows;
  // where every sequence has to have the most rows for the batch to be as long as
  // it is, none is a short one
  s.few = !s.many || (int64_t)p.kv.seqs * p.kv.max_rows > p.kv.tokens;
  s.few_chunks = s.many_chunks = 1;
  if (s.few) {
    const int64_t slots = !e4m3 && hd == 128 ? kCus : 2 * kCus;  // blocks that are at work at once
    const int64_t whole = heads <= kCus ? 20 * heads : 4096;
    int64_t parts = 1;
    if (heads > 0 && len > (whole > 512 ? whole : 512)) {
      const int64_t fill = (slots + heads - 1) / heads;
      const int64_t some = (heads < 4096 ? heads : 4096) * len * slots >> 26, most = len / 1024, even = some < most ? some : most;
      parts = (fill > even ? fill : even) | 1;
      parts = parts < 33 ? parts : 33;
    }
    // (rounding a part to 256 keys may leave an even number of them)
    do divide(parts, 256, &s.few_chunk, &s.few_chunks);
    while (s.few_chunks % 2 == 0 && s.few_chunk > 256 && heads * s.few_chunks > slots && (parts += 2));
  }
  if (s.many) {
    // full tiles of a batch of this many rows, and a sequence's short last one; a
    // sequence has to have rows for that, more than few where `few` takes the others
    const int64_t pairs = p.kv.tokens * p.rep, least = s.few ? kFewRows + 1 : p.rep;
    const int64_t ends = pairs / least < p.kv.seqs ? pairs / least : p.kv.seqs;
    // what there will be: at least a tile of each such sequence, or the short ones of
    // as few sequences as have the rows
    const int64_t full = (p.kv.tokens + p.kv.max_rows - 1) / p.kv.max_rows;
    auto most = [&](int64_t r) { return p.kv.seqs * ((rows + r - 1) / r); };
    auto about = [&](int64_t r) {
      const int64_t n = pairs / r + full > ends ? pairs / r + full : ends;
      return p.kv.nkvh * (n < most(r) ? n : most(r));
    };
    s.many_rows = about(64) > 600 ? 128 : 64;
    s.tiles = (int)(pairs / s.many_rows + ends < most(s.many_rows) ? pairs / s.many_rows + ends : most(s.many_rows));
    const int64_t blocks = about(s.many_rows);
    divide(len > 640 && blocks > 0 && blocks < kCus ? kCus / blocks : 1, 256, &s.many_chunk, &s.many_chunks);
  }
  s.few_pairs = (int)(rows < kFewRows ? rows : kFewRows);
  const int64_t of_rows = p.kv.tokens * p.nqh, of_seqs = heads * s.few_pairs;
  s.by_seq = of_seqs < of_rows;
  s.few_parts = s.few_chunks > 1 ? (s.by_seq ? of_seqs : of_rows) * s.few_chunks : 0;
  s.many_parts = s.many_chunks > 1 ? of_rows * s.many_chunks : 0;
  return s;
}

// Partial results in the workspace: all their O's, then all their maxima and sums.
// First those of short sequences, by (sequence, kv head, pair) or by (row, head), of
// which the sizes allow fewer: a prompt's rows in the batch take none of these many
// parts, nor one step's sequences the pairs of longer ones.  Then those of the
// longer tiles, by (row, head).  `pair`: of the sequence and kv head.
__device__ __forceinline__ int64_t part_index(const PagedAttnParams& p, const Split& sp, bool few, int s, int h, int pair, int64_t t, int head, int part) {
  if (!few) return sp.few_parts + (t * p.nqh + head) * sp.many_chunks + part;
  return (sp.by_seq ? ((int64_t)s * p.kv.nkvh + h) * sp.few_pairs + pair : t * p.nqh + head) * sp.few_chunks + part;
}
__device__ __forceinline__ float* part_stats(const PagedAttnParams& p, const Split& sp, int hd) {
  return p.ws + (sp.few_parts + sp.many_parts) * hd;
}

// The (row, head) pair of a lane's column; columns past the last repeat it and store
// nothing.
struct Column {
  int pos, head;
  int64_t tok;
  bool on;
  __device__ __forceinline__ void set(const PagedAttnParams& p, const SeqSpan& sq, int h, int c) {
    const int NR = sq.n * p.rep;
    asm volatile("" : "+v"(c));  // formed again for the result, not held across the loop
    on = c < NR;
    const int R = min(c, NR - 1), i = R / p.rep;
    head = h * p.rep + R % p.rep;
    tok = sq.row0 + i;
    pos = sq.pos0 + i;
  }
};

template <bool F8, int HD>
__device__ __forceinline__ void load_q(const PagedAttnParams& p, const Column& col, int g, u32x4 (&q)[HD / 32]) {
  const uint16_t* src = p.q + col.tok * p.ldq + (int64_t)col.head * HD;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e)  // in the order in which a K row's chunks come
    q[e] = *reinterpret_cast<const u32x4*>(src + (F8 ? (e >> 1) * 64 + g * 16 + (e & 1) * 8 : e * 32 + g * 8));
}

// The compiler waits here for q's loads, not at their use in the loop, where the
// tiles' loads would be waited for with them.
template <int N>
__device__ __forceinline__ void keep(u32x4 (&q)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) asm volatile("" : "+v"(q[e]));
}

// A 64-key block's K and V tiles in LDS.  K: 64 rows of CR chunks; V: the block's
// pages one after the other, each HD rows of CP chunks.  Both are copies of the
// pages but for the order of chunks within a row: chunk ^ f(row), with f such that
// the 16 lanes whose 16-byte reads the LDS serves at once (of lanes 0-31: 0-3,
// 12-15, 20-27 and the others) find 16 different bank groups.  In a fragment read
// lane (c, g) wants row c and a chunk that g adds to; so f depends on c, and for
// V on the page size.
__device__ __forceinline__ int swap3(int v) { return (0x1320 >> (4 * v)) & 3; }  // 0, 2, 3, 1
template <int CR>
__device__ __forceinline__ int k_swizzle(int c) {
  return CR == 16 ? c : CR == 8 ? c >> 1 : swap3(c >> 2);
}
template <bool F8>
__device__ __forceinline__ int v_swizzle(int c, int lcp) {
  if (F8) return lcp == 2 ? swap3(c >> 2) : 0;
  return lcp == 3 ? (c >> 1) & 5 : c >> 3;
}
// Where pages begin: lane 4 j + a holds, for the page of keys 16 a .. of block j, the
// bytes from either pool's start, or a negative number.
struct Pages {
  int lo, hi;
};
template <class F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// Block j's tile by DMA, 1 KB to an instruction; a tile's are dealt out to OF waves, of
// which this is `mine`.  A page's are a run of PER.  Pages that are none come as
// zeros (a resource of no bytes).  W32: in the order for the 32-row products below.
template <int DT, bool F8, int HD, bool W32, int OF, int LP, bool K>
__device__ __forceinline__ void load_tile(const PagedParams& kv, const Pages& pages, int j, int mine, unsigned char* to) {
  using C = Cfg<DT, F8, HD>;
  constexpr int PER = C::LI >> (6 - LP), PB = HD * C::ES << LP;  // instructions and bytes of a page
  constexpr int CW = K ? C::CR : (1 << LP) * C::ES / 16;          // chunks of a row
  int ln = threadIdx.x & 63;
  asm volatile("" : "+v"(ln));  // lane offsets are formed anew, not kept across the loop
  // the part of f(row) that the lane gives, and the one of instruction n of page pg
  int f;
  if constexpr (W32) f = (ln >> 4) & 3 & (CW - 1);  // chunk M of a page: f = (M / 16) % CW
  else if constexpr (K) f = CW == 16 ? ln >> 4 & 3 : CW == 8 ? ln >> 4 & 1 : 0;
  else if constexpr (F8) f = CW == 4 ? swap3(ln >> 4 & 3) : 0;
  else f = CW == 4 ? ln >> 5 : ln >> 4 & 1;
  const uint32_t lane_off = (uint32_t)((ln & ~(CW - 1)) | ((ln & (CW - 1)) ^ f)) * 16;
  auto off = [&](int n, int pg) {
    if constexpr (W32) return lane_off ^ (uint32_t)((4 * n & (CW - 1)) << 4);
    const int g = (pg << (LP - 4)) + n / C::KS;  // K: the 16 keys
    if constexpr (K) return lane_off ^ (uint32_t)((CW == 16 ? g << 2 : CW == 8 ? g << 1 : swap3(g)) << 4);
    return lane_off ^ (uint32_t)(!F8 && CW == 8 ? (n & 1) << 6 : 0);
  };
  auto page_src = [&](int pg, int* bytes) {
    const int lo = __builtin_amdgcn_readlane(pages.lo, j * 4 + (pg << (LP - 4)));
    const int hi = __builtin_amdgcn_readlane(pages.hi, j * 4 + (pg << (LP - 4)));
    *bytes = hi < 0 ? 0 : PB;
    return (const unsigned char*)(K ? kv.k : kv.v) + ((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
  };
  auto one = [&](auto number) {
    constexpr int I = decltype(number)::value;
    if constexpr (PER >= OF) {
      constexpr int PW = PER < OF ? 1 : PER / OF, pg = I / PW, N = I % PW * OF;  // N: of the page, the first wave's
      constexpr int B = N / 4 * 4096;                              // 4 KB: the reach of the instruction's offset
      int bytes;
      const unsigned char* src = page_src(pg, &bytes);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(src), (short)0, bytes, 0x00020000);
      QA_LDS void* dst = (QA_LDS void*)(to + pg * PER * 1024 + B + mine * 1024);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 16, off(N + mine, pg), B + mine * 1024, N % 4 * 1024, 0);
    } else {  // fewer instructions to a page than waves: pages side by side
      const int pg = I * (OF / PER) + mine / PER, n = mine % PER;
      int bytes;
      const unsigned char* src = page_src(pg, &bytes);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(src), (short)0, bytes, 0x00020000);
      QA_LDS void* dst = (QA_LDS void*)(to + (pg * PER + n) * 1024);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 16, off(n, pg), n * 1024, 0, 0);
    }
  };
  each(one, std::make_integer_sequence<int, C::LI / OF>{});
}
// Fragment addresses in the tiles.  K: product t reads row 16 (c / 4) + 4 t + c % 4,
// slice e the chunk 4 e + g.  V: row d, the chunks of keys 16 g ..
template <int DT, bool F8, int HD>
__device__ __forceinline__ int k_frag(int c, int g) {
  using C = Cfg<DT, F8, HD>;
  return ((16 * (c >> 2) + (c & 3)) * C::CR + (g ^ k_swizzle<C::CR>(c))) * 16;
}
template <int DT, bool F8, int HD>
__device__ __forceinline__ int v_frag(int c, int g, int e, int lcp) {
  const int x = g * Cfg<DT, F8, HD>::VS + e;  // the block's chunk x of this row
  return ((((x >> lcp) * HD + c) << lcp) + ((x & ((1 << lcp) - 1)) ^ v_swizzle<F8>(c, lcp))) * 16;
}

// Mask, online softmax and the 16-bit terms of P.  `have`: how many of the
// lane's 16 keys from kg on some row of the sequence sees (on a page); `f`: the scores'
// factor, log2 e / sqrt(hd) and the K scale; `vs`: the V scale.
template <int DT, bool F8, int HD>
__device__ __forceinline__ void softmax(f32x4 (&sc)[4], int pos, int kg, int have, float f, float vs, float& m, float& l, f32x4 (&o)[HD / 16],
                                        u32x4 (&ph)[2], u32x4 (&pl)[2], u32x4 (&pm)[2]) {
  using C = Cfg<DT, F8, HD>;
  const int see = min(have, pos + 1 - kg);
  if (__builtin_amdgcn_ballot_w64(see < 16)) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * t + e >= see) sc[t][e] = -INFINITY;
  }
  float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int t = 0; t < 4; ++t) max4(x[t & 1], sc[t][0], sc[t][1], sc[t][2], sc[t][3]);
  const float bm = column_max(fmaxf(x[0], x[1]) * f);
  if (__builtin_amdgcn_ballot_w64(bm > m + kLazy)) {
    const float mn = fmaxf(m, bm);
    const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    l *= al;
#pragma unroll
    for (int d = 0; d < C::ND; ++d) o[d] *= al;
    m = mn;
  }
  const float mb = (m == -INFINITY ? 0.f : m) - C::kBias;
  float sum[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e], f, -mb));
    sum[t] = (w[0] + w[1]) + (w[2] + w[3]);
    if constexpr (F8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] *= vs;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t hi = pack2<C::PV>(w[2 * e], w[2 * e + 1]), lo = residue2<C::PV>(hi, w[2 * e], w[2 * e + 1]);
      ph[t >> 1][2 * (t & 1) + e] = hi;
      pl[t >> 1][2 * (t & 1) + e] = lo;
      if constexpr (C::NT == 3) pm[t >> 1][2 * (t & 1) + e] = residue2(hi, lo, w[2 * e], w[2 * e + 1]);
    }
  }
  l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Mask of word w of a run of elements of which `left` are keys.
template <int ES>
__device__ __forceinline__ uint32_t tail_mask(int left, int w) {
  const int n = left - w * (4 / ES);
  return n >= 4 / ES ? ~0u : n <= 0 ? 0u : (1u << (8 * ES * n)) - 1;
}
// What a V tile holds behind the keys that rows see, or for no page, may be anything, NaN
// too, and 0 * NaN is not 0: a lane clears those elements of the chunks that it
// will read itself.
template <int DT, bool F8, int HD>
__device__ __forceinline__ void clear_tail(unsigned char* vt, const int (&va)[Cfg<DT, F8, HD>::VS], int lcp, int have) {
  using C = Cfg<DT, F8, HD>;
  uint32_t keep[C::VS * 4];
#pragma unroll
  for (int w = 0; w < C::VS * 4; ++w) keep[w] = tail_mask<C::ES>(have, w);
#pragma unroll 1
  for (int d = 0; d < C::ND; ++d)
#pragma unroll
    for (int e = 0; e < C::VS; ++e) {
      u32x4* x = reinterpret_cast<u32x4*>(vt + va[e] + (d * 256 << lcp));
      *x &= u32x4{keep[4 * e], keep[4 * e + 1], keep[4 * e + 2], keep[4 * e + 3]};
    }
}

// The products of a block: S = K.Q^T over the K tile at kt, and O^T += V^T.P^T over
// the V tile at vt, in slices (the 16 keys of a K product, a d tile of V), the
// fragments read kAhead slices before.  (The empty statements keep the fragments'
// addresses from being formed outside the loop and held there.)
constexpr int kAhead = 2;
template <int DT, bool F8, int HD>
__device__ __forceinline__ void multiply_k(const unsigned char* kt, int ka, const u32x4 (&q)[HD / 32], f32x4 (&sc)[4]) {
  using C = Cfg<DT, F8, HD>;
  constexpr int B = kAhead + 1;
  asm volatile("" : "+v"(ka));
  u32x4 x[B][C::KS];
  auto read = [&](int t) {
#pragma unroll
    for (int e = 0; e < C::KS; ++e) x[t % B][e] = *reinterpret_cast<const u32x4*>(kt + (ka ^ (e << 6)) + 4 * t * C::CR * 16);
  };
#pragma unroll
  for (int t = 0; t < kAhead; ++t) read(t);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t + kAhead < 4) read(t + kAhead);
#pragma unroll
    for (int e = 0; e < C::QS; ++e) {
      u32x4 a;
      if constexpr (F8) a = widen_e4m3<DT>(x[t % B][e >> 1][2 * (e & 1)], x[t % B][e >> 1][2 * (e & 1) + 1]);
      else a = x[t % B][e];
      sc[t] = mfma<DT>(a, q[e], e ? sc[t] : f32x4{0, 0, 0, 0});
    }
  }
}
template <int DT, bool F8, int HD>
__device__ __forceinline__ void multiply_v(const unsigned char* vt, const int (&va)[Cfg<DT, F8, HD>::VS], int lcp, const u32x4 (&ph)[2],
                                           const u32x4 (&pl)[2], const u32x4 (&pm)[2], f32x4 (&o)[HD / 16]) {
  using C = Cfg<DT, F8, HD>;
  constexpr int B = kAhead + 1;
  int at[C::VS];
#pragma unroll
  for (int e = 0; e < C::VS; ++e) {
    at[e] = va[e];
    asm volatile("" : "+v"(at[e]));
  }
  u32x4 x[B][C::VS];
  auto read = [&](int d) {
#pragma unroll
    for (int e = 0; e < C::VS; ++e) x[d % B][e] = *reinterpret_cast<const u32x4*>(vt + at[e] + (d * 256 << lcp));
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) read(d);
#pragma unroll
  for (int d = 0; d < C::ND; ++d) {
    if (d + kAhead < C::ND) read(d + kAhead);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4 a;
      if constexpr (F8) a = widen_e4m3<QA_BF16>(x[d % B][0][2 * j], x[d % B][0][2 * j + 1]);
      else a = x[d % B][j];
      o[d] = mfma<C::PV>(a, ph[j], o[d]);
      o[d] = mfma<C::PV>(a, pl[j], o[d]);
      if constexpr (C::NT == 3) o[d] = mfma<C::PV>(a, pm[j], o[d]);
    }
  }
}

// The waves' results joined through LDS (in order), each wave with its share of the d
// tiles, and the result or its part written.
template <int DT, int HD>
__device__ __forceinline__ void finish(const PagedAttnParams& p, const Split& sp, const SeqSpan& sq, int s, int h, int part, bool whole, float m, float l,
                                       const f32x4 (&o)[HD / 16], unsigned char* smem) {
  constexpr int ND = HD / 16, NM = ND / kFewWaves;
  const int lane = threadIdx.x & 63, wave = scalar((int)(threadIdx.x >> 6)), g = lane >> 4;
  Column col;
  col.set(p, sq, h, lane & 15);
  f32x4* xo = reinterpret_cast<f32x4*>(smem);                                    // [wave][ND][64]
  float* xs = reinterpret_cast<float*>(smem + (size_t)kFewWaves * ND * 64 * 16);  // [wave][2][64]
#pragma unroll
  for (int d = 0; d < ND; ++d) xo[(wave * ND + d) * 64 + lane] = o[d];
  xs[wave * 128 + lane] = m;
  xs[wave * 128 + 64 + lane] = column_sum(l);
  __syncthreads();
  float mm = -INFINITY, al[kFewWaves], ll = 0.f;
#pragma unroll
  for (int a = 0; a < kFewWaves; ++a) {
    al[a] = xs[a * 128 + lane];
    mm = fmaxf(mm, al[a]);
  }
  const float mu = mm == -INFINITY ? 0.f : mm;
  f32x4 w[NM] = {};
#pragma unroll
  for (int a = 0; a < kFewWaves; ++a) {
    al[a] = __builtin_amdgcn_exp2f(al[a] - mu);
    ll += xs[a * 128 + 64 + lane] * al[a];
#pragma unroll
    for (int d = 0; d < NM; ++d) w[d] += xo[(a * ND + wave * NM + d) * 64 + lane] * al[a];
  }
  if (!col.on) return;
  if (whole) {
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;  // no key: zeros
    uint16_t* dst = p.out + col.tok * p.ldo + (int64_t)col.head * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < NM; ++d) {
      const f32x4 y = w[d] * inv;
      *reinterpret_cast<u32x2*>(dst + (wave * NM + d) * 16) = u32x2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
    }
  } else {
    const int64_t at = part_index(p, sp, true, s, h, lane & 15, col.tok, col.head, part);
    float* dst = p.ws + at * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < NM; ++d) *reinterpret_cast<f32x4*>(dst + (wave * NM + d) * 16) = w[d];
    if (wave == 0 && g == 0) *reinterpret_cast<f32x2*>(part_stats(p, sp, HD) + at * 2) = (f32x2){mm, ll};
  }
}

// Pages, and e4m3 scales, of 16 blocks: lane 4 j + a those of the 16 keys from
// key(j) + 16 a on.  holes: some page of the sequence's keys is none.
// page_ids() is the part that does not need the sequence's length, so that the first
// load can go out together with it.
template <class Key>
__device__ __forceinline__ int page_ids(const PagedParams& kv, int s, Key key) {
  const int lane = threadIdx.x & 63;
  return page_at(kv, s, key(lane >> 2) + 16 * (lane & 3));
}
template <bool F8, int HD, class Key>
__device__ __forceinline__ void fetch_pages(const PagedParams& kv, const SeqSpan& sq, int found, int h, int left, Key key, Pages* pages,
                                            float* ks, float* vs, bool* holes) {
  const int lane = threadIdx.x & 63, pos = key(lane >> 2) + 16 * (lane & 3);
  const bool in = (lane >> 2) < left && pos < sq.seen();
  const int id = in ? found : -1;
  *holes |= __builtin_amdgcn_ballot_w64(in && id < 0) != 0;
  const int64_t at = id < 0 ? -1 : page_base(kv, id, h, HD) * (F8 ? 1 : 2);
  *pages = {(int)at, (int)(at >> 32)};
  if constexpr (F8) {
    const int64_t sc = (int64_t)max(id, 0) * kv.nkvh + h;
    const float x = kv.k_scale[sc], y = kv.v_scale[sc];
    *ks = id < 0 ? 1.f : x;
    *vs = id < 0 ? 0.f : y;
  }
}

// What lane 4 j + g holds, for each lane's g, without a trip to the LDS.
__device__ __forceinline__ int of_keys(int v, int j, int g) {
  const int a = __builtin_amdgcn_readlane(v, 4 * j), b = __builtin_amdgcn_readlane(v, 4 * j + 1);
  const int c = __builtin_amdgcn_readlane(v, 4 * j + 2), d = __builtin_amdgcn_readlane(v, 4 * j + 3);
  return g & 2 ? (g & 1 ? d : c) : (g & 1 ? b : a);
}
__device__ __forceinline__ float of_keys(float v, int j, int g) {
  return __uint_as_float((uint32_t)of_keys((int)__float_as_uint(v), j, g));
}

// Lane l's value for the lanes' lower half, lane l + 1's for the upper.
__device__ __forceinline__ int of_half(int v, int l, int h) {
  const int a = __builtin_amdgcn_readlane(v, l), b = __builtin_amdgcn_readlane(v, l + 1);
  return h ? b : a;
}

// Sequences of few rows: every wave has its own tiles, and waits for its own loads
// alone.  K of the next block is under way while this one's softmax and P.V run, V
// from P.V to P.V.  Block: kv head fastest, then part, then sequence.
template <int DT, bool F8, int HD>
constexpr int few_lds() {
  constexpr int tiles = kFewWaves * 2 * Cfg<DT, F8, HD>::TILE, join = kFewWaves * 64 * (HD + 8);
  return tiles > join ? tiles : join;
}
template <int DT, bool F8, int HD, int LP>
__device__ __forceinline__ void few_block(const PagedAttnParams& p, const Split& sp, int block, unsigned char* smem) {
  using C = Cfg<DT, F8, HD>;
  const PagedParams& kv = p.kv;
  const int h = block % kv.nkvh;
  const int part = block / kv.nkvh % sp.few_chunks, s = block / kv.nkvh / sp.few_chunks;
  const int wave = scalar((int)(threadIdx.x >> 6)), k0 = part * sp.few_chunk;
  auto key_of = [&](int it) { return k0 + (wave + it * kFewWaves) * 64; };
  const int found = page_ids(kv, s, key_of);
  const SeqSpan sq = seq_span(kv, s);
  if (sq.n == 0 || sq.n * p.rep > kFewRows) return;
  const int end = sq.seen();
  const int k1 = min(k0 + sp.few_chunk, end);
  if (part > 0 && k0 >= end) return;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int nb = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0, steps = (nb - wave + kFewWaves - 1) / kFewWaves;
  unsigned char *kt = smem + wave * 2 * C::TILE, *vt = kt + C::TILE;
  constexpr int lcp = LP - (F8 ? 4 : 3);
  Pages pages = {-1, -1};
  float ksc = 1.f, vsc = 0.f;
  bool holes = false;
  auto fetch = [&](int it, int ids) {
    fetch_pages<F8, HD>(kv, sq, ids, h, steps - it, [&](int j) { return key_of(it + j); }, &pages, &ksc, &vsc, &holes);
  };
  Column col;
  col.set(p, sq, h, c);
  u32x4 q[C::QS];
  load_q<F8, HD>(p, col, g, q);
  if (steps > 0) {
    fetch(0, found);
    load_tile<DT, F8, HD, false, 1, LP, true>(kv, pages, 0, 0, kt);
    load_tile<DT, F8, HD, false, 1, LP, false>(kv, pages, 0, 0, vt);
  }
  keep(q);
  f32x4 o[C::ND] = {};
  float m = -INFINITY, l = 0.f;
  const int ka = k_frag<DT, F8, HD>(c, g);
  int va[C::VS];
#pragma unroll
  for (int e = 0; e < C::VS; ++e) va[e] = v_frag<DT, F8, HD>(c, g, e, lcp);
  for (int it = 0; it < steps; ++it) {
    const bool more = it + 1 < steps;
    const int kg = key_of(it) + 16 * g;
    int have = sq.seen() - kg;
    if (holes && of_keys(pages.hi, it & 15, g) < 0) have = 0;
    float ks = 1.f, vs = 0.f;
    if constexpr (F8) {
      ks = of_keys(ksc, it & 15, g);
      vs = of_keys(vsc, it & 15, g);
    }
    wait_vmcnt<C::LI>();  // K is there; V's loads came after it
    f32x4 sc[4];
    u32x4 ph[2], pl[2], pm[2];
    multiply_k<DT, F8, HD>(kt, ka, q, sc);
    wait_lds();
    if (more) {
      if ((it & 15) == 15) fetch(it + 1, page_ids(kv, s, [&](int j) { return key_of(it + 1 + j); }));
      load_tile<DT, F8, HD, false, 1, LP, true>(kv, pages, (it + 1) & 15, 0, kt);
    }
    softmax<DT, F8, HD>(sc, col.pos, kg, have, p.scale * kLog2e * ks, vs, m, l, o, ph, pl, pm);
    if (more) wait_vmcnt<C::LI>();  // V is there; the next K's loads came after it
    else wait_vmcnt<0>();
    if (__builtin_amdgcn_ballot_w64(have < 16)) clear_tail<DT, F8, HD>(vt, va, lcp, have);
    multiply_v<DT, F8, HD>(vt, va, lcp, ph, pl, pm, o);
    wait_lds();
    if (more) load_tile<DT, F8, HD, false, 1, LP, false>(kv, pages, (it + 1) & 15, 0, vt);
  }
  __syncthreads();  // the tiles' LDS is the join's
  finish<DT, HD>(p, sp, sq, s, h, part, end <= sp.few_chunk, m, l, o, smem);
}

template <int DT, bool F8, int HD, int LP>
__global__ void __launch_bounds__(64 * kFewWaves) paged_few_kernel(const PagedAttnParams p, const Split sp) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[few_lds<DT, F8, HD>()];
  few_block<DT, F8, HD, LP>(p, sp, (int)blockIdx.x, smem);
}

// ---- tiles of 64 or 128 (row, head) pairs ----
//
// NS key splits of GW waves with 32 columns each, on v_mfma_f32_32x32x16: lane
// (c = lane & 31, h = lane >> 5) gets rows 8 a + 4 h + b of each 32-key product (a, b
// < 4), which are given keys 16 h + 4 a + b, so that it has 16 keys of its column in a
// row, twice.  A split's waves share its tiles.  A step is an MFMA phase (P.V of
// the block before, S of this one) and a VALU phase (softmax, the next loads); every
// phase ends in a block barrier, and the upper half of the splits runs one phase
// behind the lower, so that of the two waves on a SIMD one multiplies while the
// other is at its softmax.
// Rows' parts of the chunk order here: f = (16-byte chunk number in the page / 16)
// modulo the row's chunks, for K and V alike; with the keys above the lanes that the
// LDS serves at once find 16 bank groups, whatever the page size.
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <int DT>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == QA_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// P.V of one block (PVT) and S of another (SQT).  HD / 16 slices: two 32-row d tiles of
// V against 16 keys of P, and 16 of d of both 32-key products; the fragments are
// read AHEAD slices before.  (The empty statements keep their addresses from being
// formed outside the loop and held there.)
template <int DT, bool F8, int HD, bool PVT, bool SQT>
__device__ __forceinline__ void multiply32(const unsigned char* vt, const int (&va)[F8 ? 2 : 4], int lcp, const u32x4 (&ph)[2][2],
                                           const u32x4 (&pl)[2][2], const u32x4 (&pm)[2][2], f32x16 (&o)[HD / 32], const unsigned char* kt, int ka,
                                           const u32x4 (&q)[HD / 16], f32x16 (&sc)[2]) {
  using C = Cfg<DT, F8, HD>;
  constexpr int N = HD / 16, DP = HD / 64;  // slices, pairs of d tiles
  constexpr int EACH = F8 ? 2 : 1;          // slices that one read serves
  constexpr int AHEAD = 1, B = AHEAD + 1;
  int at[F8 ? 2 : 4], ak = ka;
  asm volatile("" : "+v"(ak));
#pragma unroll
  for (int e = 0; e < (F8 ? 2 : 4); ++e) {
    at[e] = va[e];
    asm volatile("" : "+v"(at[e]));
  }
  u32x4 x[B][2], y[B][2];
  // slice n: keys' half kt = n / (2 DP), d tiles 2 ((n / 2) % DP) and the next, 16 keys' half j = n % 2
  auto read = [&](int i) {  // reads number i, for slices EACH i ..
    const int n = i * EACH;
    if constexpr (PVT) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        x[i % B][u] = *reinterpret_cast<const u32x4*>(vt + at[F8 ? n / (2 * DP) : n / (2 * DP) * 2 + n % 2] +
                                                      ((2 * (n / 2 % DP) + u) * 512 << lcp));
    }
    if constexpr (SQT) {
#pragma unroll
      for (int u = 0; u < 2; ++u) y[i % B][u] = *reinterpret_cast<const u32x4*>(kt + (ak ^ (i << 5)) + u * 32 * C::CR * 16);
    }
  };
#pragma unroll
  for (int i = 0; i < AHEAD && i < N / EACH; ++i) read(i);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = n / EACH, half = n / (2 * DP), d = 2 * (n / 2 % DP), j = n % 2;
    const bool reads = n % EACH == 0 && i + AHEAD < N / EACH;
    if (reads) read(i + AHEAD);
    u32x4 v[2];
    if constexpr (PVT) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (F8) v[u] = widen_e4m3<QA_BF16>(x[i % B][u][2 * j], x[i % B][u][2 * j + 1]);
        else v[u] = x[i % B][u];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) o[d + u] = mfma32<C::PV>(v[u], ph[half][j], o[d + u]);
    }
    if constexpr (SQT) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 a;
        if constexpr (F8) a = widen_e4m3<DT>(y[i % B][u][2 * j], y[i % B][u][2 * j + 1]);
        else a = y[i % B][u];
        sc[u] = mfma32<DT>(a, q[n], n ? sc[u] : f32x16{0});
      }
    }
    if constexpr (PVT) {
#pragma unroll
      for (int u = 0; u < 2; ++u) o[d + u] = mfma32<C::PV>(v[u], pl[half][j], o[d + u]);
      if constexpr (C::NL == 3) {
#pragma unroll
        for (int u = 0; u < 2; ++u) o[d + u] = mfma32<C::PV>(v[u], pm[half][j], o[d + u]);
      }
    }
    constexpr int R = (PVT ? 2 : 0) + (SQT ? 2 : 0);
    if (reads) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    __builtin_amdgcn_sched_barrier(0);  // no more fragments at once than the registers hold
  }
}

// softmax() for a lane with one column and keys kg + 16 h .., kg + 32 + 16 h .. (two
// runs of 16, a page each).
template <int DT, bool F8, int HD>
__device__ __forceinline__ void softmax32(f32x16 (&sc)[2], int pos, int kg, const int (&have)[2], const float (&f)[2],
                                          const float (&vs)[2], float& m, float& l, f32x16 (&o)[HD / 32],
                                          u32x4 (&ph)[2][2], u32x4 (&pl)[2][2], u32x4 (&pm)[2][2]) {
  using C = Cfg<DT, F8, HD>;
  float top[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int see = min(have[u], pos + 1 - kg - 32 * u);
    if (__builtin_amdgcn_ballot_w64(see < 16)) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e >= see) sc[u][e] = -INFINITY;
    }
    float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int t = 0; t < 4; ++t) max4(x[t & 1], sc[u][4 * t], sc[u][4 * t + 1], sc[u][4 * t + 2], sc[u][4 * t + 3]);
    top[u] = fmaxf(x[0], x[1]);
  }
  const float bm = pair_max(F8 ? fmaxf(top[0] * f[0], top[1] * f[1]) : fmaxf(top[0], top[1]) * f[0]);
  if (__builtin_amdgcn_ballot_w64(bm > m + kLazy)) {
    const float mn = fmaxf(m, bm);
    const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    l *= al;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) o[d] *= al;
    m = mn;
  }
  const float mb = (m == -INFINITY ? 0.f : m) - C::kBias;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][4 * t + e], f[u], -mb));
        sum[e] += w[e];
        if constexpr (F8) w[e] *= vs[u];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t hi = pack2<C::PV>(w[2 * e], w[2 * e + 1]), lo = residue2<C::PV>(hi, w[2 * e], w[2 * e + 1]);
        ph[u][t >> 1][2 * (t & 1) + e] = hi;
        pl[u][t >> 1][2 * (t & 1) + e] = lo;
        if constexpr (C::NL == 3) pm[u][t >> 1][2 * (t & 1) + e] = residue2(hi, lo, w[2 * e], w[2 * e + 1]);
      }
    }
  l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
template <int DT, bool F8, int HD, int GW>
constexpr int many_buffers() {  // buffers of each tile: two where 128 KB hold them
  return kManyWaves / GW * 2 * Cfg<DT, F8, HD>::TILE * 2 <= 131072 ? 2 : 1;
}
template <int DT, bool F8, int HD, int GW>
constexpr int many_lds() {
  constexpr int tiles = kManyWaves / GW * 2 * Cfg<DT, F8, HD>::TILE * many_buffers<DT, F8, HD, GW>();
  constexpr int join = kManyWaves * 64 * 4 * (HD / 2 + 2), few = few_lds<DT, F8, HD>();
  return tiles > join ? (tiles > few ? tiles : few) : (join > few ? join : few);
}
// Tile number u of all the sequences' tiles of TR pairs, one sequence after the
// other, in each the last first (it sees the most keys): every wave adds up the
// sequences' tiles, 64 sequences at a time.
template <int TR>
__device__ __forceinline__ bool find_tile(const PagedAttnParams& p, const Split& sp, int u, int* seq, SeqSpan* sq, int* tile) {
  const PagedParams& kv = p.kv;
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < kv.seqs; s0 += 64) {
    int mine = 0;
    SeqSpan q = {};
    if (s0 + lane < kv.seqs) {
      q = seq_span(kv, s0 + lane);
      const int NR = q.n * p.rep;
      mine = sp.few && NR <= kFewRows ? 0 : (NR + TR - 1) / TR;
    }
    int upto = mine;
#pragma unroll
    for (int e = 1; e < 64; e <<= 1) {
      const int x = __shfl_up(upto, e, 64);
      upto += lane >= e ? x : 0;
    }
    const uint64_t after = __builtin_amdgcn_ballot_w64(upto > u);
    if (after) {
      const int at = __builtin_ctzll(after);
      *seq = scalar(s0 + at);
      *tile = __builtin_amdgcn_readlane(upto, at) - 1 - u;
      sq->row0 = __builtin_amdgcn_readlane((int)q.row0, at);
      sq->n = __builtin_amdgcn_readlane(q.n, at);
      sq->pos0 = __builtin_amdgcn_readlane(q.pos0, at);
      return true;
    }
    u -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}
template <int DT, bool F8, int HD, int LP, int GW>
__global__ void __launch_bounds__(64 * kManyWaves, 2) paged_many_kernel(const PagedAttnParams p, const Split sp) {
  using C = Cfg<DT, F8, HD>;
  constexpr int NS = kManyWaves / GW, NB = many_buffers<DT, F8, HD, GW>(), WL = C::LI / GW;  // WL: a wave's loads of a tile
  constexpr int TR = GW * 32, VX = F8 ? 2 : 4;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[many_lds<DT, F8, HD, GW>()];
  const PagedParams& kv = p.kv;
  const int mine = (int)blockIdx.x - sp.tiles * sp.many_chunks * kv.nkvh;
  if (mine >= 0) {  // behind them, the blocks of the sequences of few rows, four waves each
    // (the other waves end here, and a barrier waits for no wave that has ended)
    if (threadIdx.x < 64 * kFewWaves) few_block<DT, F8, HD, LP>(p, sp, mine, smem);
    return;
  }
  const int kvh = (int)(blockIdx.x % kv.nkvh);
  const int part = blockIdx.x / kv.nkvh / sp.tiles;
  int tile, s;
  SeqSpan sq;
  if (!find_tile<TR>(p, sp, blockIdx.x / kv.nkvh % sp.tiles, &s, &sq, &tile)) return;
  const int NR = sq.n * p.rep;
  const int end = sq.pos0 + (min((tile + 1) * TR, NR) - 1) / p.rep + 1;
  const int k0 = part * sp.many_chunk, k1 = min(k0 + sp.many_chunk, end);
  if (part > 0 && k0 >= end) return;
  // (the wave's number is left to the compiler as a lane's value: with scalar
  // control flow it spills; what a DMA instruction takes is made scalar below)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int ns = wave / GW, wg = wave % GW, off = ns / (NS / 2);
  const int nb = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0, steps = (nb - ns + NS - 1) / NS;
  auto key_of = [&](int it) { return k0 + (ns + it * NS) * 64; };
  unsigned char* base = smem + ns * 2 * NB * C::TILE;
  auto kt = [&](int it) { return base + (it & (NB - 1)) * C::TILE; };
  auto vt = [&](int it) { return base + (NB + (it & (NB - 1))) * C::TILE; };
  constexpr int lcp = LP - (F8 ? 4 : 3), cp = 1 << lcp;
  // two windows of 16 blocks' pages: loads run up to two blocks ahead of the softmax
  bool holes = false;
  Pages pages0 = {-1, -1}, pages1 = {-1, -1};
  float ks0 = 1.f, ks1 = 1.f, vs0 = 0.f, vs1 = 0.f;
  auto fetch = [&](int w) {
    Pages pg = {-1, -1};
    float x = 1.f, y = 0.f;
    auto key = [&](int j) { return key_of(16 * w + j); };
    fetch_pages<F8, HD>(kv, sq, page_ids(kv, s, key), kvh, steps - 16 * w, key, &pg, &x, &y, &holes);
    pages0.lo = w & 1 ? pages0.lo : pg.lo;
    pages0.hi = w & 1 ? pages0.hi : pg.hi;
    ks0 = w & 1 ? ks0 : x;
    vs0 = w & 1 ? vs0 : y;
    pages1.lo = w & 1 ? pg.lo : pages1.lo;
    pages1.hi = w & 1 ? pg.hi : pages1.hi;
    ks1 = w & 1 ? x : ks1;
    vs1 = w & 1 ? y : vs1;
  };
  auto pages_of = [&](int it) { return it >> 4 & 1 ? pages1 : pages0; };
  auto issue_k = [&](int it) {
    load_tile<DT, F8, HD, true, GW, LP, true>(kv, pages_of(it), scalar(it & 15), scalar(wg), smem + scalar((int)(kt(it) - smem)));
  };
  auto issue_v = [&](int it) {
    load_tile<DT, F8, HD, true, GW, LP, false>(kv, pages_of(it), scalar(it & 15), scalar(wg), smem + scalar((int)(vt(it) - smem)));
  };
  // refill(j), in step j's VALU phase: K of block j + NB (S of j has read its slot),
  // V of block j + NB - 1 (P.V of j - 1 has).  Step i's MFMA phase needs K(i) and
  // V(i - 1), of refill(i - NB): with two buffers refill(i - 1) may be under way.
  auto ahead = [&](int j) { return NB == 1 ? 0 : (j + 2 < steps) + (j + 1 < steps); };
  auto wait_ahead = [&](int j) {
    const int n = ahead(j);
    if (n == 2) wait_vmcnt<2 * WL>();
    else if (n == 1) wait_vmcnt<WL>();
    else wait_vmcnt<0>();
  };
  // the lane's (row, head) pair; lanes past the last repeat it and store nothing
  auto pair_of = [&](int64_t* tok, int* head) {
    int R = (tile * GW + wg) * 32 + c;
    asm volatile("" : "+v"(R));  // formed again for the result, not held across the loop
    const bool on = R < NR;
    R = min(R, NR - 1);
    const int i = R / p.rep;
    *tok = sq.row0 + i;
    *head = kvh * p.rep + R - i * p.rep;
    return on;
  };
  u32x4 q[HD / 16];
  int pos;
  {
    int64_t tok;
    int head;
    pair_of(&tok, &head);
    pos = (int)(tok - sq.row0) + sq.pos0;
    const uint16_t* src = p.q + tok * p.ldq + (int64_t)head * HD;
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)  // in the order in which a K row's chunks come
      q[e] = *reinterpret_cast<const u32x4*>(src + (F8 ? e / 2 * 32 + h * 16 + e % 2 * 8 : e * 16 + h * 8));
  }
  if (steps > 0) {
    fetch(0);
    if (steps > 16) fetch(1);
    issue_k(0);
    if (NB == 2 && steps > 1) issue_k(1);
    if (NB == 2) issue_v(0);
  }
  keep(q);
  f32x16 o[HD / 32] = {};
  float m = -INFINITY, l = 0.f;
  f32x16 sc[2];
  u32x4 ph[2][2], pl[2][2], pm[2][2];
  // fragment addresses: K row of the lane's key in a 32-key product, slice e at ^ (e << 5);
  // V row c, the chunks of the lane's keys
  const int key = 16 * (c >> 2 & 1) + 4 * (c >> 3) + (c & 3);
  const int ka = (key * C::CR + (h ^ (key >> (4 - C::LCR) & (C::CR - 1)))) * 16;
  int va[VX];
#pragma unroll
  for (int e = 0; e < VX; ++e) {
    const int x = F8 ? 2 * e + h : 4 * (e >> 1) + 2 * h + (e & 1);  // the block's chunk of the row
    va[e] = ((((x >> lcp) * HD + c) << lcp) + ((x & (cp - 1)) ^ (c >> (4 - lcp) & (cp - 1)))) * 16;
  }
  int have[2] = {16, 16};  // the lane's keys in the block of the last softmax
  const int n0 = (nb + NS - 1) / NS, n1 = (nb + NS / 2 - 1) / NS;  // most steps of either half
  const int phases = max(2 * n0 + 1, 2 * n1 + 2);
  if (off == 0) wait_vmcnt<0>();
  phase_barrier();
  for (int ph_no = 0; ph_no < phases; ++ph_no) {
    const int my = ph_no - off, it = my >> 1;
    if (my >= 0 && my <= 2 * steps) {
      if ((my & 1) == 0) {
        if (it > 0 && __builtin_amdgcn_ballot_w64(min(have[0], have[1]) < 16)) {
          // V behind the keys that rows see, or for no page, may be anything, NaN too: a
          // lane clears those elements of the chunks that it will read itself
#pragma unroll
          for (int e = 0; e < VX; ++e)
#pragma unroll 1
            for (int d = 0; d < HD / 32; ++d) {
              u32x4* x = reinterpret_cast<u32x4*>(vt(it - 1) + va[e] + (d * 512 << lcp));
              const int left = F8 ? have[e] : have[e >> 1] - 8 * (e & 1);
              *x &= u32x4{tail_mask<C::ES>(left, 0), tail_mask<C::ES>(left, 1), tail_mask<C::ES>(left, 2), tail_mask<C::ES>(left, 3)};
            }
        }
        if (it > 0 && it < steps) multiply32<DT, F8, HD, true, true>(vt(it - 1), va, lcp, ph, pl, pm, o, kt(it), ka, q, sc);
        else if (it > 0) multiply32<DT, F8, HD, true, false>(vt(it - 1), va, lcp, ph, pl, pm, o, kt(it), ka, q, sc);
        else if (steps > 0) multiply32<DT, F8, HD, false, true>(vt(it), va, lcp, ph, pl, pm, o, kt(it), ka, q, sc);
      } else {
        const int kg = key_of(it) + 16 * h, j = scalar(it & 15);
        float f[2], vs[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          have[u] = sq.seen() - kg - 32 * u;
          if (holes && of_half(pages_of(it).hi, 4 * j + 2 * u, h) < 0) have[u] = 0;
          f[u] = p.scale * kLog2e;
          if constexpr (F8) {
            f[u] *= __int_as_float(of_half(__float_as_int(it >> 4 & 1 ? ks1 : ks0), 4 * j + 2 * u, h));
            vs[u] = __int_as_float(of_half(__float_as_int(it >> 4 & 1 ? vs1 : vs0), 4 * j + 2 * u, h));
          }
        }
        if (it > 0 && (it & 15) == 0 && 16 * (it >> 4) + 16 < steps) fetch((it >> 4) + 1);
        if (it + NB < steps) issue_k(it + NB);
        if (it + NB - 1 < steps) issue_v(it + NB - 1);
        softmax32<DT, F8, HD>(sc, pos, kg, have, f, vs, m, l, o, ph, pl, pm);
      }
    }
    const int next = ph_no + 1 - off;
    if (next >= 0 && (next & 1) == 0 && (next >> 1) <= steps) wait_ahead((next >> 1) - 1);
    wait_lds();
    phase_barrier();
  }

  // the splits joined through LDS (in order), each with 1 / NS of the four-element
  // pieces, and the result or its part written
  constexpr int PC = HD / 8, NM = PC / NS;  // pieces of a lane: d = 32 (i / 4) + 8 (i % 4) + 4 h ..
  f32x4* xo = reinterpret_cast<f32x4*>(smem);                                     // [wave][PC][64]
  float* xs = reinterpret_cast<float*>(smem + (size_t)kManyWaves * PC * 64 * 16);  // [wave][2][64]
#pragma unroll
  for (int i = 0; i < PC; ++i) {
    const f32x16& a = o[i / 4];
    const int e = 4 * (i % 4);
    xo[(wave * PC + i) * 64 + lane] = f32x4{a[e], a[e + 1], a[e + 2], a[e + 3]};
  }
  xs[wave * 128 + lane] = m;
  xs[wave * 128 + 64 + lane] = pair_sum(l);
  __syncthreads();
  float mm = -INFINITY, al[NS], ll = 0.f;
#pragma unroll
  for (int a = 0; a < NS; ++a) {
    al[a] = xs[(a * GW + wg) * 128 + lane];
    mm = fmaxf(mm, al[a]);
  }
  const float mu = mm == -INFINITY ? 0.f : mm;
  f32x4 w[NM] = {};
#pragma unroll
  for (int a = 0; a < NS; ++a) {
    al[a] = __builtin_amdgcn_exp2f(al[a] - mu);
    ll += xs[(a * GW + wg) * 128 + 64 + lane] * al[a];
#pragma unroll
    for (int i = 0; i < NM; ++i) w[i] += xo[((a * GW + wg) * PC + ns * NM + i) * 64 + lane] * al[a];
  }
  int64_t tok;
  int head;
  if (!pair_of(&tok, &head)) return;
  auto d_of = [&](int i) { return 32 * ((ns * NM + i) >> 2) + 8 * ((ns * NM + i) & 3) + 4 * h; };
  if (end <= sp.many_chunk) {
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;  // no key: zeros
    uint16_t* dst = p.out + tok * p.ldo + (int64_t)head * HD;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const f32x4 y = w[i] * inv;
      *reinterpret_cast<u32x2*>(dst + d_of(i)) = u32x2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
    }
  } else {
    const int64_t at = part_index(p, sp, false, s, kvh, 0, tok, head, part);
#pragma unroll
    for (int i = 0; i < NM; ++i) *reinterpret_cast<f32x4*>(p.ws + at * HD + d_of(i)) = w[i];
    if (ns == 0 && h == 0) *reinterpret_cast<f32x2*>(part_stats(p, sp, HD) + at * 2) = (f32x2){mm, ll};
  }
}

// The parts of (row, head) pairs joined, HD / 4 threads to a part, four parts in
// flight for each thread.  A short sequence's pair may have many parts: a block
// takes one, 8 (hd 128) or 16 (hd 64) parts at once, whose sums meet in LDS.  A long
// sequence's have few: a block takes 8 or 16 pairs of a tile, one part after the
// other.  The grid: the tiles' blocks, as in paged_many_kernel, then the short
// sequences' pairs; of either as many as had to be split.
template <int HD>
constexpr int kJoinPairs = 1024 / HD;
template <int DT, int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttnParams p, const Split sp, int groups) {
  constexpr int TP = HD / 4, NP = kJoinPairs<HD>;
  __shared__ f32x4 xo[NP][TP];
  __shared__ float xs[NP];
  const int h = (int)(blockIdx.x % p.kv.nkvh), b = (int)(blockIdx.x / p.kv.nkvh), mine = b - groups;
  const int lane = threadIdx.x & 63, pt = threadIdx.x / TP, d = threadIdx.x % TP;
  const bool few = mine >= 0;
  SeqSpan sq;
  int R, s;
  if (few) {
    s = mine / sp.few_pairs;
    sq = seq_span(p.kv, s);
    R = mine % sp.few_pairs;
    if (sq.n * p.rep > kFewRows) return;
  } else {
    const int per = sp.many_rows / NP;  // blocks of a tile
    int tile;
    if (!(sp.many_rows == 64 ? find_tile<64>(p, sp, b / per, &s, &sq, &tile) : find_tile<128>(p, sp, b / per, &s, &sq, &tile))) return;
    R = tile * sp.many_rows + b % per * NP + pt;
  }
  const int NR = sq.n * p.rep;
  if (R >= NR) return;  // (few: the block as one)
  const int chunk = few ? sp.few_chunk : sp.many_chunk;
  const int last = few ? NR - 1 : min((R / sp.many_rows + 1) * sp.many_rows, NR) - 1;
  const int keys = sq.pos0 + last / p.rep + 1;
  if (keys <= chunk) return;  // its tile has written the result
  const int parts = (keys + chunk - 1) / chunk;
  const int i = R / p.rep, head = h * p.rep + R % p.rep;
  const int64_t t = sq.row0 + i, at = part_index(p, sp, few, s, h, R, t, head, 0);
  const float* st = part_stats(p, sp, HD) + at * 2;
  const float* src = p.ws + at * HD + d * 4;
  float mm = -INFINITY;
  if (few) {
    for (int a = lane; a < parts; a += 64) mm = fmaxf(mm, st[2 * a]);
#pragma unroll
    for (int e = 32; e > 0; e >>= 1) mm = fmaxf(mm, __shfl_xor(mm, e, 64));
  } else {
    for (int a = 0; a < parts; ++a) mm = fmaxf(mm, st[2 * a]);
  }
  const float mu = mm == -INFINITY ? 0.f : mm;
  const int first = few ? pt : 0, step = few ? NP : 1;
  float ll = 0.f;
  f32x4 y = {0, 0, 0, 0};
  for (int a0 = first; a0 < parts; a0 += 4 * step) {
    f32x4 v[4];
    f32x2 ml[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int a = min(a0 + e * step, parts - 1);
      v[e] = *reinterpret_cast<const f32x4*>(src + (int64_t)a * HD);
      ml[e] = *reinterpret_cast<const f32x2*>(st + 2 * a);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float al = a0 + e * step < parts ? __builtin_amdgcn_exp2f(ml[e][0] - mu) : 0.f;
      ll += ml[e][1] * al;
      y += v[e] * al;
    }
  }
  if (few) {
    xo[pt][d] = y;
    if (d == 0) xs[pt] = ll;
    __syncthreads();
    if (pt > 0) return;
    for (int e = 1; e < NP; ++e) {
      y += xo[e][d];
      ll += xs[e];
    }
  }
  y *= ll == 0.f ? 0.f : 1.0f / ll;
  *reinterpret_cast<u32x2*>(p.out + t * p.ldo + (int64_t)head * HD + d * 4) = u32x2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
}

template <int DT, bool F8, int HD, int LP>
hipError_t launch_one(const PagedAttnParams& p, hipStream_t s) {
  const Split sp = split_of(p, F8, HD);
  const int64_t heads = (int64_t)p.kv.seqs * p.kv.nkvh;
  if (sp.many) {
    const dim3 grid((unsigned)((int64_t)p.kv.nkvh * sp.tiles * sp.many_chunks + (sp.few ? heads * sp.few_chunks : 0)));
    const dim3 block(64 * kManyWaves);
    if (sp.many_rows == 64) hipLaunchKernelGGL((paged_many_kernel<DT, F8, HD, LP, 2>), grid, block, 0, s, p, sp);
    else hipLaunchKernelGGL((paged_many_kernel<DT, F8, HD, LP, 4>), grid, block, 0, s, p, sp);
  } else {
    hipLaunchKernelGGL((paged_few_kernel<DT, F8, HD, LP>), dim3((unsigned)(heads * sp.few_chunks)), dim3(64 * kFewWaves), 0, s, p, sp);
  }
  if (sp.few_parts + sp.many_parts > 0) {
    const int64_t groups = sp.many_chunks == 1 ? 0 : (int64_t)sp.tiles * (sp.many_rows * HD / 1024);  // the tiles' blocks, for a kv head
    const int64_t pairs = sp.few_chunks == 1 ? 0 : heads * sp.few_pairs;
    hipLaunchKernelGGL((paged_join_kernel<DT, HD>), dim3((unsigned)(p.kv.nkvh * groups + pairs)), dim3(256), 0, s, p, sp, (int)groups);
  }
  return hipGetLastError();
}

template <int DT, bool F8, int HD>
hipError_t launch_lp(const PagedAttnParams& p, hipStream_t s) {
  return p.kv.lp == 4 ? launch_one<DT, F8, HD, 4>(p, s) : p.kv.lp == 5 ? launch_one<DT, F8, HD, 5>(p, s) : launch_one<DT, F8, HD, 6>(p, s);
}

template <int DT>
hipError_t launch_dt(bool e4m3, int hd, const PagedAttnParams& p, hipStream_t s) {
  if (hd == 64) return e4m3 ? launch_lp<DT, true, 64>(p, s) : launch_lp<DT, false, 64>(p, s);
  return e4m3 ? launch_lp<DT, true, 128>(p, s) : launch_lp<DT, false, 128>(p, s);
}

}  // namespace

int64_t paged_attention_blocks(bool e4m3, int hd, const PagedAttnParams& p) {
  const Split sp = split_of(p, e4m3, hd);
  // in doubles, as no product of these sizes need fit 64 bits; the caller compares with a bound far below
  const double heads = (double)p.kv.seqs * p.kv.nkvh, tiles = (double)p.kv.nkvh * sp.tiles;
  const double most = fmax(heads * kFewRows + tiles * 16, heads * sp.few_chunks + tiles * sp.many_chunks);
  return most > 9e18 ? INT64_MAX : (int64_t)most;
}

size_t paged_attention_workspace(bool e4m3, int hd, const PagedAttnParams& p) {
  const Split sp = split_of(p, e4m3, hd);
  return (size_t)(sp.few_parts + sp.many_parts) * (hd + 2) * sizeof(float);
}

hipError_t launch_attention_paged(int dtype, bool e4m3, int hd, const PagedAttnParams& p, hipStream_t s) {
  return dtype == QA_BF16 ? launch_dt<QA_BF16>(e4m3, hd, p, s) : launch_dt<QA_F16>(e4m3, hd, p, s);
}

}  // namespace qa

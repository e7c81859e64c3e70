// qa_rope_rows.hip -- cos / sin rows for tokens whose positions have one to three
// axes (text; height and width; time, height and width).
//
// Frequency j of hd / 2 turns by pos[a(j)][t] theta^(-2j / hd): each frequency
// follows one axis, in blocks (the first sec0 frequencies axis 0, the next sec1
// axis 1, ...) or interleaved (j mod axes, while that axis has frequencies left,
// else axis 0).  The rows are those of qa_rope_tables wherever all axes are
// equal, made on the device because positions of images and video are not a
// running number: once for a step, for every layer's q / k rotation.
//
// Bound by the rows it writes: 30720 tokens of hd 128, 31 MB, 8.5 us, of which the
// f64 of angles and series is 1; 32 tokens 4.8 us, the launch.  (With the library's
// sincos, whose reduction takes any angle, 1 more.)
//
// The angle is formed in f64 (a position of 2^20 leaves an f32 angle no more
// than 4 bits of a turn's fraction), as are its cosine and sine: |angle| < 2^31
// since theta >= 1, which lets two products of a quarter turn's halves reduce it
// without loss.
#include "qa_internal.h"

namespace qa {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// f64 to f32, then f32 to the 16-bit format.  The empty statement keeps the
// compiler from rounding the f64 value to f16 in one step, which differs where
// the f32 value is a midpoint of two f16 values.
template <int DT>
__device__ __forceinline__ float round16(double x) {
  float v = (float)x;
  asm("" : "+v"(v));
  if constexpr (DT == QA_F16) return (float)(_Float16)v;
  const uint32_t u = __float_as_uint(v);
  return __uint_as_float((u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u);
}

// cos and sin of |x| < 2^31.  n quarter turns are taken off as n (H + L), H the f64
// nearest to pi / 2: x - n H is a multiple of 2^-53 below 1 and so exact, and what L
// leaves out is below 2^31 2^-107.  The remainder, within pi / 4, goes into the
// Taylor series, cut where the next term is below 2^-54 (x^17 / 17! = 5e-17,
// x^18 / 18! = 2e-18).
__device__ __forceinline__ void cos_sin(double x, double* c, double* s) {
  const double n = rint(x * 0x1.45f306dc9c883p-1);  // 2 / pi
  const double r = fma(-n, 0x1.1a62633145c07p-54, fma(-n, 0x1.921fb54442d18p+0, x)), z = r * r;
  double a = -1.0 / 1307674368000.0, b = 1.0 / 20922789888000.0;  // 15!, 16!
  constexpr double kS[6] = {1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0, -1.0 / 5040.0, 1.0 / 120.0, -1.0 / 6.0};
  constexpr double kC[7] = {-1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0, 1.0 / 40320.0, -1.0 / 720.0, 1.0 / 24.0, -0.5};
#pragma unroll
  for (int i = 0; i < 6; ++i) a = fma(a, z, kS[i]);
#pragma unroll
  for (int i = 0; i < 7; ++i) b = fma(b, z, kC[i]);
  a = fma(a * z, r, r);
  b = fma(b, z, 1.0);
  const int q = (int)n;  // < 2^31
  *c = q & 1 ? a : b;
  *s = q & 1 ? b : a;
  if ((q + 1) & 2) *c = -*c;
  if (q & 2) *s = -*s;
}

// A thread: four frequencies of one token.
template <int DT>
__global__ void __launch_bounds__(256) mrope_rows_kernel(const MropeParams p) {
  const uint32_t half = (uint32_t)p.hd >> 1, quads = half >> 2, rows = 256 / quads;  // tokens to a block
  const uint32_t row = threadIdx.x / quads, j0 = (threadIdx.x - row * quads) * 4;
  const int64_t t = (int64_t)blockIdx.x * rows + row;
  if (row >= rows || t >= p.tokens) return;
  f32x4 c, s;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double a = (double)p.pos[p.axis[j0 + e] * p.ldpos + t] * p.inv[j0 + e];
    double sd, cd;
    cos_sin(a, &cd, &sd);
    c[e] = round16<DT>(cd);
    s[e] = round16<DT>(sd);
  }
  // past the caches, which a long batch's rows would only go through (9.6 us before); an
  // append behind this call takes as long either way, for few rows too
  float* co = p.cos + t * p.hd + j0;
  float* so = p.sin + t * p.hd + j0;
  __builtin_nontemporal_store(c, reinterpret_cast<f32x4*>(co));
  __builtin_nontemporal_store(c, reinterpret_cast<f32x4*>(co + half));
  __builtin_nontemporal_store(s, reinterpret_cast<f32x4*>(so));
  __builtin_nontemporal_store(s, reinterpret_cast<f32x4*>(so + half));
}

}  // namespace

hipError_t launch_mrope_rows(int dtype, const MropeParams& p, hipStream_t s) {
  const int rows = 256 / (p.hd >> 3);
  const dim3 grid((unsigned)((p.tokens + rows - 1) / rows));
  if (dtype == QA_BF16) hipLaunchKernelGGL(mrope_rows_kernel<QA_BF16>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(mrope_rows_kernel<QA_F16>, grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace qa

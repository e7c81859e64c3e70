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
// The angle is formed in f64 (a position of 2^20 leaves an f32 angle no more
// than 4 bits of a turn's fraction), as are its cosine and sine.
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

// A thread: four frequencies of one token.
template <int DT>
__global__ void __launch_bounds__(256) mrope_rows_kernel(const MropeParams p) {
  const int half = p.hd >> 1, quads = half >> 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / quads;
  if (t >= p.tokens) return;
  const int j0 = (int)(i - t * quads) * 4;
  f32x4 c, s;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double a = (double)p.pos[p.axis[j0 + e] * p.ldpos + t] * p.inv[j0 + e];
    double sd, cd;
    sincos(a, &sd, &cd);
    c[e] = round16<DT>(cd);
    s[e] = round16<DT>(sd);
  }
  float* co = p.cos + t * p.hd + j0;
  float* so = p.sin + t * p.hd + j0;
  *reinterpret_cast<f32x4*>(co) = c;
  *reinterpret_cast<f32x4*>(co + half) = c;
  *reinterpret_cast<f32x4*>(so) = s;
  *reinterpret_cast<f32x4*>(so + half) = s;
}

}  // namespace

hipError_t launch_mrope_rows(int dtype, const MropeParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.tokens * (p.hd >> 3) + 255) / 256));
  if (dtype == QA_BF16) hipLaunchKernelGGL(mrope_rows_kernel<QA_BF16>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(mrope_rows_kernel<QA_F16>, grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace qa

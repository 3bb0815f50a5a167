// A block of values becomes 4-bit codes and a scale: what the quantisation kernel and the products that quantise
// their activations themselves have in common.
//
// Mathematics.  A block (32 values in the MX form, 16 in the NV form) has one scale s, a code is
// RNE(x / s) onto {0, .5, 1, 1.5, 2, 3, 4, 6}.
//   MX: s = 2^e with e + 127 = max(exponent field of the largest |x| - 2, 0): x / s is exact.
//   NV: s = 2^exponent * E4M3(largest |x| / (6 * 2^exponent)).  Both roundings have to be those of the exact
//       quotient.  A quotient of 24 bits by s (4 significant bits) that is not on a border between codes (3
//       bits) lies more than half of its last place away from it, and so does one by 6 from a border of
//       E4M3 (5 bits): rounded to 24 bits it stays on its side, and on the border it stays there, if only
//       the error before that rounding is small.  So the quotient is x r + x r', r an approximate reciprocal
//       and r' = r (1 - r s) its Newton correction: two operations a value (checked for every 24-bit x,
//       every s and border).
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/tetris_b200.h"

namespace tetris {

// codes of 8 values, the first in the lowest 4 bits (RNE, at most 6)
__device__ __forceinline__ uint32_t codes_of(const float *v) {
  uint32_t r;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ uint8_t e4m3_of(float v) {  // RNE, at most 448
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return (uint8_t)r;
}
__device__ __forceinline__ float e4m3_value(uint8_t b) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)b));
  return __half2float(__ushort_as_half((unsigned short)(r & 0xFFFF)));
}

// The values of a thread's part of a block become quotients by the block's scale; returns the scale's byte.
template <int FMT, int N>
__device__ __forceinline__ uint8_t scale_block(float (&v)[N], float top, float tensor_scale, float sixth, float sixth_rest) {
  if (!(top < __int_as_float(0x7F800000))) {  // codes of 1: the block is NaN whatever it meets
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 1.f;
    return FMT == TETRIS_FP4_NV ? 0x7F : 0xFF;
  }
  if (FMT == TETRIS_FP4_MX) {
    const int byte = max((int)(__float_as_uint(top) >> 23) - 2, 0);  // at most 252
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= inv;
    return (uint8_t)byte;
  }
  const float within = fminf(top, 4096.f * tensor_scale);  // (beyond 2688 the scale stays at its largest)
  const uint8_t byte = e4m3_of(__fmaf_rn(within, sixth, within * sixth_rest));
  const float s = e4m3_value(byte) * tensor_scale;
  if (top > 1e3f * s && s > 0.f) {  // far above what the exponent holds: x / s could leave FP32
    const float most = 1e3f * s;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fminf(fmaxf(v[i], -most), most);
  }
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  if (s == 0.f) r = 0.f;
  const float rest = __fmaf_rn(-r, s, 1.f) * r;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __fmaf_rn(v[i], r, v[i] * rest);
  return byte;
}

}  // namespace tetris

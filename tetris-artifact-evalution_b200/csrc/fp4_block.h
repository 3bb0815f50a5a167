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
//       and r' = r (1 - r s) its Newton correction: two operations a value.  It grows with x, so the
//       borders and one last place beside them decide for every x: tests take all of them, under every s,
//       in exact arithmetic for any r within two last places and on the device.
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

// A block's scale, from its largest |x|.
struct BlockScale {
  uint8_t byte;
  bool bad;                // an infinity or a NaN is in it: codes of 1, the block is NaN whatever it meets
  bool far;                // far above what the exponent holds: x / s could leave FP32, the values are brought near first
  float r, rest, most;     // x / s = x r + x rest; `far`: the largest |x| that makes a difference
};
template <int FMT> __device__ __forceinline__ BlockScale block_scale(float top, float tensor_scale, float sixth, float sixth_rest) {
  BlockScale b;
  b.bad = !(top < __int_as_float(0x7F800000));
  b.far = false;
  b.rest = b.most = 0.f;
  if (FMT == TETRIS_FP4_MX) {
    const int byte = max((int)(__float_as_uint(top) >> 23) - 2, 0);  // at most 252
    b.r = __uint_as_float((uint32_t)(254 - byte) << 23);
    b.byte = b.bad ? 0xFF : (uint8_t)byte;
    return b;
  }
  const float within = fminf(top, 4096.f * tensor_scale);  // (beyond 2688 the scale stays at its largest)
  b.byte = e4m3_of(__fmaf_rn(within, sixth, within * sixth_rest));
  const float s = e4m3_value(b.byte) * tensor_scale;
  b.most = 1e3f * s;
  b.far = top > b.most && s > 0.f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b.r) : "f"(s));
  if (s == 0.f) b.r = 0.f;
  b.rest = __fmaf_rn(-b.r, s, 1.f) * b.r;
  if (b.bad) b.byte = 0x7F;
  return b;
}

// Codes of 8 values of a block.
template <int FMT> __device__ __forceinline__ uint32_t block_codes(const float *v, const BlockScale &b) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = FMT == TETRIS_FP4_NV ? __fmaf_rn(v[i], b.r, v[i] * b.rest) : v[i] * b.r;
  const uint32_t c = codes_of(q);
  return b.bad ? 0x22222222u : c;
}
template <int N> __device__ __forceinline__ void bring_near(float (&v)[N], const BlockScale &b) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = fminf(fmaxf(v[i], -b.most), b.most);
}

}  // namespace tetris

// Internal declarations of the 4-bit operators: the filter handle and what fp4_api.cu, fp4_quantize.cu
// and fp4_product.cu share.  The formats and their storage are described in the public header.
#pragma once
#include <cuda.h>
#include <math.h>

#include <atomic>

#include "internal.h"

struct tetris_fp4_filter {
  int in_channel, out_channel;
  int format, exponent;
  int device, sm_count;
  int64_t pitch, code_bytes, scale_bytes;
  int64_t direct_rows;     // a product of up to so many rows quantises them itself
  uint8_t *d_codes, *d_scales;
  int *d_error;            // raised by a product that gave up on a barrier wait
  // geometries of the last numbers of rows (fp4_product.cu): the number in the upper 40 bits, 0: none yet
  mutable std::atomic<uint64_t> plans[8];
};

namespace tetris {

// Division of 0 <= n < 2^31 by a launch constant: q = (umulhi(n, mul) + n) >> shift with
// shift = ceil(log2 d) and mul = floor(2^32 (2^shift - d) / d) + 1.
struct Fp4Div {
  uint32_t d, mul, shift;
};
inline Fp4Div fp4_div(uint32_t d) {
  Fp4Div f;
  f.d = d; f.shift = 0;
  while ((1ull << f.shift) < d) ++f.shift;
  f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
  return f;
}
__device__ __forceinline__ uint32_t fp4_quot(uint32_t n, const Fp4Div &f) { return (uint32_t)(((uint64_t)__umulhi(n, f.mul) + n) >> f.shift); }

constexpr int fp4_block(int format) { return format == TETRIS_FP4_NV ? 16 : 32; }
inline int64_t fp4_pitch(int cols) { return ((int64_t)cols + 31) / 32 * 16; }
inline int fp4_tiles(int cols, int format) { return (int)(((int64_t)cols + 4 * fp4_block(format) - 1) / (4 * fp4_block(format))); }
inline int64_t fp4_scale_bytes(int64_t rows, int cols, int format) { return (rows + 127) / 128 * fp4_tiles(cols, format) * 512; }

// 2^exponent, 1 / (6 * 2^exponent) and what its rounding left.
inline void fp4_scale_factors(int exponent, float *tensor_scale, float *sixth, float *sixth_rest) {
  *tensor_scale = ldexpf(1.f, exponent);
  *sixth = ldexpf(1.f / 6.f, -exponent);
  *sixth_rest = (float)ldexp(1.0 / 6.0 - (double)(1.f / 6.f), -exponent);
}

// Rows of a quantisation that are pixels of a strided layer: row (n, oh, ow) reads pixel (n, oh * S, ow * S).
struct Fp4Pixels {
  int H, W, OH, OW, S;
};

// fp4_quantize.cu.  `px` null: row r starts at x + r * ld.
int launch_fp4_quantize(const void *x, int x_type, int64_t rows, int cols, int64_t ld, const Fp4Pixels *px, int format, int exponent,
                        uint8_t *codes, uint8_t *scales, cudaStream_t st);
int launch_fp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int cols, int format, int exponent, void *y, int y_type,
                          int64_t ld, cudaStream_t st);
// bits of the largest finite |x| of rows * cols close values, combined into *d_bits
int launch_fp4_largest(const void *x, int x_type, int64_t n, unsigned *d_bits, cudaStream_t st);

// fp4_product.cu
struct Fp4Rows {             // activations of a product
  const uint8_t *codes, *scales;  // quantised ...
  const void *x;             // ... or, where codes is null, as they are
  int x_type;
  int64_t ld;
  const Fp4Pixels *px;
};
// The rows up to which a product quantises them itself (more are quantised into a workspace first; the sums are the same
// either way): one number, so that a workspace for some rows is enough for fewer.
int64_t fp4_product_direct_rows(const tetris_fp4_filter *f);
int launch_fp4_product(const tetris_fp4_filter *f, const Fp4Rows &a, int64_t rows, int exponent, const float *bias, void *y, int y_type, int64_t ld,
                       int relu, cudaStream_t st);

}  // namespace tetris

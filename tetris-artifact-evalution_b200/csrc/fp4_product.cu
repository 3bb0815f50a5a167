// Products of 4-bit activations and a 4-bit filter: y[row][oc] = sum_k a[row][k] w[oc][k] (+ bias, ReLU).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fp4.h"

namespace tetris {
namespace {

struct ProductParams {
  const uint8_t *a, *sa, *w, *sw;
  const float *bias;
  void *y;
  int64_t rows, ld, pitch;
  int K, N, tiles;
  int relu, exponent;
};

__device__ __forceinline__ float code_value(uint32_t c) {
  const float t[8] = {0.f, .5f, 1.f, 1.5f, 2.f, 3.f, 4.f, 6.f};
  return c & 8 ? -t[c & 7] : t[c & 7];
}
template <int FMT> __device__ __forceinline__ float scale_number(uint8_t b) {
  if (FMT == TETRIS_FP4_MX) return b == 0xFF ? __int_as_float(0x7FC00000) : b ? __uint_as_float((uint32_t)b << 23) : __uint_as_float(0x00400000u);
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)b));
  return __half2float(__ushort_as_half((unsigned short)(r & 0xFFFF)));
}
__device__ __forceinline__ int64_t scale_at(int64_t row, int blk, int tiles) {
  return ((row >> 7) * tiles + (blk >> 2)) * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4 + (blk & 3);
}

// One output per thread: the simplest form.
template <typename T, int FMT> __global__ void __launch_bounds__(256) product_kernel(const ProductParams p) {
  constexpr int kBlock = FMT == TETRIS_FP4_NV ? 16 : 32;
  const int oc = blockIdx.y * 32 + threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.y;
  if (oc >= p.N || row >= p.rows) return;
  float sum = 0.f;
  for (int b = 0; b * kBlock < p.K; ++b) {
    float part = 0.f;
    for (int k = b * kBlock / 2; k < (b + 1) * kBlock / 2; ++k) {
      const uint32_t ca = p.a[row * p.pitch + k], cw = p.w[oc * p.pitch + k];
      part += code_value(ca & 15) * code_value(cw & 15) + code_value(ca >> 4) * code_value(cw >> 4);
    }
    sum += part * scale_number<FMT>(p.sa[scale_at(row, b, p.tiles)]) * scale_number<FMT>(p.sw[scale_at(oc, b, p.tiles)]);
  }
  sum = ldexpf(sum, p.exponent);
  if (p.bias) sum += p.bias[oc];
  if (p.relu && sum < 0.f) sum = 0.f;  // (a NaN stays)
  static_cast<T *>(p.y)[row * p.ld + oc] = (T)sum;
}

}  // namespace

int launch_fp4_product(const tetris_fp4_filter *f, const uint8_t *codes, const uint8_t *scales, int64_t rows, int exponent, const float *bias,
                       void *y, int y_type, int64_t ld, int relu, cudaStream_t st) {
  const ProductParams p = {codes, scales, f->d_codes, f->d_scales, bias, y, rows, ld, f->pitch, f->in_channel, f->out_channel,
                           fp4_tiles(f->in_channel, f->format), relu, exponent + f->exponent};
  const dim3 grid((unsigned)((rows + 7) / 8), (unsigned)(p.N + 31) / 32), block(32, 8);
  const bool nv = f->format == TETRIS_FP4_NV;
  count_launch();
  if (y_type == TETRIS_FP32) (nv ? product_kernel<float, TETRIS_FP4_NV> : product_kernel<float, TETRIS_FP4_MX>)<<<grid, block, 0, st>>>(p);
  else if (y_type == TETRIS_BF16) (nv ? product_kernel<__nv_bfloat16, TETRIS_FP4_NV> : product_kernel<__nv_bfloat16, TETRIS_FP4_MX>)<<<grid, block, 0, st>>>(p);
  else (nv ? product_kernel<__half, TETRIS_FP4_NV> : product_kernel<__half, TETRIS_FP4_MX>)<<<grid, block, 0, st>>>(p);
  TETRIS_CUDA_TRY(cudaGetLastError());
  return TETRIS_OK;
}

}  // namespace tetris

// Rows of floating-point values into 4-bit codes with block scales, and back.
//
// Mathematics.  A block (32 values in the MX form, 16 in the NV form) has one scale s, a code is
// RNE(x / s) onto {0, .5, 1, 1.5, 2, 3, 4, 6}.
//   MX: s = 2^e with e + 127 = max(exponent field of the largest |x| - 2, 0): x / s is exact.
//   NV: s = 2^exponent * E4M3(largest |x| / (6 * 2^exponent)).  Both roundings have to be those of the
//       exact quotient.  The division by 6 is IEEE's: a quotient of 24 bits by 6 differs from a border
//       of E4M3 (at most 5 bits) by 0 or by more than half of its own last place, so rounding it to 24
//       bits first changes nothing.  The same holds for x / s, s having 4 significant bits and a border
//       between codes 3: half a last place of the quotient is less than the distance of the nearest x
//       that is not on the border.  That quotient is taken as q = x r with r = 1 / s rounded, corrected by
//       the exact remainder (Markstein: q + r (x - q s), the correctly rounded quotient).
//
// Bound: HBM.  A thread takes 16 bytes of a row, the threads of a block find their largest value with
// shuffles, so that every load and store of a warp is contiguous; kChunks independent chunks per thread
// keep loads in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fp4.h"

namespace tetris {
namespace {

constexpr int kThreads = 256, kChunks = 4;

struct QuantizeParams {
  const void *x;
  uint8_t *codes, *scales;
  int64_t rows, ld, pitch;
  int64_t total;           // chunks of all rows
  int cols, tiles;         // tiles: scale tiles of a row
  int exponent;
  Fp4Div by_chunks;        // chunks of a row, whole scale tiles
  Fp4Pixels px;
  Fp4Div by_OH, by_OW;
};

template <typename T> __device__ __forceinline__ float to_float(T v) { return (float)v; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// max that hands a NaN on
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// codes of 8 values, the first in the lowest 4 bits (RNE, at most 6)
__device__ __forceinline__ uint32_t codes_of(const float (&v)[8]) {
  uint32_t r;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ uint16_t codes_of(const float (&v)[4]) {
  uint32_t r;
  asm("{\n.reg .b8 a, b;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "mov.b32 %0, {a, b, a, b};\n}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
  return (uint16_t)r;
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
template <int FMT, int CV>
__device__ __forceinline__ uint8_t scale_block(float (&v)[CV], float top, int exponent) {
  if (!(top < __int_as_float(0x7F800000))) {  // codes of 1: the block is NaN whatever it meets
#pragma unroll
    for (int i = 0; i < CV; ++i) v[i] = 1.f;
    return FMT == TETRIS_FP4_NV ? 0x7F : 0xFF;
  }
  if (FMT == TETRIS_FP4_MX) {
    const int byte = max((int)(__float_as_uint(top) >> 23) - 2, 0);  // at most 252
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
#pragma unroll
    for (int i = 0; i < CV; ++i) v[i] *= inv;
    return (uint8_t)byte;
  }
  const uint8_t byte = e4m3_of(__fdiv_rn(top * pow2f(-exponent), 6.f));
  const float s = e4m3_value(byte) * pow2f(exponent);
  if (top > 1e3f * s && s > 0.f) {  // far above what the exponent holds: x / s could leave FP32
    const float most = 1e3f * s;
#pragma unroll
    for (int i = 0; i < CV; ++i) v[i] = fminf(fmaxf(v[i], -most), most);
  }
  const float r = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
  for (int i = 0; i < CV; ++i) {
    const float q = v[i] * r;
    v[i] = __fmaf_rn(__fmaf_rn(-q, s, v[i]), r, q);
  }
  return byte;
}

__device__ __forceinline__ int64_t scale_at(int64_t row, int blk, int tiles) {
  return ((row >> 7) * tiles + (blk >> 2)) * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4 + (blk & 3);
}

template <typename T, int FMT, bool VEC, bool STRIDED>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantizeParams p) {
  constexpr int CV = 16 / sizeof(T);                                  // values of a chunk
  constexpr int kBlock = FMT == TETRIS_FP4_NV ? 16 : 32;
  constexpr int kLanes = kBlock / CV;                                 // threads of a block
  grid_release();
  grid_wait();
  float v[kChunks][CV];
  uint32_t chunk[kChunks];
  int64_t row[kChunks];
  const int64_t at = (int64_t)blockIdx.x * (kThreads * kChunks) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int64_t i = at + u * kThreads;
    if (p.total < (1ll << 31)) {
      const uint32_t r = fp4_quot((uint32_t)min(i, p.total), p.by_chunks);
      row[u] = i < p.total ? r : p.rows;
      chunk[u] = (uint32_t)i - r * p.by_chunks.d;
    } else {
      row[u] = i / p.by_chunks.d;
      chunk[u] = (uint32_t)(i - row[u] * p.by_chunks.d);
    }
    const int col = (int)chunk[u] * CV;
#pragma unroll
    for (int k = 0; k < CV; ++k) v[u][k] = 0.f;
    if (row[u] >= p.rows || col >= p.cols) continue;
    int64_t from = row[u] * p.ld;
    if (STRIDED) {
      const uint32_t y = fp4_quot((uint32_t)row[u], p.by_OW), ox = (uint32_t)row[u] - y * p.px.OW;
      const uint32_t n = fp4_quot(y, p.by_OH), oy = y - n * p.px.OH;
      from = (((int64_t)n * p.px.H + (int64_t)oy * p.px.S) * p.px.W + (int64_t)ox * p.px.S) * p.ld;
    }
    const T *src = static_cast<const T *>(p.x) + from + col;
    if (VEC && col + CV <= p.cols) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(src);
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int k = 0; k < CV; ++k) v[u][k] = to_float(e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < CV; ++k)
        if (col + k < p.cols) v[u][k] = to_float(src[k]);
    }
  }
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    float top = fabsf(v[u][0]);
#pragma unroll
    for (int k = 1; k < CV; ++k) top = max_nan(top, fabsf(v[u][k]));
#pragma unroll
    for (int s = 1; s < kLanes; s *= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, s));
    const uint8_t byte = scale_block<FMT>(v[u], top, p.exponent);
    if (row[u] >= p.rows) continue;
    const int col = (int)chunk[u] * CV, blk = col / kBlock, left = p.cols - col;
    auto codes = codes_of(v[u]);
    if (left < CV) codes = left <= 0 ? 0 : codes & ((1u << (4 * left)) - 1u);  // zeros behind the last column
    if (col / 2 < p.pitch) *reinterpret_cast<decltype(codes) *>(p.codes + row[u] * p.pitch + col / 2) = codes;
    if (chunk[u] % kLanes == 0) p.scales[scale_at(row[u], blk, p.tiles)] = byte;
  }
}

struct DequantizeParams {
  const uint8_t *codes, *scales;
  void *y;
  int64_t rows, ld, pitch;
  int64_t total;           // pieces of 8 columns of all rows
  int cols, tiles;
  int exponent;
  Fp4Div by_pieces;
};

__device__ __forceinline__ void values_of(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}

// The scale of a block as a number (without the tensor's exponent); NaN where the byte says so.
template <int FMT> __device__ __forceinline__ float scale_value(uint8_t b) {
  if (FMT == TETRIS_FP4_NV) return e4m3_value(b);
  return b == 0xFF ? __int_as_float(0x7FC00000) : b ? __uint_as_float((uint32_t)b << 23) : __uint_as_float(0x00400000u);
}

// A thread turns 8 codes (one block's) into values.
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const DequantizeParams p) {
  constexpr int kBlock = FMT == TETRIS_FP4_NV ? 16 : 32;
  grid_release();
  grid_wait();
  const int64_t at = (int64_t)blockIdx.x * (kThreads * kChunks) + threadIdx.x;
  const float tensor_scale = pow2f(p.exponent);
  uint32_t codes[kChunks], piece[kChunks];
  uint8_t byte[kChunks];
  int64_t row[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int64_t i = at + u * kThreads;
    if (p.total < (1ll << 31)) {
      const uint32_t r = fp4_quot((uint32_t)min(i, p.total), p.by_pieces);
      row[u] = i < p.total ? r : p.rows;
      piece[u] = (uint32_t)i - r * p.by_pieces.d;
    } else {
      row[u] = i / p.by_pieces.d;
      piece[u] = (uint32_t)(i - row[u] * p.by_pieces.d);
    }
    if (row[u] >= p.rows) continue;
    codes[u] = *reinterpret_cast<const uint32_t *>(p.codes + row[u] * p.pitch + piece[u] * 4);
    byte[u] = p.scales[scale_at(row[u], (int)piece[u] * 8 / kBlock, p.tiles)];
  }
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    if (row[u] >= p.rows) continue;
    float v[8];
    values_of(codes[u], v);
    const float s = scale_value<FMT>(byte[u]) * tensor_scale;
    const int col = (int)piece[u] * 8;
    T *dst = static_cast<T *>(p.y) + row[u] * p.ld + col;
    alignas(16) T out[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) out[k] = from_float<T>(v[k] * s);
    if (VEC && col + 8 <= p.cols) {
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4 *>(dst)[k] = reinterpret_cast<const uint4 *>(out)[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + k < p.cols) dst[k] = out[k];
    }
  }
}

// Bits of the largest finite |x|.
template <typename T> __global__ void __launch_bounds__(kThreads) largest_kernel(const T *x, int64_t n, unsigned *bits) {
  unsigned m = 0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const unsigned b = __float_as_uint(fabsf(to_float(x[i])));
    if (b < 0x7F800000u) m = max(m, b);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) atomicMax(bits, m);
}

bool vector_rows(const void *p, int64_t ld, int bytes) { return ((reinterpret_cast<uintptr_t>(p) | (uint64_t)(ld * bytes)) & 15) == 0; }

int blocks_for(int64_t total, unsigned *blocks) {
  const int64_t n = (total + kThreads * kChunks - 1) / (kThreads * kChunks);
  if (n > 0x7FFFFFFF) { set_error("a matrix of this size is outside what the kernels cover"); return TETRIS_ERR_UNSUPPORTED; }
  *blocks = (unsigned)n;
  return TETRIS_OK;
}

int launched(cudaError_t err) {
  if (err == cudaSuccess) return TETRIS_OK;
  set_error("launch failed: %s", cudaGetErrorString(err));
  return TETRIS_ERR_CUDA;
}

template <typename T> int quantize(QuantizeParams p, int format, bool strided, cudaStream_t st) {
  const bool vec = vector_rows(p.x, p.ld, sizeof(T));
  const int chunks = p.tiles * 4 * fp4_block(format) / (16 / (int)sizeof(T));
  p.by_chunks = fp4_div((uint32_t)chunks);
  p.total = p.rows * chunks;
  unsigned blocks;
  int rc = blocks_for(p.total, &blocks);
  if (rc) return rc;
  auto go = [&](void (*kernel)(const QuantizeParams)) { return launched(launch_overlapped(kernel, dim3(blocks), kThreads, 0, st, 1, p)); };
  if (format == TETRIS_FP4_NV) {
    if (strided) return vec ? go(quantize_kernel<T, TETRIS_FP4_NV, true, true>) : go(quantize_kernel<T, TETRIS_FP4_NV, false, true>);
    return vec ? go(quantize_kernel<T, TETRIS_FP4_NV, true, false>) : go(quantize_kernel<T, TETRIS_FP4_NV, false, false>);
  }
  if (strided) return vec ? go(quantize_kernel<T, TETRIS_FP4_MX, true, true>) : go(quantize_kernel<T, TETRIS_FP4_MX, false, true>);
  return vec ? go(quantize_kernel<T, TETRIS_FP4_MX, true, false>) : go(quantize_kernel<T, TETRIS_FP4_MX, false, false>);
}

template <typename T> int dequantize(DequantizeParams p, int format, cudaStream_t st) {
  const bool vec = vector_rows(p.y, p.ld, sizeof(T));
  const int pieces = (p.cols + 7) / 8;
  p.by_pieces = fp4_div((uint32_t)pieces);
  p.total = p.rows * pieces;
  unsigned blocks;
  int rc = blocks_for(p.total, &blocks);
  if (rc) return rc;
  auto go = [&](void (*kernel)(const DequantizeParams)) { return launched(launch_overlapped(kernel, dim3(blocks), kThreads, 0, st, 1, p)); };
  if (format == TETRIS_FP4_NV) return vec ? go(dequantize_kernel<T, TETRIS_FP4_NV, true>) : go(dequantize_kernel<T, TETRIS_FP4_NV, false>);
  return vec ? go(dequantize_kernel<T, TETRIS_FP4_MX, true>) : go(dequantize_kernel<T, TETRIS_FP4_MX, false>);
}

}  // namespace

int launch_fp4_quantize(const void *x, int x_type, int64_t rows, int cols, int64_t ld, const Fp4Pixels *px, int format, int exponent,
                        uint8_t *codes, uint8_t *scales, cudaStream_t st) {
  QuantizeParams p = {};
  p.x = x; p.codes = codes; p.scales = scales;
  p.rows = rows; p.cols = cols; p.ld = ld;
  p.pitch = fp4_pitch(cols);
  p.tiles = fp4_tiles(cols, format);
  p.exponent = exponent;
  if (px) {
    p.px = *px;
    p.by_OH = fp4_div((uint32_t)px->OH); p.by_OW = fp4_div((uint32_t)px->OW);
  }
  switch (x_type) {
    case TETRIS_FP32: return quantize<float>(p, format, px != nullptr, st);
    case TETRIS_BF16: return quantize<__nv_bfloat16>(p, format, px != nullptr, st);
    default: return quantize<__half>(p, format, px != nullptr, st);
  }
}

int launch_fp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int cols, int format, int exponent, void *y, int y_type,
                          int64_t ld, cudaStream_t st) {
  DequantizeParams p = {};
  p.codes = codes; p.scales = scales; p.y = y;
  p.rows = rows; p.cols = cols; p.ld = ld;
  p.pitch = fp4_pitch(cols);
  p.tiles = fp4_tiles(cols, format);
  p.exponent = exponent;
  switch (y_type) {
    case TETRIS_FP32: return dequantize<float>(p, format, st);
    case TETRIS_BF16: return dequantize<__nv_bfloat16>(p, format, st);
    default: return dequantize<__half>(p, format, st);
  }
}

int launch_fp4_largest(const void *x, int x_type, int64_t n, unsigned *d_bits, cudaStream_t st) {
  const unsigned blocks = (unsigned)std::min<int64_t>(1024, (n + kThreads - 1) / kThreads);
  switch (x_type) {
    case TETRIS_FP32: largest_kernel<<<blocks, kThreads, 0, st>>>(static_cast<const float *>(x), n, d_bits); break;
    case TETRIS_BF16: largest_kernel<<<blocks, kThreads, 0, st>>>(static_cast<const __nv_bfloat16 *>(x), n, d_bits); break;
    default: largest_kernel<<<blocks, kThreads, 0, st>>>(static_cast<const __half *>(x), n, d_bits);
  }
  return launched(cudaGetLastError());
}

}  // namespace tetris

// Rows of floating-point values into 4-bit codes with block scales, and back.
//
// The arithmetic of a block is in fp4_block.h.
//
// Bound: HBM; what stands in its way is the number of instructions, so a thread keeps one column position and walks
// down a few rows, takes 32 bytes at a time, and finds the largest one of 16-bit types as packed integers.  4096 x 8192
// (floors at 6.55 TB/s in brackets): from FP32 23.2 us MX, 23.9 NV (23.3), from BF16 15.2 and 17.9 (13.0); back to
// FP32 25.0 (23.3), to BF16 14.8 (13.0).
// Rows off the 16-byte grid (odd numbers of columns, views that begin beside it) are read and written value by value,
// neighbouring threads 32 bytes apart: the same bytes of HBM in eight to sixteen times the transactions.  4096 x 8191
// from FP32 37 us, from BF16 37, back to FP32 130, to BF16 99; 30000 x 259 FP32 9.3 and 40 (30000 x 256: 6.2 and 7.5).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "fp4.h"
#include "fp4_block.h"

namespace tetris {
namespace {

constexpr int kThreads = 256, kRows = 2, kRowsBack = 4;  // rows of a thread: quantising, and back

// How a block of threads covers a matrix cut into pieces of 8 or 16 columns: 2^lx threads side by side, the others
// below them, and again `ROWS` times.
struct Walk {
  int lx;
  uint32_t col_blocks;
};

struct QuantizeParams {
  const void *x;
  uint8_t *codes, *scales;
  uint32_t rows;
  int64_t ld, pitch;
  int cols, tiles;         // tiles: scale tiles of a row
  Walk walk;
  int wide;                // 32-byte aligned rows
  float tensor_scale;      // 2^exponent
  float sixth, sixth_rest; // 1 / (6 * 2^exponent) and what its rounding left
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

// Neighbouring values as they were loaded (32 bytes), and what is asked of them.
template <typename T> struct Piece {  // 16-bit types
  static constexpr int kValues = 16;
  uint32_t raw[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < 8; ++k) raw[k] = 0;
  }
  __device__ __forceinline__ void load(const T *src, bool wide) {
    if (wide) {
      asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]), "=r"(raw[7]) : "l"(src));
    } else {
      *reinterpret_cast<uint4 *>(raw) = reinterpret_cast<const uint4 *>(src)[0];
      *reinterpret_cast<uint4 *>(raw + 4) = reinterpret_cast<const uint4 *>(src)[1];
    }
  }
  __device__ __forceinline__ void set(int k, T v) { raw[k >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t *>(&v) << (16 * (k & 1)); }
  // Bits of |x|, two values side by side: as integers they are ordered like the numbers, NaN last.
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = raw[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int k = 1; k < 8; ++k) t = __vmaxu2(t, raw[k] & 0x7FFF7FFFu);
    return t;
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  static __device__ __forceinline__ float number(uint32_t t) {
    const uint16_t b = (uint16_t)max(t & 0xFFFFu, t >> 16);
    return to_float(*reinterpret_cast<const T *>(&b));
  }
  __device__ __forceinline__ void values(float (&v)[16]) const {
    const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = to_float(e[k]);
  }
};
template <> struct Piece<float> {
  static constexpr int kValues = 8;
  float v[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
  }
  __device__ __forceinline__ void load(const float *src, bool wide) {
    if (wide) {
      asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(src));
    } else {
      *reinterpret_cast<float4 *>(v) = reinterpret_cast<const float4 *>(src)[0];
      *reinterpret_cast<float4 *>(v + 4) = reinterpret_cast<const float4 *>(src)[1];
    }
  }
  __device__ __forceinline__ void set(int k, float x) { v[k] = x; }
  __device__ __forceinline__ uint32_t top() const {
    float t = fabsf(v[0]);
#pragma unroll
    for (int k = 1; k < 8; ++k) asm("max.NaN.f32 %0, %0, %1;" : "+f"(t) : "f"(fabsf(v[k])));
    return __float_as_uint(t);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ float number(uint32_t t) { return __uint_as_float(t); }
  __device__ __forceinline__ void values(float (&w)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = v[k];
  }
};

template <typename T, int FMT, bool VEC, bool STRIDED, int ROWS>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantizeParams p) {
  constexpr int kValues = Piece<T>::kValues;
  constexpr int kLanes = (FMT == TETRIS_FP4_NV ? 16 : 32) / kValues;  // threads of a block of values
  grid_release();
  grid_wait();
  const uint32_t row_block = blockIdx.x / p.walk.col_blocks, col_block = blockIdx.x - row_block * p.walk.col_blocks;
  const uint32_t below = kThreads >> p.walk.lx;
  const uint32_t piece = (col_block << p.walk.lx) + (threadIdx.x & ((1u << p.walk.lx) - 1u));
  const uint32_t row0 = row_block * (below * ROWS) + (threadIdx.x >> p.walk.lx);
  const int col = (int)piece * kValues, left = p.cols - col;          // (may lie behind the last column: zeros)
  const T *x = static_cast<const T *>(p.x) + col;
  Piece<T> in[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const uint32_t row = row0 + u * below;
    in[u].zero();
    if (row >= p.rows || left <= 0) continue;
    int64_t from = row;
    if (STRIDED) {
      const uint32_t y = fp4_quot(row, p.by_OW), ox = row - y * p.px.OW;
      const uint32_t n = fp4_quot(y, p.by_OH), oy = y - n * p.px.OH;
      from = ((int64_t)n * p.px.H + (int64_t)oy * p.px.S) * p.px.W + (int64_t)ox * p.px.S;
    }
    const T *src = x + from * p.ld;
    if (VEC && left >= kValues) {
      in[u].load(src, p.wide);
    } else {
#pragma unroll
      for (int k = 0; k < kValues; ++k)
        if (k < left) in[u].set(k, src[k]);
    }
  }
  // pieces cover a row's pitch (whole 32 columns); the last block also writes the zeros that fill its scale tile
  const bool has_codes = col / 2 < p.pitch, has_scale = has_codes && piece % kLanes == 0;
  const int fill = has_scale && (col + kLanes * kValues) / 2 >= p.pitch ? 3 - (int)(piece / kLanes % 4) : 0;
  auto keep = [](int left) { return left >= 8 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (4 * left)) - 1u; };  // zeros behind the last column
  const uint32_t keep0 = keep(left), keep1 = keep(left - 8);
  uint8_t *codes = p.codes + col / 2;
  uint8_t *scales = p.scales + (size_t)(piece / (4 * kLanes)) * 512 + piece / kLanes % 4;
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const uint32_t row = row0 + u * below;
    uint32_t top = in[u].top();
#pragma unroll
    for (int s = 1; s < kLanes; s *= 2) top = Piece<T>::larger(top, __shfl_xor_sync(0xffffffffu, top, s));
    float v[kValues];
    in[u].values(v);
    const BlockScale b = block_scale<FMT>(Piece<T>::number(top), p.tensor_scale, p.sixth, p.sixth_rest);
    if (b.far) bring_near(v, b);
    const uint32_t c = block_codes<FMT>(v, b) & keep0;
    if (row >= p.rows) continue;
    if (has_codes) {
      if (kValues == 16) *reinterpret_cast<uint2 *>(codes + row * p.pitch) = make_uint2(c, block_codes<FMT>(v + kValues - 8, b) & keep1);
      else *reinterpret_cast<uint32_t *>(codes + row * p.pitch) = c;
    }
    if (has_scale) {
      uint8_t *s = scales + (int64_t)(row >> 7) * p.tiles * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4;
      *s = b.byte;
      for (int k = 1; k <= fill; ++k) s[k] = 0;
    }
  }
}

struct DequantizeParams {
  const uint8_t *codes, *scales;
  void *y;
  uint32_t rows;
  int64_t ld, pitch;
  int cols, tiles;
  Walk walk;
  int wide;                // 32-byte aligned rows
  float tensor_scale;
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

template <typename T> __device__ __forceinline__ void store8(T *dst, const float (&v)[8], bool) {
  alignas(16) T out[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) out[k] = from_float<T>(v[k]);
  *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(out);
}
template <> __device__ __forceinline__ void store8(float *dst, const float (&v)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
  } else {
    reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

template <typename T, int FMT, bool VEC, int ROWS>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const DequantizeParams p) {
  constexpr int kLanes = (FMT == TETRIS_FP4_NV ? 16 : 32) / 8;
  grid_release();
  grid_wait();
  const uint32_t row_block = blockIdx.x / p.walk.col_blocks, col_block = blockIdx.x - row_block * p.walk.col_blocks;
  const uint32_t below = kThreads >> p.walk.lx;
  const uint32_t piece = (col_block << p.walk.lx) + (threadIdx.x & ((1u << p.walk.lx) - 1u));
  const uint32_t row0 = row_block * (below * ROWS) + (threadIdx.x >> p.walk.lx);
  const int col = (int)piece * 8, left = p.cols - col;
  if (left <= 0) return;
  const uint8_t *codes = p.codes + col / 2;
  const uint8_t *scales = p.scales + (size_t)(piece / (4 * kLanes)) * 512 + piece / kLanes % 4;
  uint32_t c[ROWS];
  uint8_t byte[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const uint32_t row = row0 + u * below;
    if (row >= p.rows) continue;
    c[u] = *reinterpret_cast<const uint32_t *>(codes + row * p.pitch);
    byte[u] = scales[(int64_t)(row >> 7) * p.tiles * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4];
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const uint32_t row = row0 + u * below;
    if (row >= p.rows) continue;
    float v[8];
    values_of(c[u], v);
    const float s = scale_value<FMT>(byte[u]) * p.tensor_scale;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= s;
    T *dst = static_cast<T *>(p.y) + row * p.ld + col;
    if (VEC && left >= 8) {
      store8(dst, v, p.wide);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) dst[k] = from_float<T>(v[k]);
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

bool vector_rows(const void *p, int64_t ld, int bytes, int align) { return ((reinterpret_cast<uintptr_t>(p) | (uint64_t)(ld * bytes)) & (align - 1)) == 0; }

int launched(cudaError_t err) {
  if (err == cudaSuccess) return TETRIS_OK;
  set_error("launch failed: %s", cudaGetErrorString(err));
  return TETRIS_ERR_CUDA;
}

// Threads side by side for `pieces` of a row: what leaves the fewest of them idle, more rather than fewer.
// `many`: enough blocks for every SM even with `thread_rows` rows a thread (few rows are spread over more threads).
int plan_walk(uint32_t rows, int64_t pieces, int thread_rows, Walk *w, unsigned *blocks, bool *many) {
  int64_t least = INT64_MAX;
  for (int lx = 8; lx >= 2; --lx) {
    const int64_t padded = ((pieces + (1 << lx) - 1) >> lx) << lx;
    if (padded < least) { least = padded; w->lx = lx; }
  }
  w->col_blocks = (uint32_t)(least >> w->lx);
  const int64_t below = kThreads >> w->lx;
  *many = (rows + below * thread_rows - 1) / (below * thread_rows) * w->col_blocks >= 2 * 148;
  const int64_t span = below * (*many ? thread_rows : 1), n = (rows + span - 1) / span * w->col_blocks;
  if (n > 0x7FFFFFFF) { set_error("a matrix of this size is outside what the kernels cover"); return TETRIS_ERR_UNSUPPORTED; }
  *blocks = (unsigned)n;
  return TETRIS_OK;
}

template <typename T, int FMT, bool VEC, bool STRIDED> int quantize(const QuantizeParams &p, unsigned blocks, bool many, cudaStream_t st) {
  return launched(many ? launch_overlapped(quantize_kernel<T, FMT, VEC, STRIDED, kRows>, dim3(blocks), kThreads, 0, st, 1, p)
                       : launch_overlapped(quantize_kernel<T, FMT, VEC, STRIDED, 1>, dim3(blocks), kThreads, 0, st, 1, p));
}
template <typename T, int FMT> int quantize(QuantizeParams p, bool strided, cudaStream_t st) {
  const bool vec = vector_rows(p.x, p.ld, sizeof(T), 16);
  p.wide = vector_rows(p.x, p.ld, sizeof(T), 32);
  unsigned blocks;
  bool many;
  const int rc = plan_walk(p.rows, p.pitch * 2 / Piece<T>::kValues, kRows, &p.walk, &blocks, &many);
  if (rc) return rc;
  if (strided) return vec ? quantize<T, FMT, true, true>(p, blocks, many, st) : quantize<T, FMT, false, true>(p, blocks, many, st);
  return vec ? quantize<T, FMT, true, false>(p, blocks, many, st) : quantize<T, FMT, false, false>(p, blocks, many, st);
}

template <typename T, int FMT, bool VEC> int dequantize(const DequantizeParams &p, unsigned blocks, bool many, cudaStream_t st) {
  return launched(many ? launch_overlapped(dequantize_kernel<T, FMT, VEC, kRowsBack>, dim3(blocks), kThreads, 0, st, 1, p)
                       : launch_overlapped(dequantize_kernel<T, FMT, VEC, 1>, dim3(blocks), kThreads, 0, st, 1, p));
}
template <typename T, int FMT> int dequantize(DequantizeParams p, cudaStream_t st) {
  const bool vec = vector_rows(p.y, p.ld, sizeof(T), 16);
  p.wide = vector_rows(p.y, p.ld, sizeof(T), 32);
  unsigned blocks;
  bool many;
  const int rc = plan_walk(p.rows, ((int64_t)p.cols + 7) / 8, kRowsBack, &p.walk, &blocks, &many);
  if (rc) return rc;
  return vec ? dequantize<T, FMT, true>(p, blocks, many, st) : dequantize<T, FMT, false>(p, blocks, many, st);
}

}  // namespace

int launch_fp4_quantize(const void *x, int x_type, int64_t rows, int cols, int64_t ld, const Fp4Pixels *px, int format, int exponent,
                        uint8_t *codes, uint8_t *scales, cudaStream_t st) {
  QuantizeParams p = {};
  p.x = x; p.codes = codes; p.scales = scales;
  p.rows = (uint32_t)rows; p.cols = cols; p.ld = ld;
  p.pitch = fp4_pitch(cols);
  p.tiles = fp4_tiles(cols, format);
  fp4_scale_factors(exponent, &p.tensor_scale, &p.sixth, &p.sixth_rest);
  if (px) {
    p.px = *px;
    p.by_OH = fp4_div((uint32_t)px->OH); p.by_OW = fp4_div((uint32_t)px->OW);
  }
  const bool nv = format == TETRIS_FP4_NV, strided = px != nullptr;
  switch (x_type) {
    case TETRIS_FP32: return nv ? quantize<float, TETRIS_FP4_NV>(p, strided, st) : quantize<float, TETRIS_FP4_MX>(p, strided, st);
    case TETRIS_BF16: return nv ? quantize<__nv_bfloat16, TETRIS_FP4_NV>(p, strided, st) : quantize<__nv_bfloat16, TETRIS_FP4_MX>(p, strided, st);
    default: return nv ? quantize<__half, TETRIS_FP4_NV>(p, strided, st) : quantize<__half, TETRIS_FP4_MX>(p, strided, st);
  }
}

int launch_fp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int cols, int format, int exponent, void *y, int y_type,
                          int64_t ld, cudaStream_t st) {
  DequantizeParams p = {};
  p.codes = codes; p.scales = scales; p.y = y;
  p.rows = (uint32_t)rows; p.cols = cols; p.ld = ld;
  p.pitch = fp4_pitch(cols);
  p.tiles = fp4_tiles(cols, format);
  p.tensor_scale = ldexpf(1.f, exponent);
  const bool nv = format == TETRIS_FP4_NV;
  switch (y_type) {
    case TETRIS_FP32: return nv ? dequantize<float, TETRIS_FP4_NV>(p, st) : dequantize<float, TETRIS_FP4_MX>(p, st);
    case TETRIS_BF16: return nv ? dequantize<__nv_bfloat16, TETRIS_FP4_NV>(p, st) : dequantize<__nv_bfloat16, TETRIS_FP4_MX>(p, st);
    default: return nv ? dequantize<__half, TETRIS_FP4_NV>(p, st) : dequantize<__half, TETRIS_FP4_MX>(p, st);
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

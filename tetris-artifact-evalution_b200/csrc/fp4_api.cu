// The C ABI of the 4-bit filters and products: argument checks and handle lifetime.
#include <cmath>
#include <cstring>
#include <new>

#include "fp4.h"

namespace tetris {
namespace {

constexpr int64_t kMaxRows = (1ll << 31) - 256;  // row numbers and their tiles are 32-bit in the kernels
constexpr int kMaxCols = 1 << 24;

int check_format(int format, int exponent) {
  if (format != TETRIS_FP4_MX && format != TETRIS_FP4_NV) { set_error("unknown 4-bit format %d", format); return TETRIS_ERR_INVALID; }
  if (format == TETRIS_FP4_MX ? exponent != 0 : exponent < -100 || exponent > 100) {
    set_error("exponent %d: has to be %s in this format", exponent, format == TETRIS_FP4_MX ? "0" : "-100 to 100");
    return TETRIS_ERR_INVALID;
  }
  return TETRIS_OK;
}

int check_extent(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) { set_error("bad matrix: rows=%lld cols=%lld", (long long)rows, (long long)cols); return TETRIS_ERR_INVALID; }
  if (rows > kMaxRows || cols > kMaxCols) {
    set_error("a matrix of %lld x %lld is outside what the kernels cover (%lld x %d)", (long long)rows, (long long)cols, (long long)kMaxRows, kMaxCols);
    return TETRIS_ERR_UNSUPPORTED;
  }
  return TETRIS_OK;
}

int type_bytes(int type) { return type == TETRIS_FP32 ? 4 : type == TETRIS_BF16 || type == TETRIS_FP16 ? 2 : 0; }

// A dense matrix: type, row distance (0 becomes cols), alignment of the type.
int check_dense(const char *what, const void *p, int type, int cols, int64_t *ld) {
  const int bytes = type_bytes(type);
  if (!bytes) { set_error("unknown type %d of the %s", type, what); return TETRIS_ERR_INVALID; }
  if (*ld == 0) *ld = cols;
  if (*ld < cols || *ld > (1ll << 40)) { set_error("rows of the %s lie %lld elements apart, they have %d", what, (long long)*ld, cols); return TETRIS_ERR_INVALID; }
  if (reinterpret_cast<uintptr_t>(p) % bytes) { set_error("the %s is not aligned to its type", what); return TETRIS_ERR_INVALID; }
  return TETRIS_OK;
}

// Memory that a kernel on `device` is given: a host pointer or another device's would fault there.
int check_memory(const char *what, const void *p, int device, int align) {
  if (!p) { set_error("the pointer of the %s is NULL", what); return TETRIS_ERR_INVALID; }
  if (reinterpret_cast<uintptr_t>(p) % align) { set_error("the %s has to be %d-byte aligned", what, align); return TETRIS_ERR_INVALID; }
  cudaPointerAttributes attr;
  if (cudaPointerGetAttributes(&attr, p) != cudaSuccess || !(attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged) ||
      (attr.type == cudaMemoryTypeDevice && attr.device != device)) {
    cudaGetLastError();
    set_error("the %s is not memory of device %d", what, device);
    return TETRIS_ERR_INVALID;
  }
  return TETRIS_OK;
}

int check_filter(const tetris_fp4_filter *f) {
  if (!f) { set_error("filter handle is NULL"); return TETRIS_ERR_INVALID; }
  return TETRIS_OK;
}

int64_t workspace_codes(const tetris_fp4_filter *f, int64_t rows) { return (rows * f->pitch + 255) / 256 * 256; }
int64_t workspace_bytes(const tetris_fp4_filter *f, int64_t rows) {
  return rows <= f->direct_rows ? 0 : workspace_codes(f, rows) + fp4_scale_bytes(rows, f->in_channel, f->format);
}

// Checks that all products share; the filter's device is current.
int check_product(const tetris_fp4_filter *f, int64_t rows, int exponent, const float *bias, const void *y, int y_type, int64_t *ld_y, int flags) {
  int rc;
  if ((rc = check_extent(rows, f->in_channel)) || (rc = check_format(f->format, exponent))) return rc;
  if (flags & ~TETRIS_FUSE_RELU) { set_error("unknown fusion flags 0x%x", flags); return TETRIS_ERR_INVALID; }
  if ((rc = check_dense("output", y, y_type, f->out_channel, ld_y))) return rc;
  if (rows == 0) return TETRIS_OK;
  if ((rc = check_memory("output", y, f->device, type_bytes(y_type)))) return rc;
  if (bias && (rc = check_memory("bias", bias, f->device, 4))) return rc;
  return TETRIS_OK;
}

// Floating-point activations through the workspace.
int linear(const tetris_fp4_filter *f, const void *x, int x_type, int64_t rows, int64_t ld_x, const Fp4Pixels *px, int exponent, const float *bias,
           void *y, int y_type, int64_t ld_y, int flags, void *workspace, int64_t bytes, cudaStream_t st) {
  int rc;
  if ((rc = check_product(f, rows, exponent, bias, y, y_type, &ld_y, flags))) return rc;
  if ((rc = check_dense("input", x, x_type, f->in_channel, &ld_x))) return rc;
  if (rows == 0) return TETRIS_OK;
  if ((rc = check_memory("input", x, f->device, type_bytes(x_type)))) return rc;
  const int64_t need = workspace_bytes(f, rows);
  if (bytes < need) { set_error("a workspace of %lld bytes, %lld are needed", (long long)bytes, (long long)need); return TETRIS_ERR_INVALID; }
  if (need && (rc = check_memory("workspace", workspace, f->device, 16))) return rc;
  if (!need) return launch_fp4_product(f, {nullptr, nullptr, x, x_type, ld_x, px}, rows, exponent, bias, y, y_type, ld_y, flags & TETRIS_FUSE_RELU, st);
  uint8_t *codes = static_cast<uint8_t *>(workspace), *scales = codes + workspace_codes(f, rows);
  if ((rc = launch_fp4_quantize(x, x_type, rows, f->in_channel, ld_x, px, f->format, exponent, codes, scales, st))) return rc;
  return launch_fp4_product(f, {codes, scales, nullptr, 0, 0, nullptr}, rows, exponent, bias, y, y_type, ld_y, flags & TETRIS_FUSE_RELU, st);
}

}  // namespace
}  // namespace tetris

using namespace tetris;

extern "C" {

int tetris_fp4_sizes(int64_t rows, int cols, int format, int64_t *pitch, int64_t *code_bytes, int64_t *scale_bytes) {
  int rc;
  if ((rc = check_format(format, 0)) || (rc = check_extent(rows, cols))) return rc;
  if (pitch) *pitch = fp4_pitch(cols);
  if (code_bytes) *code_bytes = rows * fp4_pitch(cols);
  if (scale_bytes) *scale_bytes = fp4_scale_bytes(rows, cols, format);
  return TETRIS_OK;
}

int tetris_fp4_quantize(const void *d_x, int x_type, int64_t rows, int cols, int64_t ld, int format, int exponent, void *d_codes,
                        void *d_scales, void *stream) {
  int rc, dev = 0;
  if ((rc = check_format(format, exponent)) || (rc = check_extent(rows, cols)) || (rc = check_dense("input", d_x, x_type, cols, &ld))) return rc;
  if (rows == 0) return TETRIS_OK;
  TETRIS_CUDA_TRY(cudaGetDevice(&dev));
  if ((rc = check_memory("input", d_x, dev, type_bytes(x_type))) || (rc = check_memory("codes", d_codes, dev, 16)) ||
      (rc = check_memory("scales", d_scales, dev, 16)))
    return rc;
  return launch_fp4_quantize(d_x, x_type, rows, cols, ld, nullptr, format, exponent, static_cast<uint8_t *>(d_codes),
                             static_cast<uint8_t *>(d_scales), (cudaStream_t)stream);
}

int tetris_fp4_dequantize(const void *d_codes, const void *d_scales, int64_t rows, int cols, int format, int exponent, void *d_y, int y_type,
                          int64_t ld, void *stream) {
  int rc, dev = 0;
  if ((rc = check_format(format, exponent)) || (rc = check_extent(rows, cols)) || (rc = check_dense("output", d_y, y_type, cols, &ld))) return rc;
  if (rows == 0) return TETRIS_OK;
  TETRIS_CUDA_TRY(cudaGetDevice(&dev));
  if ((rc = check_memory("codes", d_codes, dev, 16)) || (rc = check_memory("scales", d_scales, dev, 16)) ||
      (rc = check_memory("output", d_y, dev, type_bytes(y_type))))
    return rc;
  return launch_fp4_dequantize(static_cast<const uint8_t *>(d_codes), static_cast<const uint8_t *>(d_scales), rows, cols, format, exponent, d_y,
                               y_type, ld, (cudaStream_t)stream);
}

int tetris_fp4_filter_create(const void *weights, int w_type, int in_channel, int out_channel, int kernel_size, int format, int exponent,
                             int device, void *stream, tetris_fp4_filter_t **out) {
  if (!weights || !out) { set_error("weights or out pointer is NULL"); return TETRIS_ERR_INVALID; }
  *out = nullptr;
  int rc;
  const bool automatic = exponent == TETRIS_FP4_EXPONENT_AUTO;
  int64_t ld = 0;
  if ((rc = check_format(format, automatic ? 0 : exponent))) return rc;
  if (out_channel < 1) { set_error("bad filter shape: ic=%d oc=%d", in_channel, out_channel); return TETRIS_ERR_INVALID; }
  if ((rc = check_extent(out_channel, in_channel)) || (rc = check_dense("filter", weights, w_type, in_channel, &ld))) return rc;
  if (out_channel > kMaxCols) { set_error("%d output channels are more than the kernels cover", out_channel); return TETRIS_ERR_UNSUPPORTED; }
  if (kernel_size != 1) { set_error("a 4-bit filter is 1x1, kernel size %d is not covered", kernel_size); return TETRIS_ERR_UNSUPPORTED; }
  int n_dev = 0;
  TETRIS_CUDA_TRY(cudaGetDeviceCount(&n_dev));
  if (device < 0 || device >= n_dev) { set_error("device %d out of range (%d visible)", device, n_dev); return TETRIS_ERR_INVALID; }
  cudaPointerAttributes attr;
  bool on_device = false;
  if (cudaPointerGetAttributes(&attr, weights) == cudaSuccess) {
    on_device = attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged;
    if (attr.type == cudaMemoryTypeDevice && attr.device != device) { set_error("the filter lies on device %d, not on device %d", attr.device, device); return TETRIS_ERR_INVALID; }
  } else {
    cudaGetLastError();
  }
  DeviceGuard guard(device);
  if (!guard.ok) { set_error("cudaSetDevice(%d) failed", device); return TETRIS_ERR_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;

  tetris_fp4_filter *f = new (std::nothrow) tetris_fp4_filter();
  if (!f) { set_error("out of host memory"); return TETRIS_ERR_NOMEM; }
  f->in_channel = in_channel; f->out_channel = out_channel;
  f->format = format; f->exponent = automatic ? 0 : exponent;
  f->device = device;
  f->pitch = fp4_pitch(in_channel);
  f->code_bytes = out_channel * f->pitch;
  f->scale_bytes = fp4_scale_bytes(out_channel, in_channel, format);
  const int64_t values = (int64_t)out_channel * in_channel, dense_bytes = values * type_bytes(w_type);
  void *d_dense = nullptr;
  unsigned *d_bits = nullptr;
  auto fail = [&](int code) {
    cudaDeviceSynchronize();
    device_free(d_dense); device_free(d_bits);
    tetris_fp4_filter_destroy(f);
    return code;
  };
  auto alloc = [&](void **p, int64_t bytes, const char *what) {
    if (device_alloc(p, (size_t)bytes) == cudaSuccess) return true;
    cudaGetLastError();
    set_error("allocation of %lld bytes of device memory for %s failed", (long long)bytes, what);
    return false;
  };
  if (cudaDeviceGetAttribute(&f->sm_count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    set_error("device attributes: %s", cudaGetErrorString(cudaGetLastError()));
    return fail(TETRIS_ERR_CUDA);
  }
  f->direct_rows = fp4_product_direct_rows(f);
  if (!alloc((void **)&f->d_codes, f->code_bytes, "the codes") || !alloc((void **)&f->d_scales, f->scale_bytes, "the scales") ||
      !alloc((void **)&f->d_error, sizeof(int), "the error flag") || !alloc((void **)&d_bits, sizeof(unsigned), "the largest weight") ||
      (!on_device && !alloc(&d_dense, dense_bytes, "the dense filter")))
    return fail(TETRIS_ERR_NOMEM);
  // The pool's memory is in the order of the default stream: what was just taken is waited for there.
  if (cudaMemsetAsync(f->d_scales, 0, (size_t)f->scale_bytes, 0) != cudaSuccess || cudaMemsetAsync(f->d_error, 0, sizeof(int), 0) != cudaSuccess ||
      cudaMemsetAsync(d_bits, 0, sizeof(unsigned), 0) != cudaSuccess ||
      (!on_device && copy_to_device(d_dense, weights, (size_t)dense_bytes, 0) != cudaSuccess) || cudaStreamSynchronize(0) != cudaSuccess) {
    set_error("copy of the dense filter to the device failed: %s", cudaGetErrorString(cudaGetLastError()));
    return fail(TETRIS_ERR_CUDA);
  }
  const void *dense = on_device ? weights : d_dense;
  if (automatic && format == TETRIS_FP4_NV) {
    unsigned bits = 0;
    if ((rc = launch_fp4_largest(dense, w_type, values, d_bits, st))) return fail(rc);
    if (cudaMemcpyAsync(&bits, d_bits, sizeof(bits), cudaMemcpyDeviceToHost, st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess) {
      set_error("reading the largest weight failed: %s", cudaGetErrorString(cudaGetLastError()));
      return fail(TETRIS_ERR_CUDA);
    }
    float largest;
    memcpy(&largest, &bits, sizeof(largest));
    if (largest > 0.f) {  // the smallest k with largest <= 6 * 448 * 2^k
      int e = 0;
      const double m = std::frexp((double)largest / 2688.0, &e);
      f->exponent = m == 0.5 ? e - 1 : e;
      f->exponent = f->exponent < -100 ? -100 : f->exponent > 100 ? 100 : f->exponent;
    }
  }
  if ((rc = launch_fp4_quantize(dense, w_type, out_channel, in_channel, in_channel, nullptr, format, f->exponent, f->d_codes, f->d_scales, st))) return fail(rc);
  if (cudaStreamSynchronize(st) != cudaSuccess) {
    set_error("quantising the filter failed: %s", cudaGetErrorString(cudaGetLastError()));
    return fail(TETRIS_ERR_CUDA);
  }
  device_free(d_dense);
  device_free(d_bits);
  *out = f;
  return TETRIS_OK;
}

void tetris_fp4_filter_destroy(tetris_fp4_filter_t *f) {
  if (!f) return;
  DeviceGuard guard(f->device);
  cudaDeviceSynchronize();  // products on any stream may still read the filter
  device_free(f->d_codes);
  device_free(f->d_scales);
  device_free(f->d_error);
  delete f;
}

int tetris_fp4_filter_info(const tetris_fp4_filter_t *f, tetris_fp4_filter_info_t *info) {
  if (!f || !info) { set_error("NULL argument"); return TETRIS_ERR_INVALID; }
  memset(info, 0, sizeof(*info));
  info->in_channel = f->in_channel; info->out_channel = f->out_channel;
  info->format = f->format; info->exponent = f->exponent;
  info->pitch = f->pitch; info->code_bytes = f->code_bytes; info->scale_bytes = f->scale_bytes;
  info->device = f->device;
  return TETRIS_OK;
}

int tetris_fp4_filter_download(const tetris_fp4_filter_t *f, void *codes, void *scales) {
  int rc = check_filter(f);
  if (rc) return rc;
  DeviceGuard guard(f->device);
  if (codes) TETRIS_CUDA_TRY(copy_to_host(codes, f->d_codes, (size_t)f->code_bytes, 0));
  if (scales) TETRIS_CUDA_TRY(copy_to_host(scales, f->d_scales, (size_t)f->scale_bytes, 0));
  return TETRIS_OK;
}

int tetris_fp4_filter_check(const tetris_fp4_filter_t *f) {
  int rc = check_filter(f);
  if (rc) return rc;
  DeviceGuard guard(f->device);
  if (cudaDeviceSynchronize() != cudaSuccess) {
    set_error("device error: %s", cudaGetErrorString(cudaGetLastError()));
    return TETRIS_ERR_CUDA;
  }
  int flag = 0;
  TETRIS_CUDA_TRY(cudaMemcpy(&flag, f->d_error, sizeof(flag), cudaMemcpyDeviceToHost));
  if (!flag) return TETRIS_OK;
  TETRIS_CUDA_TRY(cudaMemset(f->d_error, 0, sizeof(int)));
  set_error("a product of this filter gave up on a bounded barrier wait; its output is invalid");
  return TETRIS_ERR_CUDA;
}

int tetris_fp4_product(const tetris_fp4_filter_t *f, const void *d_codes, const void *d_scales, int64_t rows, int exponent, const float *d_bias,
                       void *d_y, int y_type, int64_t ld, int flags, void *stream) {
  int rc = check_filter(f);
  if (rc) return rc;
  DeviceGuard guard(f->device);
  if (!guard.ok) { set_error("cudaSetDevice(%d) failed", f->device); return TETRIS_ERR_CUDA; }
  if ((rc = check_product(f, rows, exponent, d_bias, d_y, y_type, &ld, flags)) || rows == 0) return rc;
  if ((rc = check_memory("codes", d_codes, f->device, 16)) || (rc = check_memory("scales", d_scales, f->device, 16))) return rc;
  return launch_fp4_product(f, {static_cast<const uint8_t *>(d_codes), static_cast<const uint8_t *>(d_scales), nullptr, 0, 0, nullptr}, rows, exponent,
                            d_bias, d_y, y_type, ld, flags & TETRIS_FUSE_RELU, (cudaStream_t)stream);
}

int tetris_fp4_workspace(const tetris_fp4_filter_t *f, int64_t rows, int64_t *bytes) {
  int rc = check_filter(f);
  if (rc || (rc = check_extent(rows, f->in_channel))) return rc;
  if (!bytes) { set_error("bytes pointer is NULL"); return TETRIS_ERR_INVALID; }
  *bytes = workspace_bytes(f, rows);
  return TETRIS_OK;
}

int tetris_fp4_linear(const tetris_fp4_filter_t *f, const void *d_x, int x_type, int64_t rows, int64_t ld_x, int exponent, const float *d_bias,
                      void *d_y, int y_type, int64_t ld_y, int flags, void *d_workspace, int64_t workspace_bytes, void *stream) {
  int rc = check_filter(f);
  if (rc) return rc;
  DeviceGuard guard(f->device);
  if (!guard.ok) { set_error("cudaSetDevice(%d) failed", f->device); return TETRIS_ERR_CUDA; }
  return linear(f, d_x, x_type, rows, ld_x, nullptr, exponent, d_bias, d_y, y_type, ld_y, flags, d_workspace, workspace_bytes, (cudaStream_t)stream);
}

int tetris_fp4_conv2d(const tetris_fp4_filter_t *f, const float *d_input_nhwc, float *d_output_nhwc, int batch_size, int img_h, int img_w,
                      int stride, int padding, int exponent, const float *d_bias, int flags, void *d_workspace, int64_t workspace_bytes,
                      void *stream) {
  int rc = check_filter(f);
  if (rc) return rc;
  if (batch_size < 0 || img_h < 1 || img_w < 1 || stride < 1) {
    set_error("bad conv shape: batch=%d h=%d w=%d stride=%d padding=%d", batch_size, img_h, img_w, stride, padding);
    return TETRIS_ERR_INVALID;
  }
  if (padding != 0) { set_error("a 4-bit layer has no padding, got %d", padding); return TETRIS_ERR_UNSUPPORTED; }
  DeviceGuard guard(f->device);
  if (!guard.ok) { set_error("cudaSetDevice(%d) failed", f->device); return TETRIS_ERR_CUDA; }
  const Fp4Pixels px = {img_h, img_w, (img_h - 1) / stride + 1, (img_w - 1) / stride + 1, stride};
  const int64_t image = (int64_t)px.OH * px.OW;
  if (batch_size && image > kMaxRows / batch_size) { set_error("%d images of %dx%d are more rows than the kernels cover", batch_size, px.OH, px.OW); return TETRIS_ERR_UNSUPPORTED; }
  return linear(f, d_input_nhwc, TETRIS_FP32, batch_size * image, 0, stride > 1 ? &px : nullptr, exponent, d_bias, d_output_nhwc, TETRIS_FP32, 0,
                flags, d_workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"

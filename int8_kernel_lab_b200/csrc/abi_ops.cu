// abi_ops.cu - the extern "C" boundary of the products, the row quantisation
// and the group norm: argument checks, then one launch.
#include <math.h>
#include <stdint.h>

#include "int8conv.h"
#include "launch.h"

namespace {

constexpr int64_t kMaxRows = (int64_t(1) << 31) - 512;  // int32 row indices + one tile
constexpr int64_t kMaxPitch = int64_t(1) << 40;         // tensor-map stride limit, in bytes

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

uintptr_t size_of(int dtype) {
  return dtype == INT8CONV_INT8 ? 1 : (dtype == INT8CONV_BF16 || dtype == INT8CONV_FP16) ? 2 : 4;
}

bool known_activation(int a) { return a >= INT8CONV_ACT_NONE && a <= INT8CONV_ACT_SILU; }

bool good_step(float s) { return isfinite(s) && s > 0.f && isfinite(1.0f / s); }

bool is_float(int dtype) {
  return dtype == INT8CONV_BF16 || dtype == INT8CONV_FP16 || dtype == INT8CONV_FP32;
}

int8conv_status check_matmul(const int8conv_matmul *d, const int8_t *a, const int8_t *b, void *y) {
  if (d == nullptr) return INT8CONV_BAD_ARGUMENT;
  if (d->m < 0 || d->m > kMaxRows || d->n < 0 || d->n > kMaxRows) return INT8CONV_BAD_ARGUMENT;
  if (d->k < 1 || d->k > INT8CONV_MAX_PRODUCT_K) return INT8CONV_BAD_ARGUMENT;
  if (d->lda < d->k || d->lda % 16 != 0 || d->lda >= kMaxPitch) return INT8CONV_BAD_ARGUMENT;
  if (d->ldb < d->k || d->ldb % 16 != 0 || d->ldb >= kMaxPitch) return INT8CONV_BAD_ARGUMENT;
  if (!is_float(d->y_dtype) && d->y_dtype != INT8CONV_INT8) return INT8CONV_BAD_ARGUMENT;
  const int64_t size = static_cast<int64_t>(size_of(d->y_dtype));
  if (d->ldy < d->n || d->ldy >= kMaxPitch / size) return INT8CONV_BAD_ARGUMENT;
  if (!known_activation(d->activation)) return INT8CONV_BAD_ARGUMENT;
  if (d->y_dtype == INT8CONV_INT8 && !good_step(d->out_scale)) return INT8CONV_BAD_ARGUMENT;
  if (d->residual != nullptr) {
    if (d->y_dtype == INT8CONV_INT8) return INT8CONV_BAD_ARGUMENT;
    if (d->ldr < d->n || d->ldr >= kMaxPitch / size) return INT8CONV_BAD_ARGUMENT;
  }
  if (d->m == 0 || d->n == 0) return INT8CONV_OK;
  if (a == nullptr || b == nullptr || y == nullptr) return INT8CONV_BAD_POINTER;
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(y, size_of(d->y_dtype)) ||
      !aligned(d->residual, size_of(d->y_dtype)) || !aligned(d->row_scale, 4) ||
      !aligned(d->col_scale, 4) || !aligned(d->bias, 4))
    return INT8CONV_BAD_POINTER;
  return INT8CONV_OK;
}

int8conv_status check_norm(const int8conv_group_norm *d) {
  if (d == nullptr) return INT8CONV_BAD_ARGUMENT;
  if (d->n < 0 || d->pixels < 0 || d->n > kMaxRows || d->pixels > kMaxRows)
    return INT8CONV_BAD_ARGUMENT;
  if (d->channels < 1 || d->channels > INT8CONV_MAX_NORM_CHANNELS || d->groups < 1 ||
      d->groups > INT8CONV_MAX_NORM_GROUPS || d->channels % d->groups != 0)
    return INT8CONV_BAD_ARGUMENT;
  if (d->ldx < d->channels || d->ldy < d->channels || d->ldx >= kMaxPitch || d->ldy >= kMaxPitch)
    return INT8CONV_BAD_ARGUMENT;
  if (!is_float(d->x_dtype) && d->x_dtype != INT8CONV_INT32) return INT8CONV_BAD_ARGUMENT;
  if (!is_float(d->y_dtype) && d->y_dtype != INT8CONV_INT8) return INT8CONV_BAD_ARGUMENT;
  if (!isfinite(d->eps) || d->eps < 0.f) return INT8CONV_BAD_ARGUMENT;
  if (!known_activation(d->activation)) return INT8CONV_BAD_ARGUMENT;
  if (d->y_dtype == INT8CONV_INT8 && !good_step(d->out_scale)) return INT8CONV_BAD_ARGUMENT;
  if (i8c::group_norm_blocks(*d) > kMaxRows) return INT8CONV_BAD_ARGUMENT;
  return INT8CONV_OK;
}

}  // namespace

extern "C" {

int8conv_status int8conv_launch_matmul(const int8conv_matmul *desc, const int8_t *a,
                                       const int8_t *b, void *y, void *stream) {
  int8conv_status st = check_matmul(desc, a, b, y);
  if (st != INT8CONV_OK) return st;
  if (desc->m == 0 || desc->n == 0) return INT8CONV_OK;
  st = i8c::check_device();
  if (st != INT8CONV_OK) return st;
  return i8c::launch_matmul_impl(*desc, a, b, 0, nullptr, 0, y, static_cast<cudaStream_t>(stream));
}

int8conv_status int8conv_launch_grouped_matmul(const int8conv_matmul *desc, const int8_t *a,
                                               const int8_t *b, int64_t group_stride,
                                               const int32_t *offsets, int32_t groups, void *y,
                                               void *stream) {
  int8conv_status st = check_matmul(desc, a, b, y);
  if (st != INT8CONV_OK) return st;
  if (groups < 1 || groups > INT8CONV_MAX_GROUPS || desc->residual != nullptr)
    return INT8CONV_BAD_ARGUMENT;
  if (groups > 1 && (group_stride < 16 || group_stride % 16 != 0 || group_stride >= kMaxPitch))
    return INT8CONV_BAD_ARGUMENT;
  if (desc->m == 0 || desc->n == 0) return INT8CONV_OK;
  if (offsets == nullptr || !aligned(offsets, 4)) return INT8CONV_BAD_POINTER;
  st = i8c::check_device();
  if (st != INT8CONV_OK) return st;
  return i8c::launch_matmul_impl(*desc, a, b, group_stride, offsets, groups, y,
                                 static_cast<cudaStream_t>(stream));
}

int32_t int8conv_debug_matmul_form(int64_t m, int64_t n, int64_t k, int32_t groups, int32_t sms) {
  if (m < 1 || m > kMaxRows || n < 1 || n > kMaxRows || k < 1 || k > INT8CONV_MAX_PRODUCT_K ||
      groups < 0 || groups > INT8CONV_MAX_GROUPS || sms < 1)
    return 0;
  return i8c::matmul_form(m, n, k, groups, sms);
}

int8conv_status int8conv_launch_quantize_rows(int64_t m, int64_t k, int32_t x_dtype, const void *x,
                                              int64_t rows, int64_t ldx, const int32_t *index,
                                              int8_t *q, int64_t ldq, float *scale, void *stream) {
  if (m < 0 || m > kMaxRows || k < 1 || k >= kMaxPitch || rows < 0) return INT8CONV_BAD_ARGUMENT;
  if (!is_float(x_dtype)) return INT8CONV_BAD_ARGUMENT;
  if (ldx < k || ldx >= kMaxPitch || ldq < k || ldq >= kMaxPitch) return INT8CONV_BAD_ARGUMENT;
  if (index == nullptr && rows < m) return INT8CONV_BAD_ARGUMENT;
  if (m == 0) return INT8CONV_OK;
  if ((x == nullptr && rows > 0) || q == nullptr || scale == nullptr) return INT8CONV_BAD_POINTER;
  if (!aligned(x, size_of(x_dtype)) || !aligned(scale, 4) || !aligned(index, 4))
    return INT8CONV_BAD_POINTER;
  const int8conv_status st = i8c::check_device();
  if (st != INT8CONV_OK) return st;
  return i8c::launch_quantize_rows_impl(m, k, x_dtype, x, rows, ldx, index, q, ldq, scale,
                                        static_cast<cudaStream_t>(stream));
}

size_t int8conv_group_norm_workspace_bytes(const int8conv_group_norm *desc) {
  return check_norm(desc) == INT8CONV_OK ? i8c::group_norm_workspace(*desc) : 0;
}

int8conv_status int8conv_launch_group_norm(const int8conv_group_norm *desc, const void *x, void *y,
                                           void *workspace, size_t workspace_bytes, void *stream) {
  int8conv_status st = check_norm(desc);
  if (st != INT8CONV_OK) return st;
  if (desc->n == 0 || desc->pixels == 0) return INT8CONV_OK;
  if (x == nullptr || y == nullptr) return INT8CONV_BAD_POINTER;
  if (!aligned(x, size_of(desc->x_dtype)) || !aligned(y, size_of(desc->y_dtype)) ||
      !aligned(desc->scale, 4) || !aligned(desc->gamma, 4) || !aligned(desc->beta, 4))
    return INT8CONV_BAD_POINTER;
  const size_t need = i8c::group_norm_workspace(*desc);
  if (workspace_bytes < need) return INT8CONV_WORKSPACE_TOO_SMALL;
  if (need > 0 && (workspace == nullptr || !aligned(workspace, 16))) return INT8CONV_BAD_POINTER;
  st = i8c::check_device();
  if (st != INT8CONV_OK) return st;
  return i8c::launch_group_norm_impl(*desc, x, y, workspace, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

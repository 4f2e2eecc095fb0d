// rk_mx.h -- quantised rows (rk_rows): what the kernels that write, read
// and attend over them share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rk_host.h"
#include "rotatek_hip.h"

namespace rk {

constexpr int kMxBlock = 32;  // channels of one scale

inline int64_t mx_width(int64_t D) { return (D + kMxBlock - 1) / kMxBlock * kMxBlock; }
inline int64_t mx_row_bytes(int64_t D, int format) { return format == RK_ROWS_MX8 ? mx_width(D) : mx_width(D) / 2; }

// Shapes, dtypes, strides and alignment of quantised rows; `data` may be
// NULL (host-only checks).
inline int check_mx(const rk_rows* r) {
  if (!r) return RK_ERR_NULL;
  if (r->format != RK_ROWS_MX8 && r->format != RK_ROWS_MX4) return RK_ERR_ARG;
  int st = check_desc(&r->data, 4);
  if (st) return st;
  if ((st = check_desc(&r->scales, 4))) return st;
  if (r->data.dtype != RK_U8 || r->scales.dtype != RK_U8) return RK_ERR_DTYPE;
  if (r->head_dim < 0 || r->head_dim > 128) return RK_ERR_HEAD_DIM;
  const int64_t S = r->data.shape[2];
  if (r->data.shape[3] != mx_row_bytes(r->head_dim, r->format)) return RK_ERR_SHAPE;
  if (r->scales.shape[0] != r->data.shape[0] || r->scales.shape[1] != r->data.shape[1] ||
      r->scales.shape[2] != mx_width(r->head_dim) / kMxBlock ||
      r->scales.shape[3] < (S + kMxBlock - 1) / kMxBlock * kMxBlock)
    return RK_ERR_SHAPE;
  if (numel(&r->data) == 0) return RK_OK;
  if (r->data.stride[3] != 1 || r->scales.stride[3] != 1) return RK_ERR_STRIDE;
  for (int i = 0; i < 3; ++i) {
    if (r->data.shape[i] > 1 && r->data.stride[i] % 16 != 0) return RK_ERR_STRIDE;
    if (r->scales.shape[i] > 1 && r->scales.stride[i] % 8 != 0) return RK_ERR_STRIDE;
  }
  if (((uintptr_t)r->data.data & 15) != 0 || ((uintptr_t)r->scales.data & 7) != 0) return RK_ERR_STRIDE;
  // in-head byte offsets are 32 bits in the kernels, also those of a chunk's
  // rows before they are clamped to the last one
  if ((S + 64) * r->data.stride[2] + 128 >= (INT64_C(1) << 31) ||
      4 * r->scales.stride[2] + S + 64 >= (INT64_C(1) << 31))
    return RK_ERR_STRIDE;
  return RK_OK;
}

}  // namespace rk

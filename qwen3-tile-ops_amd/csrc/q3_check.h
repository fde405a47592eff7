// Checks of the operators' view arguments, shared by the files that define
// the C ABI's operators (include/q3ops.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "q3ops.h"

namespace q3 {

inline int elem_size(uint8_t dt) { return (dt == Q3_DT_I8 || dt == Q3_DT_U8) ? 1 : 4; }

// A view with no data: NULL data on a view that has rows.  A 0-row view
// may carry NULL (a caller's empty tensor); the operators then do nothing
// for it, as the reference's row loops do.
inline bool no_data(const q3_view *v) { return !v->data && v->rows != 0; }

// A dense-column view of the given dtype with at least `cols` columns.
inline int check_view(const q3_view *v, uint8_t dt) {
  if (!v || no_data(v)) return Q3_ERR_ARG;
  if (v->dtype != dt) return Q3_ERR_DTYPE;
  const int es = elem_size(dt);
  if (v->col_bytes != es) return Q3_ERR_VIEW;
  if (v->rows > 1 && (v->row_bytes < static_cast<int64_t>(v->cols) * es || v->row_bytes % es != 0))
    return Q3_ERR_VIEW;
  return Q3_OK;
}

// A per-element vector [n][1] f32 (or a [1][n] row): returns its stride in
// elements via *stride.
inline int check_vec(const q3_view *v, uint32_t n, int64_t *stride) {
  if (!v || no_data(v)) return Q3_ERR_ARG;
  if (v->dtype != Q3_DT_F32) return Q3_ERR_DTYPE;
  if (v->rows >= n && v->cols >= 1) {
    if (v->row_bytes % 4 != 0 || (n > 1 && v->row_bytes < 4)) return Q3_ERR_VIEW;
    *stride = v->row_bytes / 4;
    return Q3_OK;
  }
  if (v->rows == 1 && v->cols >= n && v->col_bytes == 4) {
    *stride = 1;
    return Q3_OK;
  }
  return Q3_ERR_VIEW;
}

// An f32 scale matrix [rows][cols] whose columns may be strided
// (col_bytes a multiple of 4): at least `rows` x `cols`, and each row long
// enough for its last column.
inline int check_scales(const q3_view *v, uint32_t rows, uint32_t cols) {
  if (!v || no_data(v)) return Q3_ERR_ARG;
  if (v->dtype != Q3_DT_F32) return Q3_ERR_DTYPE;
  if (v->row_bytes % 4 || v->col_bytes % 4 || v->col_bytes <= 0) return Q3_ERR_VIEW;
  if (v->rows < rows || v->cols < cols) return Q3_ERR_VIEW;
  if (rows > 1 && cols > 0 &&
      v->row_bytes < static_cast<int64_t>(cols - 1) * v->col_bytes + 4)
    return Q3_ERR_VIEW;
  return Q3_OK;
}

inline int64_t ld(const q3_view *v) { return v->row_bytes / elem_size(v->dtype); }

// Q3_ERR_UNSUPPORTED, or Q3_OK where q3_set_silent_unsupported is on.
int unsupported();

inline int hip_status(hipError_t e) { return e == hipSuccess ? Q3_OK : Q3_ERR_HIP; }

#define Q3_TRY(expr)                 \
  do {                               \
    const int q3_rc_ = (expr);       \
    if (q3_rc_ != Q3_OK) return q3_rc_; \
  } while (0)

}  // namespace q3

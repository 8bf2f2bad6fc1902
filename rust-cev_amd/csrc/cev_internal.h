// Internal helpers shared by the host code and the launchers.
#pragma once
#include <stdarg.h>
#include <stdint.h>

#include "../../include/cev_hip.h"

// Records a formatted thread-local message for cev_last_error() and returns
// `code`, so call sites read `return cev_fail(CEV_ERR_INVALID, "...", ...)`.
int32_t cev_fail(int32_t code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void cev_clear_error();

#define CEV_CHECK_ARG(cond, ...)                      \
  do {                                                \
    if (!(cond)) return cev_fail(CEV_ERR_INVALID, __VA_ARGS__); \
  } while (0)

// Whether `extent` rows of a stride (in elements) stay within 64-bit byte offsets.
static inline bool cev_stride_fits(int64_t stride, int64_t extent) {
  return stride >= 0 && (extent <= 1 || stride <= ((int64_t)1 << 59) / extent);
}

// Rows in memory, `stride` bytes apart (of one row it does not matter).
struct CevRows {
  const void* p;
  int64_t rows, stride, bytes;
};

// Whether two sets of rows share a byte, where those of a set do not overlap
// each other.  Columns side by side in a wider buffer share none.
extern "C" bool cev_overlap(const CevRows* a, const CevRows* b);
// Rows of `cols` elements of e bytes; none where p is null.
inline CevRows cev_rows(const void* p, int64_t rows, int64_t stride, int64_t cols, int64_t e) { return {p, p ? rows : 0, rows > 1 ? stride * e : 0, cols * e}; }
inline bool cev_same(const CevRows& a, const CevRows& b) { return a.p == b.p && (a.rows <= 1 || a.stride == b.stride); }

// Validates an attention descriptor (dtype, shapes, strides, scale); the
// planner runs it on every plan build and the launcher on every launch.
int32_t cev_check_attn_desc(const cev_attn_desc* d);

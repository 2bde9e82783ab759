// Argument checks of the microscaled operators: plain host code without a GPU call, which the CPU tests compile by itself. The
// includer provides `fail(code, format, ...)`.
#pragma once
#include <stdint.h>

#include "../../include/ill_hip.h"

namespace illm {

constexpr int64_t kMost = 1ll << 34;         // values of a call that quantises: a thread takes eight, a launch has fewer than 2^32
constexpr int64_t kMostInner = 1 << 20, kMostCols = 1 << 24, kMostRows = 1 << 26, kMostOut = 1ll << 32;   // (a launch of a product has fewer than 2^23 workgroups)

inline bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

inline int check_format(int format) {
  return format == ILL_MXF8 || format == ILL_MXF4 ? ILL_OK : fail(ILL_E_FORMAT, "mx: format %d (ILL_MXF8 or ILL_MXF4)", format);
}
inline int check_dtype(int dtype) {
  return dtype == ILL_F32 || dtype == ILL_F16 || dtype == ILL_BF16 ? ILL_OK : fail(ILL_E_FORMAT, "mx: type %d (ILL_F32, ILL_F16 or ILL_BF16)", dtype);
}
inline int check_mx(const char* what, const void* codes, const void* powers) {
  if (!codes || !powers) return fail(ILL_E_ARG, "mx: %s: null codes or powers", what);
  if (!aligned(codes, 16) || !aligned(powers, 16)) return fail(ILL_E_ARG, "mx: %s: codes or powers are not aligned to 16 bytes", what);
  return ILL_OK;
}

// Of quantize and dequantize; where rows are 0 nothing else is looked at but the sizes and types.
inline int check_rows(int format, int dtype, const void* x, int64_t stride, int64_t rows, int64_t cols, const void* codes, const void* powers) {
  if (int rc = check_format(format)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (rows < 0 || cols < 32 || cols % 32 || cols > kMost || rows > kMost / cols)
    return fail(ILL_E_ARG, "mx: %lld rows of %lld values (a multiple of 32; up to 2^34 in all)", (long long)rows, (long long)cols);
  const int unit = dtype == ILL_F32 ? 4 : 8;
  if (stride < cols || stride % unit || stride > kMost)
    return fail(ILL_E_ARG, "mx: row stride %lld (at least %lld, a multiple of %d)", (long long)stride, (long long)cols, unit);
  if (!rows) return ILL_OK;
  if (!x || !aligned(x, 16)) return fail(ILL_E_ARG, "mx: values are %s", x ? "not aligned to 16 bytes" : "null");
  return check_mx("rows", codes, powers);
}

inline int check_product(int format, const void* x, const void* xp, const void* w, const void* wp, const float* bias, const void* y, int64_t stride, int dtype,
                         int64_t rows, int64_t cols, int64_t inner) {
  if (int rc = check_format(format)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (rows < 0 || rows > kMostRows || cols < 1 || cols > kMostCols || inner < 32 || inner % 32 || inner > kMostInner || rows * cols > kMostOut)
    return fail(ILL_E_ARG, "mx: product of %lld rows and %lld columns over %lld (a multiple of 32 up to 2^20; up to 2^26 rows, 2^24 columns, 2^32 outputs)",
                (long long)rows, (long long)cols, (long long)inner);
  if (stride < cols || stride > kMost) return fail(ILL_E_ARG, "mx: output row stride %lld (at least %lld)", (long long)stride, (long long)cols);
  if (!aligned(bias, 4)) return fail(ILL_E_ARG, "mx: bias is an array of 4-byte values");
  if (!rows) return ILL_OK;
  if (!y || !aligned(y, dtype == ILL_F32 ? 4 : 2)) return fail(ILL_E_ARG, "mx: output is %s", y ? "not aligned to its type" : "null");
  if (int rc = check_mx("rows", x, xp)) return rc;
  return check_mx("matrix", w, wp);
}

}  // namespace illm

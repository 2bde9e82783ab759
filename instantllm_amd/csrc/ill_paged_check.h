// Argument checks of the paged-cache operators: plain host code without a GPU call, which the CPU
// tests compile by itself. The includer provides `fail(code, format, ...)`.
#pragma once
#include <math.h>
#include <stdint.h>

#include <utility>

#include "../../include/ill_hip.h"

namespace illp {

constexpr int64_t kMost = 1 << 30;                          // positions, strides
constexpr int64_t kMostRows = 1 << 26, kMostSeqHeads = 1 << 22;   // times heads: a launch has fewer than 2^24 workgroups of 256 threads
// Every workgroup of attention, and of append with row0 every row's wave, looks at all sequences: time grows with their square.
// Single rows behind 100 positions, 14 / 2 heads of 64: 1024 sequences 42 us, 4096 0.32 ms, 16384 4.1 ms (without a hint of max_rows
// 11); 256 key/value heads are 128 times as many workgroups.
constexpr int64_t kMostSeqs = 1 << 14;

inline bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

// Strides of three nested dimensions over runs of `dim`: none reaches into the next.
inline bool nested(int64_t dim, int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2) {
  int64_t s[3] = {s0, s1, s2}, n[3] = {n0, n1, n2}, least = dim;
  for (int i = 0; i < 3; i++) {
    int k = i;
    for (int j = i + 1; j < 3; j++)
      if (s[j] < s[k]) k = j;
    std::swap(s[i], s[k]);
    std::swap(n[i], n[k]);
    if (s[i] > INT64_MAX / 8 / n[i]) return false;
    if (n[i] > 1 && s[i] < least) return false;
    if (n[i] > 1) least = s[i] * n[i];
  }
  return true;
}

// A handle's type of queries and outputs, and of a 16-bit cache; and whether its cache is microscaled.
inline int type_of(const ill_paged_desc& d) { return d.dtype & ~ILL_MXF8; }
inline bool microscaled(const ill_paged_desc& d) { return d.dtype & ILL_MXF8; }
// Bytes of a microscaled page's codes, which its powers follow.
inline int64_t mx_codes_of(const ill_paged_desc& d) { return (int64_t)d.page_size * d.kv_heads * d.head_dim; }

// Checks a description and fills in what it leaves at 0.
inline int check_desc(ill_paged_desc& d) {
  if (type_of(d) != ILL_F16 && type_of(d) != ILL_BF16)
    return fail(ILL_E_FORMAT, "paged: cache type %d (ILL_F16 or ILL_BF16, or one of them | ILL_MXF8)", d.dtype);
  if (d.kv_heads < 1 || d.heads < d.kv_heads || d.heads % d.kv_heads || d.heads > 1024)
    return fail(ILL_E_ARG, "paged: %d query heads over %d key/value heads (a multiple, at most 1024)", d.heads, d.kv_heads);
  if (d.head_dim != 64 && d.head_dim != 128) return fail(ILL_E_ARG, "paged: head size %d (64 or 128)", d.head_dim);
  if (d.page_size < 16 || d.page_size > 1024 || (d.page_size & (d.page_size - 1)))
    return fail(ILL_E_ARG, "paged: pages of %d positions (a power of two, 16 to 1024)", d.page_size);
  if (d.rotary_dim < 0 || d.rotary_dim > d.head_dim || d.rotary_dim % 16)
    return fail(ILL_E_ARG, "paged: rotary_dim %d (a multiple of 16, up to the head size)", d.rotary_dim);
  if (d.rotary_dim && !(d.rope_base >= 1 && std::isfinite(d.rope_base))) return fail(ILL_E_ARG, "paged: rope_base %g (at least 1)", d.rope_base);
  if (!(d.norm_eps >= 0 && std::isfinite(d.norm_eps))) return fail(ILL_E_ARG, "paged: norm_eps %g", d.norm_eps);
  if (d.scale == 0) d.scale = (float)(1 / std::sqrt((double)d.head_dim));
  if (!(d.scale > 0 && std::isfinite(d.scale))) return fail(ILL_E_ARG, "paged: scale %g", d.scale);
  if (d.streams == 0) d.streams = 8;
  if (d.streams < 1 || d.streams > 256) return fail(ILL_E_ARG, "paged: %d streams (up to 256)", d.streams);
  if (microscaled(d)) {
    const int64_t bytes = mx_codes_of(d) + mx_codes_of(d) / 32;
    if (d.slot_stride || d.head_stride) return fail(ILL_E_ARG, "paged: slot and head strides of a microscaled cache (0: its pages have one layout)");
    if (!d.page_stride) d.page_stride = bytes;
    if (d.page_stride < bytes || d.page_stride % 16)
      return fail(ILL_E_ARG, "paged: microscaled pages %lld bytes apart (at least %lld, a multiple of 16)", (long long)d.page_stride, (long long)bytes);
    return d.page_stride <= INT64_MAX / 8 ? ILL_OK : fail(ILL_E_ARG, "paged: page stride %lld", (long long)d.page_stride);
  }
  if (!d.page_stride && !d.slot_stride && !d.head_stride) {
    d.head_stride = d.head_dim;
    d.slot_stride = (int64_t)d.kv_heads * d.head_dim;
    d.page_stride = d.slot_stride * d.page_size;
  }
  for (const int64_t s : {d.page_stride, d.slot_stride, d.head_stride})
    if (s < d.head_dim || s % 8) return fail(ILL_E_ARG, "paged: cache stride %lld (at least the head size, a multiple of 8)", (long long)s);
  if (d.slot_stride > kMost / 64) return fail(ILL_E_ARG, "paged: slot stride %lld (at most 2^24)", (long long)d.slot_stride);
  if (!nested(d.head_dim, d.page_stride, 1, d.slot_stride, d.page_size, d.head_stride, d.kv_heads))
    return fail(ILL_E_ARG, "paged: cache strides %lld, %lld, %lld overlap", (long long)d.page_stride, (long long)d.slot_stride,
                (long long)d.head_stride);
  return ILL_OK;
}

inline int check_batch(const ill_paged_desc& d, const ill_paged_batch* b) {
  if (!b) return fail(ILL_E_ARG, "paged: null batch");
  if (b->seqs < 0 || b->rows < 0 || b->rows > kMostRows / d.heads || b->seqs > kMostSeqHeads / d.heads || b->seqs > kMostSeqs)
    return fail(ILL_E_ARG, "paged: %d sequences, %lld rows (up to 2^14 sequences, rows x heads up to 2^26, sequences x heads up to 2^22)", b->seqs,
                (long long)b->rows);
  if (b->pages < 1 || b->pages > INT32_MAX || b->table_width < 1 || b->table_width > kMost / d.page_size || b->table_stride < b->table_width ||
      b->table_stride > kMost)
    return fail(ILL_E_ARG, "paged: %lld pages, table of %d entries, %lld apart (positions up to 2^30)", (long long)b->pages, b->table_width,
                (long long)b->table_stride);
  if (b->max_rows < 0) return fail(ILL_E_ARG, "paged: max_rows %lld", (long long)b->max_rows);
  if (b->seqs && (!b->lens || !b->table)) return fail(ILL_E_ARG, "paged: null lens or table");
  if (!b->row0 && b->rows < b->seqs) return fail(ILL_E_ARG, "paged: %lld rows for %d sequences of one row each", (long long)b->rows, b->seqs);
  if (!aligned(b->lens, 4) || !aligned(b->table, 4) || !aligned(b->row0, 4))
    return fail(ILL_E_ARG, "paged: lens, table and row0 are arrays of 4-byte values");
  if (microscaled(d)) {
    if (d.page_stride > INT64_MAX / 8 / b->pages) return fail(ILL_E_ARG, "paged: %lld pages, %lld bytes apart", (long long)b->pages, (long long)d.page_stride);
  } else if (!nested(d.head_dim, d.page_stride, b->pages, d.slot_stride, d.page_size, d.head_stride, d.kv_heads))
    return fail(ILL_E_ARG, "paged: cache strides %lld, %lld, %lld overlap for %lld pages", (long long)d.page_stride, (long long)d.slot_stride,
                (long long)d.head_stride, (long long)b->pages);
  return ILL_OK;
}

// A buffer of rows: its address, and its row stride against the width of a row.
inline int check_rows(const char* what, const void* at, int64_t stride, int64_t width, int type) {
  const int unit = type == ILL_F32 ? 4 : 8;
  if (!at || !aligned(at, 16)) return fail(ILL_E_ARG, "paged: %s is %s", what, at ? "not aligned to 16 bytes" : "null");
  if (stride < width || stride % unit || stride > kMost)
    return fail(ILL_E_ARG, "paged: %s: row stride %lld (at least %lld, a multiple of %d)", what, (long long)stride, (long long)width, unit);
  return ILL_OK;
}

inline int check_caches(const void* k, const void* v) {
  return k && v && aligned(k, 16) && aligned(v, 16) ? ILL_OK : fail(ILL_E_ARG, "paged: caches are null or not aligned to 16 bytes");
}

inline int check_append(const ill_paged_desc& d, const ill_paged_batch* b, const ill_paged_rows* x, const void* kc, const void* vc) {
  if (int rc = check_batch(d, b)) return rc;
  if (!x) return fail(ILL_E_ARG, "paged: null rows");
  if (x->dtype != ILL_F32 && x->dtype != type_of(d)) return fail(ILL_E_FORMAT, "paged: rows of type %d (ILL_F32 or the handle's)", x->dtype);
  const int64_t qw = (int64_t)d.heads * d.head_dim, kw = (int64_t)d.kv_heads * d.head_dim;
  if (x->q) {
    if (int rc = check_rows("q", x->q, x->q_stride, qw, x->dtype)) return rc;
    if (int rc = check_rows("q_out", x->q_out, x->q_out_stride, qw, type_of(d))) return rc;
    if (x->q_out == x->q && (x->dtype != type_of(d) || x->q_stride != x->q_out_stride))
      return fail(ILL_E_ARG, "paged: q_out is q, of another type or stride");
  }
  if (int rc = check_rows("k", x->k, x->k_stride, kw, x->dtype)) return rc;
  if (int rc = check_rows("v", x->v, x->v_stride, kw, x->dtype)) return rc;
  if (!aligned(x->bias, 4) || !aligned(x->q_norm, 4) || !aligned(x->k_norm, 4) || !aligned(x->positions, 4))
    return fail(ILL_E_ARG, "paged: bias, norms and positions are arrays of 4-byte values");
  return check_caches(kc, vc);
}

inline int check_attend(const ill_paged_desc& d, const ill_paged_batch* b, const void* q, int64_t q_stride, const void* kc, const void* vc, int window,
                        int sinks, const void* out, int64_t out_stride, int out_dtype) {
  if (int rc = check_batch(d, b)) return rc;
  if (out_dtype != ILL_F32 && out_dtype != type_of(d)) return fail(ILL_E_FORMAT, "paged: output of type %d (ILL_F32 or the handle's)", out_dtype);
  const int64_t w = (int64_t)d.heads * d.head_dim;
  if (int rc = check_rows("q", q, q_stride, w, type_of(d))) return rc;
  if (int rc = check_rows("out", out, out_stride, w, out_dtype)) return rc;
  if (out == q) return fail(ILL_E_ARG, "paged: out is q");
  if (window < 0 || sinks < 0) return fail(ILL_E_ARG, "paged: window %d, sinks %d", window, sinks);
  return check_caches(kc, vc);
}

inline int check_read(const ill_paged_desc& d, const ill_paged_batch* b, const void* kc, const void* vc, const void* k, int64_t k_stride, const void* v,
                      int64_t v_stride, int out_dtype) {
  if (int rc = check_batch(d, b)) return rc;
  if (out_dtype != ILL_F32 && out_dtype != type_of(d)) return fail(ILL_E_FORMAT, "paged: output of type %d (ILL_F32 or the handle's)", out_dtype);
  const int64_t w = (int64_t)d.kv_heads * d.head_dim;
  if (int rc = check_rows("k", k, k_stride, w, out_dtype)) return rc;
  if (int rc = check_rows("v", v, v_stride, w, out_dtype)) return rc;
  if (k == v) return fail(ILL_E_ARG, "paged: k is v");
  return check_caches(kc, vc);
}

}  // namespace illp

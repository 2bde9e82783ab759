// Index bounds of the paged-cache operators: plain functions of sizes, used by the host, by the
// kernels and, compiled by themselves, by the CPU tests.
#pragma once
#include <stdint.h>
#ifndef __host__
#define PG_FN inline
#else
#define PG_FN __host__ __device__ __forceinline__
#endif

// A batch as the kernels read it (ill_paged_batch with the handle's geometry).
struct PgBatch {
  const int32_t* lens;    // [seqs] positions of a sequence, its new rows included
  const int32_t* table;   // [seqs][table_stride] page of each page_size positions
  const int32_t* row0;    // [seqs + 1] first new row of each sequence; null: row s is sequence s's only one
  int64_t table_stride, pages;
  int32_t seqs, rows, table_width, page_log;
};

// Lengths as the kernels use them: none below 0, and none whose positions pass 2^30.
PG_FN int pg_len(int len) { return len < 0 ? 0 : len < 1 << 30 ? len : 1 << 30; }

// Positions that a sequence's table has pages for (at most 2^30: the entry points check it); the
// ones past them are neither written nor seen.
PG_FN int pg_cap(const PgBatch& b) { return b.table_width << b.page_log; }

// Whether the row at position p sees position j.
PG_FN bool pg_sees(int p, int j, int window, int sinks) { return j >= 0 && j <= p && (window == 0 || j > p - window || j < sinks); }

// Work division and index bounds of the paged-cache operators: plain functions of sizes, used by
// the host, by the kernels and, compiled by themselves, by the CPU tests.
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#define PG_FN __host__ __device__ __forceinline__
#else
#define PG_FN inline
#endif

#define PG_MOST (1 << 30)    // positions, rows x heads, windows and sinks: at most this many
#define PG_MAXSPLIT 256      // parts that the keys of a tile of rows are cut into at most
#define PG_FAN 16            // of which so many are joined at a time, in two steps (131071 keys in 256 parts: 20.1 us; 32: 21.7)

// A batch as the kernels read it (ill_paged_batch with the handle's geometry).
struct PgBatch {
  const int32_t* lens;    // [seqs] positions of a sequence, its new rows included
  const int32_t* table;   // [seqs][table_stride] page of each page_size positions
  const int32_t* row0;    // [seqs + 1] first new row of each sequence; null: row s is sequence s's only one
  int64_t table_stride, pages;
  int32_t seqs, rows, table_width, page_log;
};

PG_FN int pg_min(int a, int b) { return a < b ? a : b; }
PG_FN int pg_max(int a, int b) { return a > b ? a : b; }
PG_FN int pg_up(uint32_t a, uint32_t b) { return (int)((a + b - 1) / b); }   // a / b rounded up, a <= 2^30

// Lengths as the kernels use them: none below 0, and none whose positions pass 2^30.
PG_FN int pg_len(int len) { return pg_min(pg_max(len, 0), PG_MOST); }

// Positions that a sequence's table has pages for (at most 2^30: the entry points check it); the
// ones past them are neither written nor seen.
PG_FN int pg_cap(const PgBatch& b) { return b.table_width << b.page_log; }

// A sequence's new rows: rows first .. first + n - 1 of the buffers, at positions p0 ..; `begin` and
// `end` are its entries of row0. Rows that the buffers do not have are left out.
struct PgSeq {
  int first, n, p0;
};
PG_FN PgSeq pg_seq(int begin, int end, int len, int rows) {
  const int a = pg_min(pg_max(begin, 0), rows), e = pg_min(pg_max(end, a), rows);
  const int64_t p0 = (int64_t)pg_len(len) - ((int64_t)end - a);
  return {a, e - a, p0 < -PG_MOST ? -PG_MOST : (int)p0};
}

// Whether the row at position p sees position j.
PG_FN bool pg_sees(int p, int j, int window, int sinks) { return j >= 0 && j <= p && (window == 0 || j > p - window || j < sinks); }

// Rows of a workgroup of the append kernel, whose 256 threads take `items` pieces of each row: as few as fill the threads'
// turns to four fifths, up to 8, and fewer where there would be less than two workgroups for each CU. (64 rows of 384 pieces
// at 4 rows to a workgroup, 16 workgroups of six turns: 10.2 us; at one row 6.9.)
PG_FN int pg_append_rows(int rows, int items) {
  int best = 1;
  for (int r = 1; r <= 8; r++) {
    const int used = r * items, room = pg_up(used, 256) * 256;
    if (5 * used >= 4 * room) {
      best = r;
      break;
    }
    if (r == 1 || used * (pg_up(best * items, 256) * 256) > best * items * room) best = r;
  }
  return pg_max(1, pg_min(best, rows / 512));
}

// ---- the work of an attention call -------------------------------------------------------
// A sequence's n new rows and the G query heads of a key/value head make n G flat rows (row f / G,
// head f % G), which read the same keys; M of them are a tile of rows. Keys come in tiles of KT.
struct PgCut {
  uint32_t G, kv;
  int32_t M, KT, window, sinks;
  int32_t log;       // 2^log parts are wanted in all, where there are that many
  int32_t least;     // tiles of keys in a part at least
  int32_t lo, hi;    // sequences with lo < n G <= hi are this kernel's
  int32_t shared;    // the other kernel runs too: lo or hi hold as pg_share says
};

// Two kernels evaluate a batch. Sequences of up to PG_FEW flat rows are always the step kernel's (16 flat rows to a tile);
// the others are the prompt kernel's (128) if they have PG_MANY tiles of 128 in all, times key/value heads, about one for
// each CU, and the step kernel's otherwise. (Step against prompt kernel, us, 14 / 2 heads of 64: 512 rows, 56 tiles, 7.1 against
// 21.5; 1024 rows behind 4000, 112 tiles, 55 against 51; 2048 rows, 224 tiles, 35.8 against 34.0; 8 x 512 rows, 448 tiles, 58
// against 20. 32 / 8 heads of 128: 512 rows behind 4000, 128 tiles, 84 against 90; 4 x 256, 256 tiles, 36 against 16; but 64 x
// 2 rows behind 1000, 512 tiles of 8 flat rows, 44 against 50.)
#define PG_FEW 32
#define PG_MANY 224
PG_FN int pg_prompt_tiles(int n, uint32_t G, uint32_t kv) {
  const uint32_t f = (uint32_t)n * G;
  return f > PG_FEW ? (int)((f + 127) / 128 * kv) : 0;
}
// The limits of the step kernel (M 16) or of the prompt kernel, from the sum of pg_prompt_tiles over the sequences.
PG_FN void pg_share(PgCut& c, int64_t tiles) {
  const bool many = tiles >= PG_MANY;
  if (c.M == 16) c.hi = many ? PG_FEW : PG_MOST;
  else c.lo = many ? PG_FEW : PG_MOST;
}

PG_FN int pg_qtiles(int n, const PgCut& c) {
  const uint32_t f = (uint32_t)n * c.G;   // (rows x heads: at most 2^26)
  return f > (uint32_t)c.lo && f <= (uint32_t)c.hi ? (int)((f + c.M - 1) / (uint32_t)c.M) : 0;
}

// Tiles of keys that rows at positions p0 .. p1 see some of: 0 .. sink - 1, and the ones from lo on, n
// in all. Positions from `cap` on are not there.
struct PgRange {
  int sink, lo, n;
};
PG_FN PgRange pg_range(int p0, int p1, int cap, const PgCut& c) {
  const int end = pg_min(p1 + 1, cap);
  if (end <= 0) return {0, 0, 0};
  const int hi = pg_up(end, c.KT);
  const int lo = c.window ? pg_min((int)((uint32_t)pg_max(p0 - c.window + 1, 0) / (uint32_t)c.KT), hi) : 0;
  const int sink = pg_min(pg_up(c.sinks, c.KT), lo);
  return {sink, lo, sink + hi - lo};
}
PG_FN int pg_key_tile(const PgRange& r, int t) { return t < r.sink ? t : t - r.sink + r.lo; }

// A bound of pg_range(..).n over the tiles of rows of a sequence with `end` positions.
PG_FN int pg_most(int end, int cap, const PgCut& c) {
  const int all = pg_up(pg_max(pg_min(end, cap), 0), c.KT);
  if (!c.window) return all;
  // M flat rows reach into at most (M - 2) / G + 2 rows
  const int some = pg_up(c.sinks, c.KT) + pg_up(c.window + (int)((uint32_t)(c.M - 2) / c.G) + c.KT, c.KT) + 1;
  return pg_min(some, all);
}

// Tiles of keys in a part, from the sum over the sequences of qtiles x kv x most. A sequence is cut into parts if its
// `most` is over that; the parts of all cut ones are then at most 2 x 2^log (most / part + 1 <= 2 most / part each), their
// tiles of rows at most 2^log.
PG_FN int pg_part(int64_t work, const PgCut& c) {
  const int64_t p = (work + (1ll << c.log) - 1) >> c.log;
  return p < c.least ? c.least : p < PG_MOST ? (int)p : PG_MOST;
}
PG_FN int pg_splits(int most, int part) { return most <= part ? 1 : pg_min(pg_up(most, part), PG_MAXSPLIT); }

// Units of work, at most, as far as the host can tell: a workgroup for each. `shared`: as pg_share divides the sequences, the step
// kernel has the ones of PG_FEW flat rows and, where there are fewer than PG_MANY tiles of 128, also those.
PG_FN int64_t pg_grid(int seqs, int rows, bool one_row, int cap, const PgCut& c) {
  const int64_t G = c.G;
  int64_t tiles = (one_row ? (G + c.M - 1) / c.M * seqs : rows * G / c.M + seqs) * c.kv;
  if (c.shared && c.M == 16) {
    const int64_t some = (int64_t)seqs * c.kv * (PG_FEW / 16) + PG_MANY * (128 / 16);
    tiles = some < tiles ? some : tiles;
  }
  const int64_t cut = tiles * pg_splits(pg_most(cap, cap, c), c.least);
  return cut < tiles + (1 << c.log) ? cut : tiles + (1 << c.log);
}

// Rows of a workgroup of the read kernel: up to 16, and fewer where there would be less than four workgroups for each CU.
PG_FN int pg_read_rows(int rows) { return pg_max(1, pg_min(16, rows / 1024)); }

// Kernels of the paged-cache operators (ill_paged_* in include/ill_hip.h).
//
// A cache is two arrays of pages of 2^page_log positions, keys and values; position t of sequence
// s is slot t % page_size of page table[s][t / page_size]. A batch's new rows are the last ones
// of their sequences. Page numbers outside 0 .. pages - 1 are never followed.
//
// MX: a cache of microscaled e4m3 codes. A page holds [kv heads][page size][D] codes and, `powers_at` bytes on, [kv heads][page size][D / 32]
// powers, so that neighbouring positions of a head are neighbours in memory; page_stride is in bytes. TC is then the
// type that keys and values are multiplied in, the queries'.
#pragma once
#include <type_traits>
#include <utility>
#include "ill_device.h"
#include "ill_lds.h"
#include "ill_mx_codes.h"
#include "ill_paged_plan.h"
#include "ill_values.h"

// A pair of floats in parts of type T, each the rest of the one before: two parts of f16 keep 22 bits, three of bf16 24. Weights
// go to the product with the values as such parts for float32 outputs. For 16-bit outputs they are rounded once, to the cache's
// type: against float64 the outputs are then off by 0.0020 (8000 rows of 28 / 4 heads of 128, bf16), of which their own rounding alone is
// 0.0017; in three parts the call takes 795 us in place of 469.
template <int T>
constexpr int PG_PARTS = T == PG_BF16 ? 3 : 2;
template <int T, int N>
__device__ __forceinline__ void pg_parts2(float a, float b, uint32_t* part) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    part[i] = pg_pack2<T>(a, b);
    float y[2];
    pg_unpack2<T>(part[i], y);
    a -= y[0];
    b -= y[1];
  }
}
// ---- new rows into the cache -------------------------------------------------------------
struct PgAppend {
  PgBatch b;
  const uint8_t *q, *k, *v;   // q null: keys and values only
  uint8_t *qo, *kc, *vc;
  int64_t qs, ks, vs, qos;                          // row strides in elements
  int64_t page_stride, slot_stride, head_stride;    // of the caches, in elements
  const float *bias, *qn, *kn;                      // null: none
  const double* freq;                               // [rot / 2] turns per position
  const int32_t* positions;                         // null: the positions in the sequence
  int32_t heads, kv, rot, interleaved;
  float eps;
  int64_t powers_at;   // MX
};

// The sequence of new row r: the last one whose first row is at most r. One wave; every lane
// returns it (seqs: a row behind the last sequence; -1: one before the first).
__device__ __forceinline__ int pg_seq_of(const PgBatch& b, int r, int lane) {
  int below = 0;
  for (int j0 = 0; j0 <= b.seqs; j0 += 64) {
    const int j = j0 + lane;
    below += __popcll(__ballot(j <= b.seqs && gld(b.row0 + min(j, b.seqs)) <= r));
  }
  return below - 1;
}

__device__ __forceinline__ PgSeq pg_seq_at(const PgBatch& b, int s) {
  const int begin = b.row0 ? gld(b.row0 + s) : s, end = b.row0 ? gld(b.row0 + s + 1) : s + 1;
  return pg_seq(begin, end, gld(b.lens + s), b.rows);
}

// Eight floats from an address aligned to 4 bytes.
__device__ __forceinline__ void pg_floats8(const float* p, float* y) {
  typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));
  const v4u a = *(const GAS v4u*)p, b = *(const GAS v4u*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    y[i] = a[i];
    y[4 + i] = b[i];
  }
}

// A workgroup takes R rows; a thread takes 16 values of one head at a time: the eight first and the
// eight second halves of eight rotated pairs (or eight whole pairs twice where pairs are
// interleaved), so that a pair never leaves its thread and a head's square sum stays within D / 16
// neighbouring lanes. The angles' sines and cosines are computed once per row and pair, from turns
// in float64 (a position of 2^20 has to keep 2^-20 of a turn and more), and shared through LDS. A thread's
// first values are on their way while the rows' places and angles are found, the next ones while it
// computes. One row waits for three loads one after the other (a kernel of 3.5 us), many rows for memory: 343 MB of
// bf16 heads of 128 in 73 us, 4.7 TB/s, where a large copy reaches 5.1.
// MX: 4096 rows of 14 / 2 heads of 64 from float32 11.4 us; the block's largest sizes are found by exchanges between a head's lanes.
template <int TX, int TC, int D, bool MX = false>
__global__ __launch_bounds__(256) void pg_append_kernel(PgAppend a, int R) {
  extern __shared__ __attribute__((aligned(16))) uint8_t pg_lds[];
  constexpr int C = D / 16, EB = TX == PG_F32 ? 4 : 2;   // threads of a head; bytes of a value
  const int half = a.rot >> 1;
  int64_t* place = (int64_t*)pg_lds;             // [R] element offset of the row's slot (MX: byte offset of its page); -1: no sequence's row; -2: it has no place
  int* angle_of = (int*)(place + R);             // [R] position that turns the row
  float2* cs = (float2*)(angle_of + (R + 1) / 2 * 2);   // [R][half]
  int* slot_of = (int*)(cs + R * half);                 // MX: [R]
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, first = blockIdx.x * R;
  const int h0 = a.q ? 0 : a.heads, nh = a.heads + 2 * a.kv - h0, items = R * nh * C;
  struct Item {
    int i, r, head, kind, hk, d[2];   // row of the workgroup's and of the buffers; head of all, of its kind (q, k, v); first dims of the two runs
    bool turn;
  };
  auto item = [&](int it) {
    Item x;
    const uint32_t c = (uint32_t)it % C, v = (uint32_t)it / C;
    if constexpr (MX) {   // queries first, so that few waves have both them and what is quantised
      const uint32_t qs = R * (uint32_t)(a.heads - h0), nk = 2 * a.kv;
      x.i = v < qs ? v / (uint32_t)a.heads : (v - qs) / nk;
      x.head = v < qs ? v - x.i * a.heads : a.heads + (v - qs) - x.i * nk;
    } else {
      x.i = v / (uint32_t)nh;
      x.head = h0 + v - x.i * nh;
    }
    x.r = first + x.i;
    x.kind = x.head < a.heads ? 0 : x.head < a.heads + a.kv ? 1 : 2;
    x.hk = x.head - (x.kind == 0 ? 0 : x.kind == 1 ? a.heads : a.heads + a.kv);
    x.turn = x.kind < 2 && (int)c < a.rot / 16;
    // values keep their order, and so do the dims behind the rotated ones
    const bool split = x.turn && !a.interleaved;
    x.d[0] = split ? 8 * c : 16 * c;
    x.d[1] = x.d[0] + (split ? half : 8);
    return x;
  };
  uint4 raw[2][EB / 2];
  auto fetch = [&](const Item& x) {
    if (x.r >= a.b.rows) return;
    const uint8_t* src = (x.kind == 0 ? a.q : x.kind == 1 ? a.k : a.v) + EB * (x.r * (x.kind == 0 ? a.qs : x.kind == 1 ? a.ks : a.vs) + (int64_t)x.hk * D);
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int n = 0; n < EB / 2; n++) raw[u][n] = gld((const uint4*)(src + EB * x.d[u]) + n);
  };
  Item x = item(tid);
  if (tid < items) fetch(x);
  for (int i = w; i < R; i += 4) {
    const int r = first + i;
    int64_t off = -1;
    int at = 0, slot = 0;
    const int s = r >= a.b.rows ? -1 : a.b.row0 ? pg_seq_of(a.b, r, lane) : r;
    if (s >= 0 && s < a.b.seqs) {
      const PgSeq q = pg_seq_at(a.b, s);
      const int t = q.p0 + (r - q.first);
      at = a.positions ? gld(a.positions + r) : t;
      off = -2;   // (a row without a place in the cache: its query is turned all the same)
      if (t >= 0 && t < pg_cap(a.b)) {
        const int page = gld(a.b.table + s * a.b.table_stride + (t >> a.b.page_log));
        slot = t & ((1 << a.b.page_log) - 1);
        if (page >= 0 && page < a.b.pages) off = page * a.page_stride + (MX ? 0 : slot * a.slot_stride);
      }
    }
    if (lane == 0) {
      if constexpr (MX) slot_of[i] = slot;
      place[i] = off;
      angle_of[i] = at;
    }
  }
  __syncthreads();
  for (int i = tid; i < R * half; i += 256) {
    const double turns = (double)angle_of[i / half] * gld(a.freq + i % half);
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = {c, s};
  }
  __syncthreads();
  for (int it = tid; it < items; it += 256) {
    const Item y = x;
    float v[2][8];
#pragma unroll
    for (int u = 0; u < 2; u++) pg_unpack<TX>(raw[u], v[u]);
    if (it + 256 < items) {
      x = item(it + 256);
      fetch(x);
    }
    const int64_t at = place[y.i];   // (the same for all lanes of a head)
    if (at == -1) {
#pragma unroll
      for (int n = 0; n < 8; n++) v[0][n] = v[1][n] = 0.f;   // (rows past the last were not fetched)
    }
    if (a.bias) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float b[8];
        pg_floats8(a.bias + y.head * D + y.d[u], b);
#pragma unroll
        for (int n = 0; n < 8; n++) v[u][n] += b[n];
      }
    }
    const float* gamma = y.kind == 0 ? a.qn : y.kind == 1 ? a.kn : nullptr;
    if (a.qn || a.kn) {   // (the lanes of a head agree; other heads' lanes take part in the exchange)
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 8; n++) sum = fmaf(v[0][n], v[0][n], fmaf(v[1][n], v[1][n], sum));
#pragma unroll
      for (int m = 1; m < C; m <<= 1) sum += __shfl_xor(sum, m);
      if (gamma) {
        const float inv = 1.f / sqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float g[8];
          pg_floats8(gamma + y.d[u], g);
#pragma unroll
          for (int n = 0; n < 8; n++) v[u][n] *= inv * g[n];
        }
      }
    }
    if (at == -1 || (y.kind > 0 && at < 0)) continue;
    if (y.turn) {
      const float2* row = cs + y.i * half;
      if (a.interleaved) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int n = 0; n < 8; n += 2) {
            const float2 t = row[(y.d[u] + n) >> 1];
            const float p = v[u][n], q = v[u][n + 1];
            v[u][n] = fmaf(p, t.x, -(q * t.y));
            v[u][n + 1] = fmaf(q, t.x, p * t.y);
          }
      } else {
#pragma unroll
        for (int n = 0; n < 8; n++) {
          const float2 t = row[y.d[0] + n];
          const float p = v[0][n], q = v[1][n];
          v[0][n] = fmaf(p, t.x, -(q * t.y));
          v[1][n] = fmaf(q, t.x, p * t.y);
        }
      }
    }
    if constexpr (MX) {
      if (y.kind > 0) {
        // the largest size of each of the head's blocks, over its lanes: each run of eight is part of one block
        uint32_t most[2] = {0, 0}, byte[D / 32];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int n = 0; n < 8; n++) most[u] = max(most[u], __float_as_uint(v[u][n]) & 0x7FFFFFFFu);
#pragma unroll
        for (int b = 0; b < D / 32; b++) {
          uint32_t m = max(y.d[0] >> 5 == b ? most[0] : 0, y.d[1] >> 5 == b ? most[1] : 0);
#pragma unroll
          for (int i = 1; i < C; i <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, i));
          byte[b] = mx_power_of<MX_F8>(m);
        }
        uint8_t* page = (y.kind == 1 ? a.kc : a.vc) + at;
        const int row = (y.hk << a.b.page_log) + slot_of[y.i];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          uint32_t own = byte[0];
#pragma unroll
          for (int b = 1; b < D / 32; b++) own = y.d[u] >> 5 == b ? byte[b] : own;
          const uint2 z = mx_codes<MX_F8>(v[u], own);
          gst((gu32x2*)(page + row * D + y.d[u]), (gu32x2){z.x, z.y});
        }
        if ((it & (C - 1)) == 0) {
          uint8_t* powers = page + a.powers_at + row * (D / 32);
          if constexpr (D == 64) gst((uint16_t*)powers, (uint16_t)(byte[0] | byte[1] << 8));
          else gst((uint32_t*)powers, byte[0] | byte[1] << 8 | byte[2] << 16 | byte[D / 32 - 1] << 24);
        }
        continue;
      }
    }
    uint16_t* dst = y.kind == 0 ? (uint16_t*)a.qo + y.r * a.qos + (int64_t)y.hk * D
                                : (uint16_t*)(y.kind == 1 ? a.kc : a.vc) + at + y.hk * a.head_stride;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint4 z = pg_pack8<TC>(v[u]);
      gst((gu32x4*)(dst + y.d[u]), (gu32x4){z.x, z.y, z.z, z.w});
    }
  }
}

// ---- rows out of the cache -----------------------------------------------------------------
struct PgRead {
  PgBatch b;
  const uint8_t *kc, *vc;
  void *k, *v;
  int64_t ks, vs;                                           // row strides in elements
  int64_t page_stride, slot_stride, head_stride, powers_at;   // as PgAppend's
  int32_t kv;
};

// The batch's rows as append would place them: their keys and values as the cache holds them, zeros where a row has no place. A workgroup
// takes R rows, a thread eight values at a time, neighbours the same row's. Bound by memory: 63000 rows of 8 heads of 128 from a microscaled cache to bf16, 396
// MB, 84 to 93 us.
template <int TO, int TC, bool MX, int D>
__global__ __launch_bounds__(256) void pg_read_kernel(PgRead a, int R) {
  extern __shared__ __attribute__((aligned(16))) uint8_t pg_lds[];
  int64_t* place = (int64_t*)pg_lds;   // [R] element offset of the row's slot (MX: byte offset of its page); -1: no sequence's row; -2: it has no place
  int* slot_of = (int*)(place + R);    // [R]
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, first = blockIdx.x * R;
  // The sequences of a wave's rows one after the other, then their places side by side (a lane a row).
  if (w * 64 < R) {
    const int r = first + w * 64 + lane, rows = min(R - w * 64, 64);
    int s = a.b.row0 ? -1 : r;
    if (a.b.row0) {
      int below = 0;
      for (int j0 = 0; j0 <= a.b.seqs; j0 += 64) {
        const int j = j0 + lane, begin = j <= a.b.seqs ? gld(a.b.row0 + j) : 0x7FFFFFFF;
        for (int i = 0; i < rows; i++) {
          const int n = __popcll(__ballot(j <= a.b.seqs && begin <= first + w * 64 + i));
          if (lane == i) below += n;
        }
      }
      s = below - 1;
    }
    int64_t off = -1;
    int slot = 0;
    if (lane < rows && r < a.b.rows && s >= 0 && s < a.b.seqs) {
      const PgSeq q = pg_seq_at(a.b, s);
      const int t = q.p0 + (r - q.first);
      off = -2;
      if (t >= 0 && t < pg_cap(a.b)) {
        const int page = gld(a.b.table + s * a.b.table_stride + (t >> a.b.page_log));
        slot = t & ((1 << a.b.page_log) - 1);
        if (page >= 0 && page < a.b.pages) off = page * a.page_stride + (MX ? 0 : slot * a.slot_stride);
      }
    }
    if (lane < rows) {
      place[w * 64 + lane] = off;
      slot_of[w * 64 + lane] = slot;
    }
  }
  __syncthreads();
  constexpr int C = D / 8;
  const uint32_t each = 2 * a.kv * C;   // of a row: keys, then values
  for (uint32_t it = tid; it < R * each; it += 256) {
    const uint32_t i = it / each, x = it - i * each, head = x / C, d = 8 * (x - head * C);   // (of both, keys' heads first)
    const int64_t at = place[i];
    if (at == -1) continue;
    const bool value = head >= (uint32_t)a.kv;
    const int h = head - (value ? a.kv : 0);
    const uint8_t* cache = value ? a.vc : a.kc;
    float y[8] = {};
    uint4 raw = {0, 0, 0, 0};
    if (at >= 0) {
      if constexpr (MX) {
        const int row = (h << a.b.page_log) + slot_of[i];
        mx_values<MX_F8>(gld((const uint2*)(cache + at + row * D + d)), gld(cache + at + a.powers_at + row * (D / 32) + (d >> 5)), y);
      } else {
        raw = gld((const uint4*)((const uint16_t*)cache + at + h * a.head_stride + d));
        pg_unpack<TC>(&raw, y);
      }
    }
    const int64_t to = (int64_t)(first + i) * (value ? a.vs : a.ks) + h * D + d;
    void* out = value ? a.v : a.k;
    if constexpr (TO == PG_F32) {
      gst((gu32x4*)((float*)out + to), (gu32x4){__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])});
      gst((gu32x4*)((float*)out + to + 4), (gu32x4){__float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7])});
    } else {
      const uint4 z = MX ? pg_pack8<TO>(y) : raw;   // (a 16-bit cache's values in its own type: as they are)
      gst((gu32x4*)((uint16_t*)out + to), (gu32x4){z.x, z.y, z.z, z.w});
    }
  }
}

// ---- attention over the cache ------------------------------------------------------------
struct PgAttend {
  PgBatch b;
  const uint16_t *q, *kc, *vc;
  void* out;
  int64_t qs, os;                                   // row strides in elements
  int64_t page_stride, slot_stride, head_stride;
  int32_t heads, kv, window, sinks, out_f32;
  float scale;
  int64_t powers_at;   // MX
};

// What the unit of work u is: a part of the keys for a tile of rows of one key/value head.
struct PgUnit {
  int s, head, q, split, splits, part_at, tile_at;   // part_at, tile_at: its places in the workspace, if it is one of several parts
  PgSeq seq;
};

// The same unit, held as values that the compiler knows to be every lane's.
__device__ __forceinline__ PgUnit pg_uniform(const PgUnit& u) {
  auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  return {one(u.s), one(u.head), one(u.q), one(u.split), one(u.splits), one(u.part_at), one(u.tile_at), {one(u.seq.first), one(u.seq.n), one(u.seq.p0)}};
}

// Workgroups of attention: waves and threads, for the kernels and their launches.
constexpr int PG_WAVES = 4, PG_THREADS = 64 * PG_WAVES;

// What launching the units of many keys first takes in LDS: the units of the waves' sequences, by their keys.
template <bool LONGEST>
struct PgClasses {
  int4 classes[PG_WAVES];
};
template <>
struct PgClasses<false> {};

// The division of a call's work, found by every workgroup from the lengths: sequence s is thread s % NT's. LONGEST: of up to 256 sequences
// the units of many keys are launched first (microscaled caches: a constant, as asking it of every call costs the kernels of 16-bit ones 3 to
// 12 spilled scalar registers).
template <bool LONGEST>
struct PgFinder {
  static constexpr int NW = PG_WAVES, NT = PG_THREADS;
  const PgBatch& b;
  PgCut c;
  int part, units;   // tiles of keys in a part; units of work in all
  const int grid;    // workgroups that the launch has for them
  struct Lds : PgClasses<LONGEST> {
    int64_t tiles[NW], work[NW];
    int units[NW], parts[NW], cut[NW];
    PgUnit found;
  };
  Lds& lds;

  PgSeq q;
  int most, n;   // the rows of sequence `threadIdx.x` (of one sequence: every thread's), a bound of their tiles of keys, their tiles x heads

  __device__ __forceinline__ void look(int s) {
    q = {0, 0, 0};
    most = n = 0;
    if (s >= b.seqs) return;
    q = pg_seq_at(b, s);
    most = pg_most(q.p0 + q.n, pg_cap(b), c);
    n = pg_qtiles(q.n, c) * (int)c.kv;
  }
  template <class T>
  static __device__ __forceinline__ T over_wave(T v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
  }
  __device__ __forceinline__ PgFinder(const PgBatch& b_, const PgCut& c_, int grid_, Lds& lds_) : b(b_), c(c_), grid(grid_), lds(lds_) {
    if (b.seqs == 1) {   // (one sequence is one kernel's: shared is 0)
      look(0);
      part = pg_part((int64_t)n * most, c);
      units = n * pg_splits(most, part);
      whole_if_more();
      return;
    }
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int64_t tiles = 0, work = 0;
    int s;
    if (c.shared) {
      for (s = threadIdx.x; s < b.seqs; s += NT) tiles += pg_prompt_tiles(pg_seq_at(b, s).n, c.G, c.kv);
      tiles = over_wave(tiles);
      if (lane == 0) lds.tiles[w] = tiles;
      __syncthreads();
      tiles = 0;
#pragma unroll
      for (int i = 0; i < NW; i++) tiles += lds.tiles[i];
      pg_share(c, tiles);
      tiles = 0;
      __syncthreads();
    }
    s = threadIdx.x;
    do {
      look(s);
      tiles += n;
      work += (int64_t)n * most;
      s += NT;
    } while (s - (int)threadIdx.x < b.seqs);
    tiles = over_wave(tiles);
    work = over_wave(work);
    if (lane == 0) {
      lds.tiles[w] = tiles;
      lds.work[w] = work;
    }
    __syncthreads();
    tiles = work = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
      tiles += lds.tiles[i];
      work += lds.work[i];
    }
    part = pg_part(work, c);
    units = (int)min(tiles, (int64_t)PG_MOST);   // of uncut sequences: a unit for each. (As many only where row0 does not ascend.)
    int u = 0;
    for (s = threadIdx.x; s - (int)threadIdx.x < b.seqs; s += NT) {
      if (b.seqs > NT) look(s);
      u += n * (pg_splits(most, part) - 1);
    }
    u = over_wave(u);
    if (lane == 0) lds.units[w] = u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; i++) units += lds.units[i];
    whole_if_more();
  }
  // The launch has a workgroup for each unit if row0 ascends. If not, nothing is cut: no part waits in vain for another.
  __device__ __forceinline__ void whole_if_more() {
    if (units > grid) part = PG_MOST;
  }

  // Unit u of sequence s: u is counted from the sequence's first, parts and tiles are what the sequences before it have.
  __device__ __forceinline__ PgUnit unit(uint32_t u, int s, uint32_t splits, int parts, int tiles) const {
    // the heads in turn, so that the workgroups of an XCD (every eighth) read few heads; of a head, the
    // parts of its last rows first, which have the most keys
    const uint32_t qt = (uint32_t)n / c.kv, v = u / c.kv, head = u - v * c.kv, back = splits == 1 ? v : v / splits, at = qt - 1 - back;
    const int tile = (int)(head * qt + at);
    return {s, (int)head, (int)at, (int)(v - back * splits), (int)splits, parts + tile * (int)splits, tiles + tile, q};
  }
  __device__ __forceinline__ PgUnit find(int u) {
    if (b.seqs == 1) return unit(u, 0, pg_splits(most, part), 0, 0);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int before = 0, parts = 0, tiles = 0;
    if (threadIdx.x == 0) lds.found.seq.n = 0;   // (stays so only where lengths change meanwhile)
    for (int s0 = 0; s0 < b.seqs; s0 += NT) {
      if (b.seqs > NT) look(s0 + threadIdx.x);
      const int splits = pg_splits(most, part);
      int3 sum = {n * splits, splits > 1 ? n * splits : 0, splits > 1 ? n : 0}, own = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int x = __shfl_up(sum.x, m), y = __shfl_up(sum.y, m), z = __shfl_up(sum.z, m);
        if (lane >= m) {
          sum.x += x;
          sum.y += y;
          sum.z += z;
        }
      }
      __syncthreads();
      if (lane == 63) {
        lds.units[w] = sum.x;
        lds.parts[w] = sum.y;
        lds.cut[w] = sum.z;
      }
      __syncthreads();
      int first = before + sum.x - own.x, y = parts + sum.y - own.y, z = tiles + sum.z - own.z;
#pragma unroll
      for (int i = 0; i < NW; i++) {
        const int x = lds.units[i], p = lds.parts[i], t = lds.cut[i];
        if (i < w) {
          first += x;
          y += p;
          z += t;
        }
        before += x;
        parts += p;
        tiles += t;
      }
      if constexpr (LONGEST) {
        if (b.seqs <= NT) {   // (then this is the only turn) the units of the most keys first, in four classes
          const int keys = own.x ? pg_up(most, splits) : 0, of = 2 * keys > part ? 0 : 4 * keys > part ? 1 : 8 * keys > part ? 2 : 3;
          int4 up = {of == 0 ? own.x : 0, of == 1 ? own.x : 0, of == 2 ? own.x : 0, of == 3 ? own.x : 0};
#pragma unroll
          for (int m = 1; m < 64; m <<= 1) {
            const int4 o = {__shfl_up(up.x, m), __shfl_up(up.y, m), __shfl_up(up.z, m), __shfl_up(up.w, m)};
            if (lane >= m) {
              up.x += o.x;
              up.y += o.y;
              up.z += o.z;
              up.w += o.w;
            }
          }
          if (lane == 63) lds.classes[w] = up;
          __syncthreads();
          int4 all = {0, 0, 0, 0}, here = up;   // (here: with the waves before)
#pragma unroll
          for (int i = 0; i < NW; i++) {
            const int4 o = lds.classes[i];
            all = {all.x + o.x, all.y + o.y, all.z + o.z, all.w + o.w};
            if (i < w) here = {here.x + o.x, here.y + o.y, here.z + o.z, here.w + o.w};
          }
          first = (of == 0 ? here.x : of == 1 ? all.x + here.y : of == 2 ? all.x + all.y + here.z : all.x + all.y + all.z + here.w) - own.x;
        }
      }
      if (u >= first && u < first + own.x) lds.found = unit(u - first, s0 + threadIdx.x, splits, y, z);
      if (u < before) break;
    }
    __syncthreads();
    return lds.found;
  }
};

template <int TC>
__device__ __forceinline__ v4f pg_mfma16(uint4 a, uint4 b, v4f c) {   // 16 x 16 x 32
  if constexpr (TC == PG_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Where the 16-byte unit u of key `key` of a tile lies in LDS, in units: a key's units in a row, permuted so that the
// eight keys of an eighth of an operand read, and the 4 keys x 64 bytes of half a transposed read, are on different banks.
template <int D>
__device__ __forceinline__ int pg_swz(int key) {
  return D == 64 ? ((key & 2) << 1) | ((key >> 2) & 2) | ((key >> 4) & 1) : ((key & 3) << 2) | ((key >> 2) & 2) | ((key >> 4) & 1);
}
template <int D>
__device__ __forceinline__ int pg_unit_at(int key, int u) { return key * (D / 8) + (u ^ pg_swz<D>(key)); }

typedef LAS gu32x4 pg_lds4;   // 16 bytes of a tile
__device__ __forceinline__ uint4 pg_get(const LAS uint8_t* p) {
  const gu32x4 x = *(const pg_lds4*)p;
  return {x[0], x[1], x[2], x[3]};
}
// Keys key .. key + 7 of dim d0 + i, d0 a multiple of 16, from the rows of a tile of values; `p` is where pg_values_at says.
// Each 16 lanes read 4 keys x 16 dims twice, and the transposing read hands lane i its dim.
__device__ __forceinline__ uint2 pg_tr(const LAS uint8_t* p) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LAS v4s*)p));
}
template <int D>
__device__ __forceinline__ uint4 pg_values(const LAS uint8_t* p) {
  const uint2 a = pg_tr(p), b = pg_tr(p + 4 * 2 * D);   // (the permutation ignores bit 2 of the key)
  return {a.x, a.y, b.x, b.y};
}
template <int D>
__device__ __forceinline__ int pg_values_at(int key, int d0, int i) {
  return 16 * pg_unit_at<D>(key + (i >> 2), d0 / 8 + ((i >> 1) & 1)) + 8 * (i & 1);
}

// Infinities and NaN of eight values: whether there are any; the values with zeros in their place; and marks
// that a product with ones for the keys a row sees adds up (1 for inf, 2^7 for -inf, 2^14 for NaN; at most 64 keys).
template <int TC>
__device__ __forceinline__ uint32_t pg_wild2(uint32_t x) {   // the top bit of each half: its exponent is all ones
  constexpr uint32_t E = TC == PG_BF16 ? 0x7F807F80u : 0x7C007C00u, STEP = TC == PG_BF16 ? 0x00800080u : 0x04000400u;
  return ((x & E) + STEP) & 0x80008000u;
}
template <int TC>
__device__ __forceinline__ uint32_t pg_wild(uint4 v) {
  return pg_wild2<TC>(v.x) | pg_wild2<TC>(v.y) | pg_wild2<TC>(v.z) | pg_wild2<TC>(v.w);
}
template <int TC>
__device__ __forceinline__ uint4 pg_tamed(uint4 v, uint4& marks) {
  constexpr uint32_t ONE = TC == PG_BF16 ? 0x3F803F80u : 0x3C003C00u, STEP = TC == PG_BF16 ? 0x03800380u : 0x1C001C00u;   // 1, and a factor of 2^7
  constexpr uint32_t S = TC == PG_BF16 ? 0x007F007Fu : 0x03FF03FFu;
  auto all = [](uint32_t top) { return top | (top - (top >> 15)); };   // all bits of the halves whose top bit is set
  uint32_t y[4] = {v.x, v.y, v.z, v.w}, k[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t wild = all(pg_wild2<TC>(y[i])), nan = all(((y[i] & S) + (0x80008000u - 0x00010001u)) & 0x80008000u);
    k[i] = wild & (ONE + (nan & 2 * STEP) + (~nan & all(y[i] & 0x80008000u) & STEP));
    y[i] &= ~wild;
  }
  marks = {k[0], k[1], k[2], k[3]};
  return {y[0], y[1], y[2], y[3]};
}
// Whether a tile of N units has any, for the whole wave.
template <int TC, int N>
__device__ __forceinline__ bool pg_wild_tile(const LAS uint8_t* v, int lane) {
  uint32_t w = 0;
#pragma unroll 2
  for (int i = lane; i < N; i += 64) w |= pg_wild<TC>(pg_get(v + 16 * i));
  return __any(w != 0);
}
// Ones for the keys of eight bits.
template <int TC>
__device__ __forceinline__ uint4 pg_ones(uint32_t seen) {
  constexpr uint32_t ONE = TC == PG_BF16 ? 0x3F80u : 0x3C00u;
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = (seen >> (2 * i) & 1 ? ONE : 0u) | (seen >> (2 * i + 1) & 1 ? ONE << 16 : 0u);
  return {y[0], y[1], y[2], y[3]};
}
// Tiles that all rows see go to the product as they are. An infinity or NaN there makes its sums infinite or NaN, whatever
// its weight is, but not the right one: a weight's lesser parts may be 0 or negative, and a small weight rounds to 0. So a wave
// (the prompt kernel: a workgroup) that ends with such a sum evaluates its keys once more, and then sets them aside in every tile.
// Finite values pay for the look at the sums and a barrier: 8000 rows of 28 / 4 heads of 128, 449 -> 454 us; 200 single rows
// in a window 24.2 -> 24.4.
template <int N, class V>
__device__ __forceinline__ bool pg_any_wild(const V* sums) {   // of the wave's
  float z[4] = {};
#pragma unroll
  for (int d = 0; d < N; d++)
#pragma unroll
    for (int r = 0; r < (int)(sizeof(V) / 4); r++) z[r & 3] = fmaf(sums[d][r], 0.f, z[r & 3]);
  const float y = (z[0] + z[1]) + (z[2] + z[3]);
  return __any(y != y);
}
// The factor by which sums to reference `from` are moved to `to`, which is not below it; never 0, so that infinite sums stay
// what they are where it underflows. (The exponential ends at 2^-126: 2^-149, the least number, is no further off.)
__device__ __forceinline__ float pg_moved(float from, float to) {
  return to == -INFINITY ? 1.f : fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-149f);
}
__device__ __forceinline__ float pg_wild_sum(float marks) {
  const int n = (int)marks;
  float y = n & 127 ? INFINITY : 0.f;
  if (n >> 7 & 127) y -= INFINITY;
  return n >> 14 ? NAN : y;
}

// The exponents' reference of a row follows its greatest score, PG_UP below it, and is moved only when a score
// passes it by more than PG_UP + PG_SLACK. For f16 weights then stay below 2^15, in its range: one rounding keeps their 11 bits
// down to 2^-24 of the greatest one, two parts (float32 outputs) 22 bits down to 2^-13 of it, and 2^-35 of it below that. bf16
// has float32's range: weights up to 1, so that sums overflow only where a softmax with its greatest weight at 1 does too (with
// the greatest at 2^10, 34 even values of 1e34 overflowed).
#define PG_SLACK 5.f
template <int TC>
constexpr float PG_UP = TC == PG_BF16 ? -PG_SLACK : 10.f;

struct PgWork {        // a call's share of the handle's workspace
  float2* ml;          // [2 x 2^log][M] reference and sum of a part's rows
  float* o;            // [2 x 2^log][M][D] its weighted values
  int32_t* joined;     // [2^log][1 + PG_MAXSPLIT / PG_FAN] parts of a tile of rows that are done, in all and of each PG_FAN; 0 between calls
};

// Four dims of a row's output.
template <int TC>
__device__ __forceinline__ void pg_store(const PgAttend& a, int row, int head, int d, int D, v4f y) {
  const int64_t at = row * a.os + (int64_t)head * D + d;
  if (a.out_f32) gst((gu32x4*)((float*)a.out + at), __builtin_bit_cast(gu32x4, y));
  else gst((gu32x2*)((uint16_t*)a.out + at), (gu32x2){pg_pack2<TC>(y[0], y[1]), pg_pack2<TC>(y[2], y[3])});
}

// Parts are written and read with agent-scope accesses, which go through to where all XCDs see them: a workgroup only has
// to wait until its own stores are acknowledged. (An agent-scope release instead writes the XCD's whole L2 back: 333 rows of
// 14 heads took 41 us with it, 18 us without.)
__device__ __forceinline__ void pg_share(float* p, v4f v) {
  const gu32x4 x = __builtin_bit_cast(gu32x4, v);
  astore64((uint64_t*)p, (uint64_t)x[0] | (uint64_t)x[1] << 32);
  astore64((uint64_t*)p + 1, (uint64_t)x[2] | (uint64_t)x[3] << 32);
}
__device__ __forceinline__ v4f pg_shared(const float* p) {
  const uint64_t x = aload64((const uint64_t*)p), y = aload64((const uint64_t*)p + 1);
  return (v4f){__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32)), __uint_as_float((uint32_t)y), __uint_as_float((uint32_t)(y >> 32))};
}

// Whether this is the last of `count` workgroups to come here, whose parts it then sees (the same for every thread). The
// counter is left at 0 for the next call.
__device__ __forceinline__ bool pg_last(int32_t* counter, int count, int* lds) {
  PG_WAIT(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool all = __hip_atomic_fetch_add((GAS int32_t*)counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
    if (all) astore32(counter, 0);
    *lds = all;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*lds) != 0;
}

// Writes a part's state of row r, four dims from d on.
template <int D, int M>
__device__ __forceinline__ void pg_put_part(const PgWork& w, int part, int r, int d, float m, float l, v4f o) {
  const size_t at = (size_t)part * M + r;
  if (d == 0) astore64((uint64_t*)(w.ml + at), (uint64_t)__float_as_uint(m) | (uint64_t)__float_as_uint(l) << 32);
  pg_share(w.o + at * D + d, o);
}

static_assert(PG_FAN * PG_FAN >= PG_MAXSPLIT, "two steps");
// What pg_join takes of LDS for tiles of M rows, in place of the tiles of keys and values, which nobody reads any more.
template <int M>
struct PgJoinLds {
  __attribute__((aligned(16))) float weights[PG_FAN * M], sums[PG_FAN * M], rows[2 * M];   // of each part's rows; of the rows joined: reference and sum
  v4f part[PG_THREADS - PG_THREADS / 4];   // states of all groups of threads but the first, up to four groups
};
// Joins `count` <= PG_FAN parts (from part `first` on, every step-th) of a tile of rows in their order, by one workgroup:
// into the output, or into the first of them.
template <int TC, int D, int M>
__device__ __forceinline__ void pg_join(const PgAttend& a, const PgCut& c, const PgWork& pw, const PgUnit& un, int first, int step, int count, bool out,
                                        int f0, int live, PgJoinLds<M>& lds) {
  constexpr int NT = PG_THREADS, T = NT / M >= 64 ? 64 : NT / M < 1 ? 1 : NT / M;   // T threads of a row, neighbours in a wave
  const int tid = threadIdx.x;
  LAS float *wt = (LAS float*)lds.weights, *ls = (LAS float*)lds.sums, *rows = (LAS float*)lds.rows;
  // few items (four dims of a row): `groups` threads each, every groups-th part to one of them, its values fetched along
  // with the statistics
  const int items = live * (D / 4), groups = items <= NT / 4 ? 4 : items <= NT / 2 ? 2 : 1, width = NT / groups;
  const int g = tid / width, i_first = tid % width;
  auto part_of = [&](int i, int x) { return pw.o + ((size_t)(first + x * step) * M + i / (D / 4)) * D + 4 * (i % (D / 4)); };
  v4f ahead[PG_FAN / 2];
  if (groups > 1)
#pragma unroll
    for (int u = 0; u < PG_FAN / 2; u++)
      if (g + u * groups < count && i_first < items) ahead[u] = pg_shared(part_of(i_first, g + u * groups));
  for (int i = tid; i < count * M; i += NT) {
    const int x = i / M, r = i % M;
    const uint64_t v = r < live ? aload64((const uint64_t*)(pw.ml + (size_t)(first + x * step) * M + r)) : 0;
    wt[i] = __uint_as_float((uint32_t)v);
    ls[i] = __uint_as_float((uint32_t)(v >> 32));
  }
  __syncthreads();
  if (tid < M * T) {
    const int r = tid / T, j = tid % T;
    float m = -INFINITY, l = 0.f;
    for (int x = j; x < count; x += T) m = fmaxf(m, wt[x * M + r]);
#pragma unroll
    for (int k = 1; k < T; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
    for (int x = j; x < count; x += T) {
      const float e = pg_moved(wt[x * M + r], m);
      wt[x * M + r] = e;
      l += ls[x * M + r] * e;
    }
#pragma unroll
    for (int k = 1; k < T; k <<= 1) l += __shfl_xor(l, k);
    if (j == 0) {
      rows[r] = m;
      rows[M + r] = l;
    }
  }
  __syncthreads();
  for (int i = i_first; i - i_first < items; i += width) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    v4f y = {0.f, 0.f, 0.f, 0.f};
    if (i < items) {
      if (groups > 1) {
#pragma unroll
        for (int u = 0; u < PG_FAN / 2; u++)
          if (g + u * groups < count) y += ahead[u] * wt[(g + u * groups) * M + r];
      } else {
#pragma unroll 8
        for (int x = 0; x < count; x++) y += pg_shared(part_of(i, x)) * wt[x * M + r];
      }
    }
    if (groups > 1) {   // (items <= width: once)
      LAS v4f* sums = (LAS v4f*)lds.part;
      if (g && i < items) sums[(g - 1) * width + i] = y;
      __syncthreads();
      if (g == 0 && i < items)
        for (int x = 1; x < groups; x++) y += sums[(x - 1) * width + i];
    }
    if (g == 0 && i < items) {
      const float m = rows[r], l = rows[M + r];
      if (out) pg_store<TC>(a, un.seq.first + (uint32_t)(f0 + r) / c.G, un.head * c.G + (uint32_t)(f0 + r) % c.G, d, D, l == 0.f ? (v4f){0.f, 0.f, 0.f, 0.f} : y / l);
      else pg_put_part<D, M>(pw, first, r, d, m, l, y);
    }
  }
}

// What follows a part of several: the last workgroup of PG_FAN parts joins them, and the last of those joins theirs.
template <int TC, int D, int M>
__device__ __forceinline__ void pg_finish(const PgAttend& a, const PgCut& c, const PgWork& w, const PgUnit& un, int f0, int live, PgJoinLds<M>& lds, int* last) {
  const int g = un.split / PG_FAN, groups = pg_up(un.splits, PG_FAN);
  int32_t* joined = w.joined + un.tile_at * (PG_MAXSPLIT / PG_FAN + 1);
  int first = un.part_at + g * PG_FAN, step = 1, count = min(PG_FAN, un.splits - g * PG_FAN);
  int32_t* counter = joined + 1 + g;
  for (bool out = groups == 1;; out = true) {   // (once or twice)
    if (!pg_last(counter, count, last)) return;
    pg_join<TC, D, M>(a, c, w, un, first, step, count, out, f0, live, lds);
    if (out) return;
    first = un.part_at;
    step = PG_FAN;
    count = groups;
    counter = joined;
  }
}

struct PgStep {
  PgAttend a;
  PgCut c;
  PgWork w;
};

// Attention of few rows per sequence. A workgroup of four waves takes a part of the keys for 16 flat rows of a
// key/value head, and each wave every fourth tile of keys of it: 8 KB of keys and 8 KB of values at a time go
// straight into the wave's own LDS, so that the waves never wait for each other; the next tile's keys start
// as soon as this one's have been read, its values after this one's. Scores are keys x rows and outputs dims
// x rows (v_mfma 16 x 16 x 32), so a row's statistics are its lanes' own, and the keys are dealt to the score
// products' rows such that a lane's weights are the next product's operand as they stand (block b, row 4 g
// + r: key 32 (b / 2) + 8 g + 4 (b % 2) + r). Values are transposed by the LDS read. The waves' states are
// joined in LDS; a tile of rows whose keys are in several parts is joined by the workgroup that ends last, in
// the parts' order.
// Bound by memory where there is enough of it: 64 sequences of 100 to 9000 positions, 32 / 8 heads of 128, 432 MB in 97 us,
// 4.4 TB/s (a large copy: 5.1). One sequence of 131071, 14 / 2 heads of 64, 67 MB in 19.6 us: 13 at the copy's rate, the rest the
// launch, three dependent loads at the start (3) and the join. One of 500: 6.5 us, all latency.
// MX: codes are multiplied as values of type TC, keys converted in the registers that they come in, values on their way into LDS; the scores' and the
// weights' keys are dealt so that a load has 16 neighbours. The 64 sequences, 220 MB, take 57 us, 3.9 TB/s (64 of 4000: 5.5), the long one 17.7.
// Two workgroups to a CU: with three the 168 registers spill inside the loop (94 us).
template <bool MX>
struct PgStepLds {
  static constexpr int UNITS = MX ? 544 : 1024;   // of a wave: keys and values of a tile, 8 KB each (MX: values); its state, 16 x (D + 4) floats
  union {
    __attribute__((aligned(16))) uint4 lds[PG_WAVES][UNITS];
    PgJoinLds<16> join;
  };
  float smx[PG_WAVES][16], sls[PG_WAVES][16];
  int last;
  typename PgFinder<MX>::Lds found;
};
template <int TC, int D, bool FINE, bool MX>   // FINE: weights in parts that keep float32 (float32 outputs)
__device__ __forceinline__ void pg_step(const PgStep& p, int block, int grid, PgStepLds<MX>& shared) {
  constexpr int NW = PG_WAVES, KT = D == 64 ? 64 : 32, UPR = D / 8, KPI = 64 / UPR, NB = KT / 16, KS = D / 32, ND = D / 16, NS = KT / 32, NG = KT / 16;
  constexpr int N = FINE ? PG_PARTS<TC> : 1;   // parts of a weight
  constexpr int RF = D + 4;   // floats between the rows of a state in LDS
  auto &lds = shared.lds;
  auto &smx = shared.smx, &sls = shared.sls;
  const PgAttend& a = p.a;
  PgCut c = p.c;
  c.M = 16;   // (as the host has them, for the compiler)
  c.KT = KT;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int cap = pg_cap(a.b), pmask = (1 << a.b.page_log) - 1;
  LAS uint8_t* kl = (LAS uint8_t*)lds[w];
  LAS uint8_t* vl = MX ? kl : kl + 8192;
  const uint32_t mine_lds = pg_lds_at(lds[w]);
  constexpr std::integral_constant<int, 0> KEYS{};
  constexpr std::integral_constant<int, 8192> VALUES{};
  // this lane's operands in a tile: of the keys for each 32 dims, of the values for each 16. Other keys of the lane's are
  // whole multiples of 4 or 32 rows further: the permutation does not see them.
  int ka[KS], va[ND];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) ka[ks] = 16 * pg_unit_at<D>(8 * (n >> 2) + (n & 3), 4 * ks + kg);
#pragma unroll
  for (int d = 0; d < ND; d++) {
    const int key = 4 * kg + (n >> 2), u = 2 * d + (n >> 1 & 1);
    va[d] = MX ? 16 * (key * UPR + (u ^ (D == 64 ? key & 6 : (key & 7) << 1))) + 8 * (n & 1) : pg_values_at<D>(8 * kg, 16 * d, n);
  }
  const float sc2 = a.scale * 1.4426950408889634f;
  PgFinder<MX> finder(a.b, c, grid, shared.found);
  auto over_kg = [](float v, auto op) {   // over the lanes of the same row
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = op(__int_as_float((int)x[0]), __int_as_float((int)x[1]));
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return op(__int_as_float((int)y[0]), __int_as_float((int)y[1]));
  };
  uint32_t lane_off[8];   // bytes from a group of 16 keys to what this lane loads of it, per load
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int key = KPI * i + lane / UPR;
    lane_off[i] = 2 * ((uint32_t)(key & 15) * (uint32_t)a.slot_stride + 8 * ((lane % UPR) ^ pg_swz<D>(key)));
  }
  if (block >= __builtin_amdgcn_readfirstlane(finder.units)) return;
  const PgUnit un = pg_uniform(finder.find(block));
  if (un.seq.n == 0) return;
  const int G = c.G, flat = un.seq.n * G, f0 = 16 * un.q, live = min(16, flat - f0);   // (n G is at most 2^26)
  const uint32_t f = min(f0 + n, flat - 1), at_row = f / c.G;
  const int row = un.seq.first + at_row, head = un.head * G + (f - at_row * c.G);
  const int pos = un.seq.p0 + at_row, p0 = __builtin_amdgcn_readlane(pos, 0), p1 = __builtin_amdgcn_readlane(pos, 15);
  const PgRange range = pg_range(p0, p1, cap, c);
  const int per = pg_up(range.n, un.splits), c0 = min(un.split * per, range.n), c1 = min(c0 + per, range.n);
  const int end = min(p1 + 1, cap);
  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) qf[ks] = gld((const uint4*)(a.q + row * a.qs + (int64_t)head * D + (MX ? 64 * (ks >> 1) + 16 * kg + 8 * (ks & 1) : 32 * ks + 8 * kg)));
  const int mine = c0 + w < c1 ? (c1 - c0 - w + NW - 1) / NW : 0;   // this wave's tiles
  // where the keys of the wave's next 64 / NG tiles are, 16 of them a lane: elements from the cache's begin; -1: not there
  int64_t group = -1;
  auto groups = [&](int k) {
    const int t = c0 + w + NW * (k + lane / NG);
    group = -1;
    if (t < c1) {
      const int g = pg_key_tile(range, t) * KT + 16 * (lane % NG), key = min(g, end - 1);
      const int page = gld(a.b.table + un.s * a.b.table_stride + (key >> a.b.page_log));
      if (page >= 0 && page < a.b.pages) group = page * a.page_stride + (MX ? 0 : (g & pmask) * a.slot_stride + un.head * a.head_stride);
    }
  };
  auto group_at = [&](int k, int g) {   // (the same for every lane)
    const int at = (k * NG + g) & 63;
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)group, at) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(group >> 32), at) << 32);
  };
  auto load = [&](const uint16_t* from, auto to, int k) {
    pg_each<NG>([&](auto g) {
      const int64_t at = group_at(k, g);
      const uint16_t* base = from + (at < 0 ? 0 : at);   // (the first page is there, and masked)
      pg_each<8 / NG>([&](auto i) {
        constexpr int I = g * 8 / NG + i;
        pg_dma16<to + 1024 * I>(base, lane_off[I], mine_lds);
      });
    });
  };
  // MX: a tile's codes and powers come through registers, the next tile's as soon as this one's have been used; the values go on into LDS as 16-bit
  // ones. A lane's codes of a key are 16 dims of 64 at a time (the products' dims are dealt the same way to queries and keys), block b's
  // keys are 16 b + n: a load has neighbouring keys of one page.
  uint4 kreg[NB][D / 64], vreg[4];
  uint32_t kpow[NB], vpow[4];
  auto mx_group = [&](const void* cache, int k, int g, const uint8_t*& powers) {   // where a group's codes and powers are (behind the last tile: the first page's, which are there)
    const int64_t at = group_at(k, g), page = k < mine && at > 0 ? at : 0;
    const int slot = (un.head << a.b.page_log) + (k < mine ? (pg_key_tile(range, c0 + w + NW * k) * KT + 16 * g) & pmask : 0);
    powers = (const uint8_t*)cache + page + a.powers_at + slot * (D / 32);
    return (const uint8_t*)cache + page + slot * D;
  };
  auto mx_keys = [&](int k) {
    pg_each<NB>([&](auto b) {
      const uint8_t *powers, *codes = mx_group(a.kc, k, b, powers);
#pragma unroll
      for (int j = 0; j < D / 64; j++) kreg[b][j] = gld((const uint4*)(codes + (uint32_t)(D * n + 16 * kg) + 64 * j));
      if constexpr (D == 64) kpow[b] = gld(powers + (uint32_t)(2 * n + (kg >> 1)));
      else kpow[b] = gld((const uint32_t*)(powers + (uint32_t)(4 * n)));
    });
  };
  constexpr int VL = 16 * D / 1024, LPK = D / 16;   // loads of a group's values; lanes of a key
  auto mx_vals = [&](int k) {
    pg_each<NG>([&](auto g) {
      const uint8_t *powers, *codes = mx_group(a.vc, k, g, powers);
#pragma unroll
      for (int j = 0; j < VL; j++) {
        vreg[VL * g + j] = gld((const uint4*)(codes + (uint32_t)(16 * lane) + 1024 * j));
        vpow[VL * g + j] = gld(powers + (uint32_t)((D / 32) * (lane / LPK) + (lane % LPK >> 1)) + 32 * j);
      }
    });
  };
  // Where the 16 bytes u of a key's values lie: the 16 keys x 32 bytes of a transposed read are on different banks.
  auto mx_unit = [](int key, int u) { return 16 * (key * UPR + (u ^ (D == 64 ? key & 6 : (key & 7) << 1))); };
  auto mx_put = [&] {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int key = 64 / LPK * i + lane / LPK, u = 2 * (lane % LPK);
      const uint4 lo = mx_16<TC, MX_F8>({vreg[i].x, vreg[i].y}, vpow[i]), hi = mx_16<TC, MX_F8>({vreg[i].z, vreg[i].w}, vpow[i]);
      *(pg_lds4*)(vl + mx_unit(key, u)) = (gu32x4){lo.x, lo.y, lo.z, lo.w};
      *(pg_lds4*)(vl + mx_unit(key, u + 1)) = (gu32x4){hi.x, hi.y, hi.z, hi.w};
    }
  };
  // This lane's operand of 32 keys' values, 16 dims: keys 4 kg .. and 16 + 4 kg .., as its weights are.
  auto values = [&](int d, int t) {
    if constexpr (MX) {
      const uint2 x = pg_tr(vl + va[d] + 32 * t * 2 * D), y = pg_tr(vl + va[d] + (32 * t + 16) * 2 * D);
      return uint4{x.x, x.y, y.x, y.y};
    } else {
      return pg_values<D>(vl + va[d] + 32 * t * 2 * D);
    }
  };
  float Mx, Ls;   // Ls: this lane's keys only
  v4f O[ND];
  for (bool careful = false;; careful = true) {   // (twice only for infinities and NaN, pg_any_wild)
    Mx = -INFINITY;
    Ls = 0.f;
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] = (v4f){0.f, 0.f, 0.f, 0.f};
    groups(0);
    PG_WAIT_OWN();
    if constexpr (MX) {
      mx_keys(0);
      mx_vals(0);
    } else if (mine > 0) {
      load(a.kc, KEYS, 0);
      load(a.vc, VALUES, 0);
    }
    for (int k = 0; k < mine; k++) {
      const int kt = pg_key_tile(range, c0 + w + NW * k) * KT;
      const bool more = k + 1 < mine;
      int good = 0;   // groups of 16 keys whose pages are there
#pragma unroll
      for (int g = 0; g < NG; g++) good |= (__builtin_amdgcn_readlane((int)(group >> 32), (k * NG + g) & 63) >= 0) << g;
      if constexpr (!MX) PG_WAIT(8);   // the keys; the 8 loads after them are the values
      v4f s[NB];
#pragma unroll
      for (int b = 0; b < NB; b++) {
        s[b] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          if constexpr (MX) {
            const uint4 c = kreg[b][ks / 2];
            s[b] = pg_mfma16<TC>(mx_16<TC, MX_F8>(ks & 1 ? uint2{c.z, c.w} : uint2{c.x, c.y}, D == 64 ? kpow[b] : kpow[b] >> (8 * (kg >> 1) + 16 * (ks / 2)) & 255), qf[ks], s[b]);
          } else {
            s[b] = pg_mfma16<TC>(pg_get(kl + ka[ks] + (32 * (b >> 1) + 4 * (b & 1)) * 2 * D), qf[ks], s[b]);
          }
        }
      }
      if constexpr (MX) {
        mx_put();   // (before the groups: these are this tile's)
        if (((k + 1) & (64 / NG - 1)) == 0) groups(k + 1);
        mx_keys(k + 1);
        mx_vals(k + 1);
      } else {
        PG_WAIT_LDS();   // the keys have been read
        if (more) {
          if (((k + 1) & (64 / NG - 1)) == 0) groups(k + 1);
          load(a.kc, KEYS, k + 1);
        }
      }
      // every row sees the whole tile, or the rows' masks (wave-uniform)
      const bool whole = good == (1 << NG) - 1 && kt + KT - 1 <= p0 && kt + KT <= end && (c.window == 0 || kt > p1 - c.window || kt + KT <= c.sinks);
      uint32_t seen = ~0u;
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int key = MX ? 16 * b + 4 * kg + r : 32 * (b >> 1) + 8 * kg + 4 * (b & 1) + r, j = kt + key;
            // pg_sees, by selects
            const bool on = j < cap & j <= pos & (c.window == 0 | j > pos - c.window | j < c.sinks) & (good >> (key >> 4) & 1);
            s[b][r] = on ? s[b][r] : -INFINITY;
            seen |= (uint32_t)on << (4 * b + r);
          }
      }
      float mc = s[0][0];
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int r = 0; r < 4; r++) mc = fmaxf(mc, s[b][r]);
      mc *= sc2;
      if (__any(mc > Mx + (PG_UP<TC> + PG_SLACK))) {
        mc = over_kg(mc, OpMaxF{});
        const float mn = mc == -INFINITY ? Mx : fmaxf(mc - PG_UP<TC>, Mx), up = pg_moved(Mx, mn);
        Mx = mn;
        Ls *= up;
#pragma unroll
        for (int d = 0; d < ND; d++) O[d] *= up;
      }
      const float ref = Mx == -INFINITY ? 0.f : Mx;
      gu32x4 ph[N][NS];
#pragma unroll
      for (int b = 0; b < NB; b++) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          e[r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], sc2, -ref));
          Ls += e[r];
        }
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          uint32_t x[N];
          pg_parts2<TC, N>(e[r], e[r + 1], x);
#pragma unroll
          for (int i = 0; i < N; i++) ph[i][b >> 1][2 * (b & 1) + r / 2] = x[i];
        }
      }
      if constexpr (!MX) {
        if (more) PG_WAIT(8);   // the values; the 8 loads after them are the next keys
        else PG_WAIT(0);
      }
      bool wild = false;
      if (!whole || careful) wild = pg_wild_tile<TC, KT * UPR>(vl, lane);   // what a row does not see must not reach it as 0 x inf
      if (wild) {
#pragma unroll
        for (int d = 0; d < ND; d++) {
          v4f m = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < NS; t++) {
            uint4 marks;
            const uint4 v = pg_tamed<TC>(values(d, t), marks);
#pragma unroll
            for (int i = 0; i < N; i++) O[d] = pg_mfma16<TC>(v, __builtin_bit_cast(uint4, ph[i][t]), O[d]);
            m = pg_mfma16<TC>(marks, pg_ones<TC>(seen >> (8 * t)), m);
          }
#pragma unroll
          for (int r = 0; r < 4; r++) O[d][r] += pg_wild_sum(m[r]);
        }
      } else {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
          for (int t = 0; t < NS; t++) {
            const uint4 v = values(d, t);
#pragma unroll
            for (int i = 0; i < N; i++) O[d] = pg_mfma16<TC>(v, __builtin_bit_cast(uint4, ph[i][t]), O[d]);
          }
      }
      if constexpr (!MX) {
        PG_WAIT_LDS();   // the values have been read
        if (more) load(a.vc, VALUES, k + 1);
      }
    }
    if (careful || !pg_any_wild<ND>(O)) break;
  }
  // the waves' states, each in its own LDS
  Ls = over_kg(Ls, OpAddF{});
  LAS float* st = (LAS float*)lds[w];
#pragma unroll
  for (int d = 0; d < ND; d++) *(LAS v4f*)(st + n * RF + 16 * d + 4 * kg) = O[d];
  if (kg == 0) {
    smx[w][n] = Mx;
    sls[w][n] = Ls;
  }
  __syncthreads();
  for (int i = tid; i < live * (D / 4); i += PG_THREADS) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float m = smx[0][r];
#pragma unroll
    for (int x = 1; x < NW; x++) m = fmaxf(m, smx[x][r]);
    float l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NW; x++) {
      const float e = pg_moved(smx[x][r], m);
      l += sls[x][r] * e;
      o += *(const LAS v4f*)((const LAS float*)lds[x] + r * RF + d) * e;
    }
    if (un.splits == 1) {
      pg_store<TC>(a, un.seq.first + (uint32_t)(f0 + r) / c.G, un.head * c.G + (uint32_t)(f0 + r) % c.G, d, D, l == 0.f ? (v4f){0.f, 0.f, 0.f, 0.f} : o / l);
    } else {
      pg_put_part<D, 16>(p.w, un.part_at + un.split, r, d, m, l, o);
    }
  }
  if (un.splits > 1) pg_finish<TC, D, 16>(a, c, p.w, un, f0, live, shared.join, &shared.last);
}

template <int TC>
__device__ __forceinline__ v16f pg_mfma32(uint4 a, uint4 b, v16f c) {   // 32 x 32 x 16
  if constexpr (TC == PG_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Attention of many rows per sequence. A workgroup of four waves takes 128 flat rows of a key/value head, 32 to a wave;
// tiles of 64 keys and their values go straight into LDS, one while the one before is evaluated. As in the step kernel,
// scores are keys x rows and outputs dims x rows (v_mfma 32 x 32 x 16), so a row's statistics are two lanes' own, and
// the keys are dealt to the score products' rows such that a lane's weights are the next product's operand as they
// stand (row m of block b: key 32 b + m with bits 2 and 3 of m swapped).
// What a row does not see must not reach it as 0 x inf either: in a tile that some row does not see whole, infinities and
// NaN among the values are replaced by 0 in LDS, and added afterwards to the rows that see them.
// One prompt of 8000 rows, 28 / 4 heads of 128, bf16: 454 to 471 us on several cards, 0.97 to 1.01 PFLOP/s, 0.83 to 0.87 of a large matrix
// product's rate; the card lowers its clock in both. With heads of 64 a score costs as many exponentials and sums for half the
// products: 4096 rows of 14 / 2 heads in a window of 1024 take 35 to 37 us, 0.41 to 0.43 PFLOP/s. By the counters vector
// instructions take 13 and the matrix units 7 us of it: a wave's scores, exponentials and weighted values follow each other, and
// the one other wave of a SIMD does not fill its waits. Heads of 128 use all 256 registers and spill 19 outside the loop over tiles.
// MX: a tile's codes and powers go into LDS as they are and are converted once for all four waves, into the one 16-bit buffer, between two barriers; the
// next tile's follow into the same place. 9 sequences of up to 700 new rows, 32 / 8 heads of 128: 158 us, with a bf16 cache 146.
template <int D, bool MX>
struct PgTiles {
  __attribute__((aligned(16))) uint4 lds[2][2][8 * D];   // [buffer][keys, values]
};
template <int D>
struct PgTiles<D, true> {
  __attribute__((aligned(16))) uint4 lds[1][2][8 * D];
  __attribute__((aligned(16))) uint8_t raw[2 * (64 * D + 1024)];   // keys and values, each codes [64][D], then the powers of 16 keys in 256 bytes
};
template <int D, bool MX>
struct PgPromptLds {
  union {
    PgTiles<D, MX> tiles;
    PgJoinLds<128> join;
  };
  int last, tamed, wild;   // tamed: 1 + the last tile whose values were changed; wild: a wave has infinite sums or NaN
  typename PgFinder<MX>::Lds found;
};
template <int TC, int D, bool FINE, bool MX>   // FINE: weights in parts that keep float32 (float32 outputs)
__device__ __forceinline__ void pg_prompt(const PgStep& p, int block, int grid, PgPromptLds<D, MX>& shared) {
  constexpr int N = FINE ? PG_PARTS<TC> : 1;   // parts of a weight
  constexpr int M = 128, KT = 64, UPR = D / 8, KS = D / 16, ND = D / 32, T = KT * UPR, LOADS = MX ? D / 64 + 1 : T / PG_THREADS;   // LOADS: of keys, and of values, per wave and tile
  auto& lds = shared.tiles.lds;
  int& tamed = shared.tamed;
  const PgAttend& a = p.a;
  PgCut c = p.c;
  c.M = M;   // (as the host has them, for the compiler)
  c.KT = KT;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int cap = pg_cap(a.b), pmask = (1 << a.b.page_log) - 1;
  const float sc2 = a.scale * 1.4426950408889634f;
  PgFinder<MX> finder(a.b, c, grid, shared.found);
  auto over_h = [](float v, auto op) {   // over the two lanes of a row
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return op(__int_as_float((int)x[0]), __int_as_float((int)x[1]));
  };
  // a wave loads 16 keys of a tile, and their values: bytes from the group to what this lane loads of its first and last
  // 8 keys; with LOADS 4, every second load is 4 keys further
  uint32_t lane_off[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int key = 16 * w + 8 * i + lane / UPR;
    lane_off[i] = 2 * ((uint32_t)(key & 15) * (uint32_t)a.slot_stride + 8 * ((lane % UPR) ^ pg_swz<D>(key)));
  }
  static_assert(M == 32 * PG_WAVES && KT == 16 * PG_WAVES, "a wave has 32 rows, and loads 16 keys");
  static_assert(MX || LOADS == 2 || LOADS == 4, "two or four keys x 16 bytes x lanes");
  constexpr int RAW = 64 * D + 1024;   // MX: bytes of a tile's keys, or values
  uint32_t mine_lds;
  if constexpr (MX) mine_lds = pg_lds_at(shared.tiles.raw);
  else mine_lds = pg_lds_at(&lds[0][0][64 * LOADS * w]);
  // this lane's operands in a tile: of the keys for each 16 dims, of the values for each 32 and for even and odd 16 keys;
  // others are whole multiples of 32 rows further
  int ka[KS], va[ND][2];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) ka[ks] = 16 * pg_unit_at<D>((n & 19) + ((n & 4) << 1) + ((n & 8) >> 1), 2 * ks + h);
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int t = 0; t < 2; t++) va[d][t] = pg_values_at<D>(16 * t + 8 * h, 32 * d + 16 * ((lane >> 4) & 1), lane & 15);
  if (block >= __builtin_amdgcn_readfirstlane(finder.units)) return;
  const PgUnit un = pg_uniform(finder.find(block));
  if (un.seq.n == 0) return;
  const int G = c.G, flat = un.seq.n * G, f0 = M * un.q, live = min(M, flat - f0);   // (n G is at most 2^26)
  const uint32_t f = min(f0 + 32 * w + n, flat - 1), at_row = f / c.G;
  const int row = un.seq.first + at_row, head = un.head * G + (f - at_row * c.G);
  const int pos = un.seq.p0 + at_row, w0 = __builtin_amdgcn_readlane(pos, 0), w1 = __builtin_amdgcn_readlane(pos, 31);   // of the wave's rows
  const int p0 = un.seq.p0 + (uint32_t)f0 / c.G, p1 = un.seq.p0 + (uint32_t)(f0 + live - 1) / c.G;
  const PgRange range = pg_range(p0, p1, cap, c);
  const int per = pg_up(range.n, un.splits), c0 = min(un.split * per, range.n), count = min(per, range.n - c0);
  const int end = min(p1 + 1, cap), wend = 32 * w < live ? min(w1 + 1, cap) : 0;
  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) qf[ks] = gld((const uint4*)(a.q + row * a.qs + (int64_t)head * D + 16 * ks + 8 * h));
  // where the 16 keys from `key` on are: elements from the cache's begin; -1: not there
  auto place = [&](int key) -> int64_t {
    const int page = gld(a.b.table + un.s * a.b.table_stride + (min(key, end - 1) >> a.b.page_log));
    return page >= 0 && page < a.b.pages ? page * a.page_stride + (MX ? 0 : (key & pmask) * a.slot_stride + un.head * a.head_stride) : -1;
  };
  auto mx_slot = [&](int key) { return (un.head << a.b.page_log) + (key & pmask); };   // MX: a key's place among all of its page
  int all_hi = min(p0 + 1, end) - KT;
  const int all_lo = c.window ? p1 - c.window : -1, mine_hi = min(w0 + 1, wend) - KT, mine_lo = c.window ? w1 - c.window : -1;
  int64_t group = -1;   // of the next 16 tiles, 16 keys a lane
  uint64_t there = 0;   // which of them have a place
  auto groups = [&](int k) {
    const int t = k + lane / 4;
    group = -1;
    if (t < count) group = place(pg_key_tile(range, c0 + t) * KT + 16 * (lane % 4));
    there = __ballot(group >= 0);
  };
  // Loads of a tile, 2 x LOADS of them, one at a time between the products of the tile before: together, right behind the
  // barrier, they held every wave up for 900 cycles (D 128), a quarter of a tile. A tile behind the last is the first page.
  const uint16_t *next_k, *next_v;
  int64_t next_powers;   // MX: bytes from the codes to their powers
  auto next = [&](int k) {
    const int at = (4 * k + w) & 63;
    const int64_t e = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)group, at) |
                                (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(group >> 32), at) << 32);
    const int64_t off = k < count && e > 0 ? e : 0;   // (where there is none, the first page is loaded, and masked)
    if constexpr (MX) {
      const int slot = mx_slot(k < count ? pg_key_tile(range, c0 + k) * KT + 16 * w : 0);
      next_k = (const uint16_t*)((const uint8_t*)a.kc + off + slot * D);
      next_v = (const uint16_t*)((const uint8_t*)a.vc + off + slot * D);
      next_powers = a.powers_at - slot * (D - D / 32);
    } else {
      next_k = a.kc + off;
      next_v = a.vc + off;
    }
  };
  auto load = [&](auto i, auto buffer) {
    constexpr int I = i % LOADS;
    if constexpr (MX) {   // 16 keys of the wave's: D / 64 loads of codes, one of powers (which the lanes read several times)
      const uint8_t* from = (const uint8_t*)(i < LOADS ? next_k : next_v);
      constexpr int AT = i < LOADS ? 0 : RAW;
      if constexpr (I < D / 64) pg_dma16<AT + 1024 * I>(from + 1024 * I, 16 * lane, mine_lds + 16 * D * w);
      else pg_dma4<AT + 64 * D>(from + next_powers, 4 * (lane % (D / 8)), mine_lds + 256 * w);
    } else pg_dma16<32 * T * buffer + (i < LOADS ? 0 : 16 * T) + 1024 * I>((i < LOADS ? next_k : next_v) + (LOADS == 4 && (I & 1) ? 4 * a.slot_stride : 0), lane_off[I * 2 / LOADS],
                                                                mine_lds);
  };
  const auto B0 = std::integral_constant<int, 0>{};
  float Mx, Ls;   // Ls: this lane's keys only
  v16f O[ND];
  auto tile = [&](int k, auto buffer) {   // buffer: k % 2
    constexpr int BUF = decltype(buffer)::value;
    constexpr std::integral_constant<int, 1 - BUF> OTHER{};
    const int kt = pg_key_tile(range, c0 + k) * KT;
    const int good = (int)(there >> (4 * k & 63)) & 15;   // groups of 16 keys that are there
    // whether all rows of the workgroup, and of the wave, see the whole tile (the same for every lane)
    const bool all = good == 15 && kt <= all_hi && (kt > all_lo || kt + KT <= c.sinks), mine = good == 15 && kt <= mine_hi && (kt > mine_lo || kt + KT <= c.sinks);
    if (((k + 1) & 15) == 0) groups(k + 1);
    next(k + 1);
    PG_WAIT(0);
    __syncthreads();   // the tile is there, and every wave is done with the buffer filled next
    const LAS uint8_t* kl = (const LAS uint8_t*)lds[BUF][0];
    LAS uint8_t* vl = (LAS uint8_t*)lds[BUF][1];
    if constexpr (MX) {   // codes and powers as 16-bit values where the other caches' loads put them
      const LAS uint8_t* raw = (const LAS uint8_t*)shared.tiles.raw;
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int j = 0; j < D / 64; j++) {
          const int i = tid + PG_THREADS * j, key = i / (D / 16), u = i % (D / 16);
          const uint4 c = pg_get(raw + RAW * x + 16 * i);
          const uint32_t byte = raw[RAW * x + 64 * D + 256 * (key >> 4) + (D / 32) * (key & 15) + (u >> 1)];
#pragma unroll
          for (int half = 0; half < 2; half++) {
            uint4 y = mx_16<TC, MX_F8>(half ? uint2{c.z, c.w} : uint2{c.x, c.y}, byte);
            if (x == 1 && !all && pg_wild<TC>(y)) {
              uint4 marks;
              y = pg_tamed<TC>(y, marks);
              tamed = k + 1;
            }
            *(pg_lds4*)((x ? vl : (LAS uint8_t*)lds[BUF][0]) + 16 * pg_unit_at<D>(key, 2 * u + half)) = (gu32x4){y.x, y.y, y.z, y.w};
          }
        }
      PG_TURN();
    } else if (!all) {
#pragma unroll 1
      for (int i = tid; i < T; i += PG_THREADS) {
        uint4 marks;
        const uint4 v = pg_get(vl + 16 * i);
        if (pg_wild<TC>(v)) {
          const uint4 y = pg_tamed<TC>(v, marks);
          *(pg_lds4*)(vl + 16 * i) = (gu32x4){y.x, y.y, y.z, y.w};
          tamed = k + 1;
        }
      }
      PG_TURN();
    }
    if (kt >= wend) {   // behind all of the wave's rows
      pg_each<2 * LOADS>([&](auto i) { load(i, OTHER); });
      return;
    }
    // operands are read a group of products ahead; the fences keep the compiler from moving the reads back to their products
    v16f s[2] = {};
    uint4 kf[2][2][2];   // [group's turn][16 dims][32 keys]
    auto keys = [&](int g) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int b = 0; b < 2; b++) kf[g & 1][i][b] = pg_get(kl + ka[2 * g + i] + 32 * b * 2 * D);
      __builtin_amdgcn_sched_barrier(0);
    };
    keys(0);
    pg_each<KS / 2>([&](auto g) {
      if constexpr (g + 1 < KS / 2) keys(g + 1);
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int b = 0; b < 2; b++) s[b] = pg_mfma32<TC>(kf[g & 1][i][b], qf[2 * g + i], s[b]);
      constexpr int PER = (4 * LOADS + KS - 1) / KS;
      pg_each<PER>([&](auto i) {
        if constexpr (PER * g + i < 2 * LOADS) load(std::integral_constant<int, PER * g + i>{}, OTHER);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    uint4 vf[2][ND];   // [group's turn][32 dims]: the values of 16 keys
    auto values = [&](int t) {
#pragma unroll
      for (int d = 0; d < ND; d++) vf[t & 1][d] = pg_values<D>(vl + va[d][t & 1] + 32 * (t >> 1) * 2 * D);
      __builtin_amdgcn_sched_barrier(0);
    };
    values(0);
    uint32_t seen = ~0u;
    if (!mine) {
      seen = 0;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int key = 32 * b + 16 * (r >> 3) + 8 * h + (r & 7), j = kt + key;
          const bool on = j < cap & j <= pos & (c.window == 0 | j > pos - c.window | j < c.sinks) & (good >> (2 * b + (r >> 3)) & 1);   // pg_sees
          s[b][r] = on ? s[b][r] : -INFINITY;
          seen |= (uint32_t)on << (16 * b + r);
        }
    }
    float mc = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int r = 0; r < 16; r++) mc = fmaxf(mc, s[b][r]);
    mc *= sc2;
    if (__any(mc > Mx + (PG_UP<TC> + PG_SLACK))) {
      mc = over_h(mc, OpMaxF{});
      const float mn = mc == -INFINITY ? Mx : fmaxf(mc - PG_UP<TC>, Mx), up = pg_moved(Mx, mn);
      Mx = mn;
      Ls *= up;
#pragma unroll
      for (int d = 0; d < ND; d++) O[d] *= up;
    }
    const float ref = Mx == -INFINITY ? 0.f : Mx;
    gu32x4 ph[4][N];   // weights of 16 keys each; in parts only where they are used, and until then in the scores' place
    auto parts = [&](int t) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint32_t x[N];
        pg_parts2<TC, N>(s[t >> 1][8 * (t & 1) + i], s[t >> 1][8 * (t & 1) + i + 1], x);
#pragma unroll
        for (int n = 0; n < N; n++) ph[t][n][i >> 1] = x[n];
      }
    };
#pragma unroll
    for (int t = 0; t < 4; t++) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int r = 8 * (t & 1) + i;
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[t >> 1][r], sc2, -ref)), e1 = __builtin_amdgcn_exp2f(fmaf(s[t >> 1][r + 1], sc2, -ref));
        sum += e0 + e1;
        s[t >> 1][r] = e0;
        s[t >> 1][r + 1] = e1;
      }
      Ls += sum;
      if constexpr (!FINE) parts(t);
    }
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if (t < 3) values(t + 1);
      if constexpr (FINE) parts(t);
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int n = 0; n < N; n++) O[d] = pg_mfma32<TC>(vf[t & 1][d], __builtin_bit_cast(uint4, ph[t][n]), O[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!all && __builtin_amdgcn_readfirstlane(tamed) == k + 1) {   // the values as they were, from memory
#pragma unroll
      for (int d = 0; d < ND; d++) {
        v16f m = {};
#pragma unroll 1
        for (int t = 0; t < 4; t++) {
          const int64_t at = place(kt + 16 * t);
          uint32_t x[4];
          if constexpr (MX) {
            const uint8_t* page = (const uint8_t*)a.vc + (at < 0 ? 0 : at);
            const int first = mx_slot(kt + 16 * t) + 8 * h;
            auto value = [&](int i) { return mx_16<TC, MX_F8>({gld(page + (first + i) * D + 32 * d + n), 0}, gld(page + a.powers_at + (first + i) * (D / 32) + d)).x & 0xFFFF; };
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = value(2 * i) | value(2 * i + 1) << 16;
          } else {
            const uint16_t* v = a.vc + (at < 0 ? 0 : at) + 8 * h * a.slot_stride + 32 * d + n;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = gld(v + 2 * i * a.slot_stride) | (uint32_t)gld(v + (2 * i + 1) * a.slot_stride) << 16;
          }
          uint4 marks;
          pg_tamed<TC>(make_uint4(x[0], x[1], x[2], x[3]), marks);
          m = pg_mfma32<TC>(marks, pg_ones<TC>(seen >> (8 * t)), m);
        }
#pragma unroll
        for (int r = 0; r < 16; r++) O[d][r] += pg_wild_sum(m[r]);
      }
    }
  };
  if (tid == 0) shared.wild = 0;
  for (bool careful = false;; careful = true) {   // (twice only for infinities and NaN, pg_any_wild)
    Mx = -INFINITY;
    Ls = 0.f;
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] = (v16f){};
    if (tid == 0) tamed = 0;
    groups(0);
    PG_WAIT_OWN();
    if (count > 0) {
      next(0);
      pg_each<2 * LOADS>([&](auto i) { load(i, B0); });
    }
    if constexpr (MX) {
      for (int k = 0; k < count; k++) tile(k, B0);
    } else {
      for (int k = 0; k < count; k += 2) {
        tile(k, std::integral_constant<int, 0>{});
        if (k + 1 < count) tile(k + 1, std::integral_constant<int, 1>{});
      }
    }
    PG_WAIT(0);   // (a load behind the last tile)
    if (careful || count == 0) break;
    if (pg_any_wild<ND>(O) && lane == 0) shared.wild = 1;   // (set to 0 before the first tile's barrier)
    __syncthreads();
    if (!__builtin_amdgcn_readfirstlane(shared.wild)) break;
    all_hi = -KT;   // no tile counts as seen whole by all rows
  }
  Ls = over_h(Ls, OpAddF{});
  const int r = 32 * w + n;
  if (r < live) {
    const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const v4f o = {O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]};
        const int dim = 32 * d + 8 * i + 4 * h;
        if (un.splits == 1) pg_store<TC>(a, row, head, dim, D, Ls == 0.f ? (v4f){0.f, 0.f, 0.f, 0.f} : o * inv);
        else pg_put_part<D, M>(p.w, un.part_at + un.split, r, dim, Mx, Ls, o);
      }
  }
  if (un.splits > 1) pg_finish<TC, D, M>(a, c, p.w, un, f0, live, shared.join, &shared.last);
}

template <int TC, int D, bool FINE, bool MX>
__global__ __launch_bounds__(PG_THREADS, 2) void pg_step_kernel(PgStep p) {
  __shared__ PgStepLds<MX> lds;
  pg_step<TC, D, FINE, MX>(p, blockIdx.x, gridDim.x, lds);
}
template <int TC, int D, bool FINE, bool MX>
__global__ __launch_bounds__(PG_THREADS, 2) void pg_prompt_kernel(PgStep p) {
  __shared__ PgPromptLds<D, MX> lds;
  pg_prompt<TC, D, FINE, MX>(p, blockIdx.x, gridDim.x, lds);
}
// Both in one launch: prompts in its first workgroups, and what waits for memory beside them.
struct PgBoth {
  PgAttend a;
  PgCut prompt, step;
  PgWork prompt_work, step_work;
  int32_t prompts;   // workgroups
};
template <int TC, int D, bool FINE, bool MX>
__global__ __launch_bounds__(PG_THREADS, 2) void pg_both_kernel(PgBoth p) {
  __shared__ union Lds {
    PgStepLds<MX> step;
    PgPromptLds<D, MX> prompt;
    __device__ Lds() {}
  } lds;
  if ((int)blockIdx.x < p.prompts) pg_prompt<TC, D, FINE, MX>({p.a, p.prompt, p.prompt_work}, blockIdx.x, p.prompts, lds.prompt);
  else pg_step<TC, D, FINE, MX>({p.a, p.step, p.step_work}, blockIdx.x - p.prompts, gridDim.x - p.prompts, lds.step);
}

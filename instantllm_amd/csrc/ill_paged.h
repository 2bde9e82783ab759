// Kernels of the paged-cache operators (ill_paged_* in include/ill_hip.h).
//
// A cache is two arrays of pages of 2^page_log positions, keys and values; position t of sequence
// s is slot t % page_size of page table[s][t / page_size]. A batch's new rows are the last ones
// of their sequences. Page numbers outside 0 .. pages - 1 are never followed.
#pragma once
#include "ill_device.h"
#include "ill_paged_plan.h"

enum PgType { PG_F32 = 0, PG_F16 = 1, PG_BF16 = 2 };   // ILL_F32, ILL_F16, ILL_BF16

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// Eight values of type T as floats, and back with one rounding to nearest, ties to even.
template <int T>
__device__ __forceinline__ void pg_unpack(const uint4* p, float* x) {
  if constexpr (T == PG_F32) {
    *(uint4*)x = p[0];
    *(uint4*)(x + 4) = p[1];
  } else {
    const uint32_t w[4] = {p->x, p->y, p->z, p->w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (T == PG_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
    }
  }
}
template <int T>
__device__ __forceinline__ uint32_t pg_pack2(float a, float b) {
  if constexpr (T == PG_BF16)
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16;
  else
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
}
template <int T>
__device__ __forceinline__ uint4 pg_pack8(const float* x) {
  return {pg_pack2<T>(x[0], x[1]), pg_pack2<T>(x[2], x[3]), pg_pack2<T>(x[4], x[5]), pg_pack2<T>(x[6], x[7])};
}
template <int T>
__device__ __forceinline__ float pg_one(const uint16_t* p) {
  const uint16_t w = gld(p);
  return T == PG_BF16 ? __uint_as_float((uint32_t)w << 16) : (float)__builtin_bit_cast(_Float16, w);
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

// A workgroup takes R rows; a thread takes 16 values of one head at a time: the eight first and the
// eight second halves of eight rotated pairs (or eight whole pairs twice where pairs are
// interleaved), so that a pair never leaves its thread and a head's square sum stays within D / 16
// neighbouring lanes. The angles' sines and cosines are computed once per row and pair, from turns
// in float64 (a position of 2^20 has to keep 2^-20 of a turn and more), and shared through LDS.
template <int TX, int TC, int D>
__global__ __launch_bounds__(256) void pg_append_kernel(PgAppend a, int R) {
  extern __shared__ __attribute__((aligned(16))) uint8_t pg_lds[];
  constexpr int C = D / 16;   // threads of a head
  const int half = a.rot >> 1;
  int64_t* place = (int64_t*)pg_lds;             // [R] element offset of the row's slot, -1: nothing to write
  int* angle_of = (int*)(place + R);             // [R] position that turns the row
  float2* cs = (float2*)(angle_of + (R + 1) / 2 * 2);   // [R][half]
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, first = blockIdx.x * R;
  for (int i = w; i < R; i += 4) {
    const int r = first + i;
    int64_t off = -1;
    int at = 0;
    const int s = r >= a.b.rows ? -1 : a.b.row0 ? pg_seq_of(a.b, r, lane) : r;
    if (s >= 0 && s < a.b.seqs) {
      const int len = pg_len(gld(a.b.lens + s));
      const int t = a.b.row0 ? len - (gld(a.b.row0 + s + 1) - r) : len - 1;
      at = a.positions ? gld(a.positions + r) : t;
      if (t >= 0 && t < pg_cap(a.b)) {
        const int page = gld(a.b.table + s * a.b.table_stride + (t >> a.b.page_log));
        if (page >= 0 && page < a.b.pages) off = page * a.page_stride + (t & ((1 << a.b.page_log) - 1)) * a.slot_stride;
        else off = -2;
      } else {
        off = -2;   // a row without a place in the cache: its query is turned all the same
      }
    }
    if (lane == 0) {
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
  const int nh = a.heads + 2 * a.kv, h0 = a.q ? 0 : a.heads;
  for (int it = tid; it < R * (nh - h0) * C; it += 256) {
    const int c = it % C, head = h0 + it / C % (nh - h0), i = it / C / (nh - h0), r = first + i;
    const bool live = place[i] != -1;   // (the same for all lanes of a head)
    const int kind = head < a.heads ? 0 : head < a.heads + a.kv ? 1 : 2, hk = kind == 0 ? head : kind == 1 ? head - a.heads : head - a.heads - a.kv;
    const bool turn = kind < 2 && c < a.rot / 16;
    const int da = a.rot == 0 || c >= a.rot / 16 || a.interleaved ? 16 * c : 8 * c;
    const int db = turn && !a.interleaved ? da + half : da + 8;
    // values keep their order (kind 2), and so do the dims behind the rotated ones
    const int d[2] = {kind == 2 ? 16 * c : da, kind == 2 ? 16 * c + 8 : db};
    float x[2][8] = {};
    constexpr int EB = TX == PG_F32 ? 4 : 2;
    if (live) {
      const uint8_t* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + EB * (r * (kind == 0 ? a.qs : kind == 1 ? a.ks : a.vs) + (int64_t)hk * D);
#pragma unroll
      for (int u = 0; u < 2; u++) {
        uint4 raw[EB / 2];
#pragma unroll
        for (int n = 0; n < EB / 2; n++) raw[n] = gld((const uint4*)(src + EB * d[u]) + n);
        pg_unpack<TX>(raw, x[u]);
        if (a.bias)
#pragma unroll
          for (int n = 0; n < 8; n++) x[u][n] += gld(a.bias + head * D + d[u] + n);
      }
    }
    const float* gamma = kind == 0 ? a.qn : kind == 1 ? a.kn : nullptr;
    if (a.qn || a.kn) {   // (the lanes of a head agree; other heads' lanes take part in the exchange)
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 8; n++) sum = fmaf(x[0][n], x[0][n], fmaf(x[1][n], x[1][n], sum));
#pragma unroll
      for (int m = 1; m < C; m <<= 1) sum += __shfl_xor(sum, m);
      if (gamma) {
        const float inv = 1.f / sqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int n = 0; n < 8; n++) x[u][n] *= inv * gld(gamma + d[u] + n);
      }
    }
    if (!live) continue;
    if (turn) {
      const float2* row = cs + i * half;
      if (a.interleaved) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int n = 0; n < 8; n += 2) {
            const float2 t = row[(d[u] + n) >> 1];
            const float p = x[u][n], q = x[u][n + 1];
            x[u][n] = fmaf(p, t.x, -(q * t.y));
            x[u][n + 1] = fmaf(q, t.x, p * t.y);
          }
      } else {
#pragma unroll
        for (int n = 0; n < 8; n++) {
          const float2 t = row[d[0] + n];
          const float p = x[0][n], q = x[1][n];
          x[0][n] = fmaf(p, t.x, -(q * t.y));
          x[1][n] = fmaf(q, t.x, p * t.y);
        }
      }
    }
    if (kind > 0 && place[i] < 0) continue;
    uint16_t* dst = kind == 0 ? (uint16_t*)a.qo + r * a.qos + (int64_t)hk * D
                              : (uint16_t*)(kind == 1 ? a.kc : a.vc) + place[i] + hk * a.head_stride;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint4 y = pg_pack8<TC>(x[u]);
      gst((gu32x4*)(dst + d[u]), (gu32x4){y.x, y.y, y.z, y.w});
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
};

// One wave per new row and query head: 64 positions at a time, a lane's score each, then the
// running softmax and the values, a lane's D / 64 dims each.
template <int TC, int D>
__global__ __launch_bounds__(64) void pg_attend_simple_kernel(PgAttend a) {
  const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int s = a.b.row0 ? pg_seq_of(a.b, r, lane) : r;
  if (s < 0 || s >= a.b.seqs) return;
  const int len = pg_len(gld(a.b.lens + s));
  const int p = a.b.row0 ? len - (gld(a.b.row0 + s + 1) - r) : len - 1;
  __shared__ float q[D];
  for (int d = lane; d < D; d += 64) q[d] = pg_one<TC>(a.q + r * a.qs + (int64_t)h * D + d);
  __syncthreads();
  const int64_t hoff = (int64_t)(h / (a.heads / a.kv)) * a.head_stride;
  const int mask = (1 << a.b.page_log) - 1;
  float m = -INFINITY, l = 0.f, o[D / 64] = {};
  const int end = min(p + 1, pg_cap(a.b));
  for (int j0 = 0; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    const int page = j < end ? gld(a.b.table + s * a.b.table_stride + (j >> a.b.page_log)) : -1;
    const bool on = pg_sees(p, j, a.window, a.sinks) && page >= 0 && page < a.b.pages;
    const int64_t off = on ? page * a.page_stride + (j & mask) * a.slot_stride + hoff : 0;
    float sc = -INFINITY;
    if (on) {
      float x = 0.f;
      for (int d = 0; d < D; d++) x = fmaf(q[d], pg_one<TC>(a.kc + off + d), x);
      sc = x * a.scale;
    }
    float mn = fmaxf(m, sc);
    for (int k = 1; k < 64; k <<= 1) mn = fmaxf(mn, __shfl_xor(mn, k));
    if (mn == -INFINITY) continue;
    const float up = expf(m - mn), e = on ? expf(sc - mn) : 0.f;
    m = mn;
    l = l * up + e;
    for (int u = 0; u < D / 64; u++) o[u] *= up;
    for (uint64_t left = __ballot(on); left; left &= left - 1) {
      const int k = __ffsll((unsigned long long)left) - 1;
      const int64_t ok = __shfl(off, k);
      const float ek = __shfl(e, k);
      for (int u = 0; u < D / 64; u++) o[u] = fmaf(ek, pg_one<TC>(a.vc + ok + lane + 64 * u), o[u]);
    }
  }
  for (int k = 1; k < 64; k <<= 1) l += __shfl_xor(l, k);
  for (int u = 0; u < D / 64; u++) {
    const float y = m == -INFINITY ? 0.f : o[u] / l;
    const int64_t at = r * a.os + (int64_t)h * D + lane + 64 * u;
    if (a.out_f32) gst((float*)a.out + at, y);
    else gst((uint16_t*)a.out + at, (uint16_t)pg_pack2<TC>(y, 0.f));
  }
}

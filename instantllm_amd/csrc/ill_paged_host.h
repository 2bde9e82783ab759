// Host side of the paged-cache operators: argument checks and launches (ill_paged_* in
// include/ill_hip.h). Included by ill_engine.hip after its error helpers.
#pragma once
#include "ill_paged.h"
#include "ill_paged_check.h"
#include "ill_paged_claims.h"

struct ill_paged {
  ill_paged_desc d{};
  int device = 0, page_log = 0;
  double* freq = nullptr;   // [rotary_dim / 2] turns per position
  uint8_t* work = nullptr;   // workspaces of attention parts
  size_t work_bytes = 0;
  illp::Workspaces workspaces;
};

namespace illp {

// The current device is the handle's while this lives.
struct OnDevice {
  int was = -1, rc = ILL_OK;
  explicit OnDevice(int dev) {
    if (hipGetDevice(&was) != hipSuccess) rc = fail(ILL_E_HIP, "no HIP device");
    else if (was != dev && hipSetDevice(dev) != hipSuccess) rc = fail(ILL_E_HIP, "device %d cannot be made current", dev);
    if (was == dev || rc) was = -1;
  }
  ~OnDevice() {
    if (was >= 0) hipSetDevice(was);
  }
};

PgBatch batch_of(const ill_paged* p, const ill_paged_batch& b) {
  return {b.lens, b.table, b.row0, b.table_stride, b.pages, b.seqs, (int)b.rows, b.table_width, p->page_log};
}

// A call's parts. The step kernel cuts the keys into about a part for each CU (2^8), of 8 tiles of keys at least, two for each
// wave: with 2^9 parts or 4 tiles the joining cost more than it gave (us, 2^8 / 2^9: one sequence of 131071 20.3 / 21.1, 200
// through a window of 1024 25.1 / 33.7, but 64 ragged ones 97.7 / 95; 8 / 4 tiles: one of 500 6.8 / 8.3). The prompt kernel cuts
// a tile of rows whose keys are over 2^-7 of the call's work; a prompt alone, with PG_MANY tiles at least, never is. More parts, for the 512
// workgroups that run at a time, have not been measured on batches that they would cut.
PgCut step_cut(const ill_paged_desc& d, int window, int sinks) {
  return {(uint32_t)(d.heads / d.kv_heads), (uint32_t)d.kv_heads, 16, d.head_dim == 64 ? 64 : 32, window, sinks, 8, 8, 0, PG_MOST, 0};
}
PgCut prompt_cut(const ill_paged_desc& d, int window, int sinks) {
  return {(uint32_t)(d.heads / d.kv_heads), (uint32_t)d.kv_heads, 128, 64, window, sinks, 7, 4, 0, PG_MOST, 0};
}

// Bytes of a workspace where 2^log parts are wanted, over tiles of M rows.
size_t counters(int log) { return al256(((size_t)(PG_MAXSPLIT / PG_FAN + 1) << log) * 4); }
size_t work_size(int log, int M, int D) { return al256((size_t)M * (D + 2) * 4 << (log + 1)) + counters(log); }

PgWork work_of(uint8_t* at, int log, int M, int D) {
  PgWork w;
  w.joined = (int32_t*)at;
  w.o = (float*)(at + counters(log));
  w.ml = (float2*)(w.o + ((size_t)M * D << (log + 1)));
  return w;
}

// The workspace of the stream, or of its capture.
int workspace(ill_paged* p, hipStream_t st, uint8_t** out) {
  if (st == hipStreamLegacy) st = nullptr;
  int w = p->workspaces.bound_to(st);
  if (w < 0) {
    unsigned long long id = 0;
    if (st) {
      hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
      HCK(hipStreamGetCaptureInfo(st, &status, &id));
      if (status == hipStreamCaptureStatusNone) id = 0;
    }
    w = p->workspaces.claim(st, id);
  }
  if (w < 0)
    return fail(ILL_E_ARG, "paged: calls have come on as many streams and captures as the handle has workspaces for, %d (ill_paged_bind, ill_paged_release)",
                p->d.streams);
  *out = p->work + w * p->work_bytes;
  return ILL_OK;
}

// Enqueues a kernel and returns this launch's error (hipGetLastError may hold one of the program's own calls).
template <class... P>
hipError_t launch(void (*kernel)(P...), int64_t blocks, int threads, int lds, hipStream_t st, std::common_type_t<P>... args) {
  void* p[] = {&args...};
  return hipLaunchKernel((const void*)kernel, dim3(blocks), dim3(threads), p, lds, st);
}

// `steps`, `prompts`: workgroups of each kind.
template <int TC, int D, bool FINE>
hipError_t launch_attend(const PgBoth& s, int64_t steps, hipStream_t st) {
  if (!s.prompts) return launch(pg_step_kernel<TC, D, FINE>, steps, PG_THREADS, 0, st, PgStep{s.a, s.step, s.step_work});
  if (!steps) return launch(pg_prompt_kernel<TC, D, FINE>, s.prompts, PG_THREADS, 0, st, PgStep{s.a, s.prompt, s.prompt_work});
  return launch(pg_both_kernel<TC, D, FINE>, s.prompts + steps, PG_THREADS, 0, st, s);
}
template <int TC, int D>
hipError_t launch_attend(const PgBoth& s, int64_t steps, hipStream_t st) {
  return s.a.out_f32 ? launch_attend<TC, D, true>(s, steps, st) : launch_attend<TC, D, false>(s, steps, st);
}

template <int TX, int TC>
hipError_t launch_append(const PgAppend& a, int D, int R, int lds, hipStream_t st) {
  const int64_t blocks = ((int64_t)a.b.rows + R - 1) / R;
  return D == 64 ? launch(pg_append_kernel<TX, TC, 64>, blocks, 256, lds, st, a, R) : launch(pg_append_kernel<TX, TC, 128>, blocks, 256, lds, st, a, R);
}

}  // namespace illp

extern "C" {

int ill_paged_destroy(ill_paged* p) {
  if (!p) return ILL_OK;
  {
    illp::OnDevice on(p->device);
    hipFree(p->freq);
    hipFree(p->work);
  }
  delete p;
  return ILL_OK;
}

int ill_paged_create(const ill_paged_desc* desc, ill_paged** out) {
  if (!out) return fail(ILL_E_ARG, "null output handle");
  *out = nullptr;
  if (!desc) return fail(ILL_E_ARG, "paged: null description");
  ill_paged_desc d = *desc;
  if (int rc = illp::check_desc(d)) return rc;
  ill_paged* p = new (std::nothrow) ill_paged();
  if (!p) return fail(ILL_E_ARG, "paged: out of host memory");
  auto bad = [&](int rc) { ill_paged_destroy(p); return rc; };
  p->d = d;
  while (1 << p->page_log < d.page_size) p->page_log++;
  if (hipGetDevice(&p->device) != hipSuccess) return bad(fail(ILL_E_HIP, "no HIP device"));
  double freq[64] = {};
  for (int i = 0; i < d.rotary_dim / 2; i++) freq[i] = std::pow(d.rope_base, -2.0 * i / d.rotary_dim) / (2 * M_PI);
  if (hipMalloc(&p->freq, sizeof freq) != hipSuccess || hipMemcpy(p->freq, freq, sizeof freq, hipMemcpyHostToDevice) != hipSuccess)
    return bad(fail(ILL_E_HIP, "paged: buffer allocation failed"));
  for (const PgCut& c : {illp::step_cut(d, 0, 0), illp::prompt_cut(d, 0, 0)}) p->work_bytes += illp::work_size(c.log, c.M, d.head_dim);
  if (hipMalloc(&p->work, p->work_bytes * d.streams) != hipSuccess || hipMemset(p->work, 0, p->work_bytes * d.streams) != hipSuccess ||
      hipDeviceSynchronize() != hipSuccess)
    return bad(fail(ILL_E_HIP, "paged: %d workspaces of %zu bytes cannot be allocated", d.streams, p->work_bytes));
  p->workspaces.count = d.streams;
  try {
    p->workspaces.claims.reserve(d.streams);
  } catch (const std::exception&) {
    return bad(fail(ILL_E_ARG, "paged: out of host memory"));
  }
  *out = p;
  return ILL_OK;
}

int ill_paged_release(ill_paged* p) {
  if (!p) return fail(ILL_E_ARG, "paged: null handle");
  p->workspaces.clear();
  return ILL_OK;
}

int ill_paged_bind(ill_paged* p, void* stream, int workspace) {
  if (!p) return fail(ILL_E_ARG, "paged: null handle");
  hipStream_t st = (hipStream_t)stream;
  if (st == hipStreamPerThread) return fail(ILL_E_ARG, "paged: the per-thread default stream is several streams; pass a stream of your own");
  if (st == hipStreamLegacy) st = nullptr;
  if (workspace < -1 || workspace >= p->d.streams) return fail(ILL_E_ARG, "paged: workspace %d of %d", workspace, p->d.streams);
  if (workspace < 0) {
    p->workspaces.forget(st);
    return ILL_OK;
  }
  try {
    if (!p->workspaces.bind(st, workspace)) {
      const int now = p->workspaces.bound_to(st);
      if (now >= 0) return fail(ILL_E_ARG, "paged: the stream is bound to workspace %d", now);
      return fail(ILL_E_ARG, "paged: workspace %d is held by the calls of a stream that is not bound", workspace);
    }
  } catch (const std::exception&) {
    return fail(ILL_E_ARG, "paged: out of host memory");
  }
  return ILL_OK;
}

int ill_paged_append(ill_paged* p, const ill_paged_batch* batch, const ill_paged_rows* x, void* k_cache, void* v_cache, void* stream) {
  if (!p) return fail(ILL_E_ARG, "paged: null handle");
  const ill_paged_desc& d = p->d;
  if (int rc = illp::check_append(d, batch, x, k_cache, v_cache)) return rc;
  if (!batch->seqs || !batch->rows) return ILL_OK;
  PgAppend a{};
  a.b = illp::batch_of(p, *batch);
  a.q = (const uint8_t*)x->q;
  a.k = (const uint8_t*)x->k;
  a.v = (const uint8_t*)x->v;
  a.qo = (uint8_t*)x->q_out;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.qs = x->q_stride;
  a.ks = x->k_stride;
  a.vs = x->v_stride;
  a.qos = x->q_out_stride;
  a.page_stride = d.page_stride;
  a.slot_stride = d.slot_stride;
  a.head_stride = d.head_stride;
  a.bias = x->bias;
  a.qn = x->q ? x->q_norm : nullptr;
  a.kn = x->k_norm;
  a.freq = p->freq;
  a.positions = x->positions;
  a.heads = d.heads;
  a.kv = d.kv_heads;
  a.rot = d.rotary_dim;
  a.interleaved = d.interleaved != 0;
  a.eps = d.norm_eps;
  illp::OnDevice on(p->device);
  if (on.rc) return on.rc;
  const int R = pg_append_rows(a.b.rows, ((a.q ? d.heads : 0) + 2 * d.kv_heads) * d.head_dim / 16), lds = R * 8 + (R + 1) / 2 * 8 + R * (d.rotary_dim / 2) * 8;
  hipStream_t st = (hipStream_t)stream;
  if (x->dtype == ILL_F32) {
    if (d.dtype == ILL_F16) HCK((illp::launch_append<PG_F32, PG_F16>(a, d.head_dim, R, lds, st)));
    else HCK((illp::launch_append<PG_F32, PG_BF16>(a, d.head_dim, R, lds, st)));
  } else if (d.dtype == ILL_F16) {
    HCK((illp::launch_append<PG_F16, PG_F16>(a, d.head_dim, R, lds, st)));
  } else {
    HCK((illp::launch_append<PG_BF16, PG_BF16>(a, d.head_dim, R, lds, st)));
  }
  return ILL_OK;
}

int ill_paged_attend(ill_paged* p, const ill_paged_batch* batch, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                     int window, int sinks, void* out, int64_t out_stride, int out_dtype, void* stream) {
  if (!p) return fail(ILL_E_ARG, "paged: null handle");
  const ill_paged_desc& d = p->d;
  if (int rc = illp::check_attend(d, batch, q, q_stride, k_cache, v_cache, window, sinks, out, out_stride, out_dtype)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (st == hipStreamPerThread) return fail(ILL_E_ARG, "paged: the per-thread default stream is several streams; pass a stream of your own");
  if (!batch->seqs || !batch->rows) return ILL_OK;
  PgAttend a{};
  a.b = illp::batch_of(p, *batch);
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.out = out;
  a.qs = q_stride;
  a.os = out_stride;
  a.page_stride = d.page_stride;
  a.slot_stride = d.slot_stride;
  a.head_stride = d.head_stride;
  a.heads = d.heads;
  a.kv = d.kv_heads;
  a.window = (int)std::min<int64_t>(window, illp::kMost);
  a.sinks = (int)std::min<int64_t>(sinks, illp::kMost);
  a.out_f32 = out_dtype == ILL_F32;
  a.scale = d.scale;
  illp::OnDevice on(p->device);
  if (on.rc) return on.rc;
  // One of the kernels where the sizes that the host knows say which, else both in one launch: the sequences are divided by pg_share.
  const int64_t G = d.heads / d.kv_heads, most = !a.b.row0 ? 1 : std::min<int64_t>(a.b.rows, batch->max_rows ? batch->max_rows : a.b.rows);
  PgBoth s{a, illp::prompt_cut(d, a.window, a.sinks), illp::step_cut(d, a.window, a.sinks), {}, {}, 0};
  const int cap = pg_cap(a.b);
  const bool prompts = most * G > PG_FEW && std::min((a.b.rows * G / 128 + a.b.seqs), (most * G + 127) / 128 * a.b.seqs) * d.kv_heads >= PG_MANY;
  const bool both = prompts && a.b.seqs > 1;
  s.prompt.shared = s.step.shared = both;
  auto cuts = [&](const PgCut& c) { return pg_splits(pg_most(cap, cap, c), c.least) > 1; };
  if ((prompts && cuts(s.prompt)) || ((both || !prompts) && cuts(s.step))) {
    uint8_t* work = nullptr;
    if (int rc = illp::workspace(p, st, &work)) return rc;
    s.step_work = illp::work_of(work, s.step.log, s.step.M, d.head_dim);
    s.prompt_work = illp::work_of(work + illp::work_size(s.step.log, s.step.M, d.head_dim), s.prompt.log, s.prompt.M, d.head_dim);
  }
  // (below 2^24 workgroups: rows x heads are at most 2^26, sequences x heads 2^22)
  const int64_t steps = both || !prompts ? pg_grid(a.b.seqs, a.b.rows, !a.b.row0, cap, s.step) : 0;
  s.prompts = prompts ? (int)pg_grid(a.b.seqs, a.b.rows, !a.b.row0, cap, s.prompt) : 0;
  if (!s.prompts && !steps) return ILL_OK;
  if (d.dtype == ILL_F16) {
    if (d.head_dim == 64) HCK((illp::launch_attend<PG_F16, 64>(s, steps, st)));
    else HCK((illp::launch_attend<PG_F16, 128>(s, steps, st)));
  } else {
    if (d.head_dim == 64) HCK((illp::launch_attend<PG_BF16, 64>(s, steps, st)));
    else HCK((illp::launch_attend<PG_BF16, 128>(s, steps, st)));
  }
  return ILL_OK;
}

}  // extern "C"

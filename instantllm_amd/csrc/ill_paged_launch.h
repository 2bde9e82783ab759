// Launches of the paged-cache kernels, for caches of 16-bit values and for microscaled ones: each kind is instantiated in a
// translation unit of its own.
#pragma once
#include "ill_launch.h"
#include "ill_paged.h"

namespace illp {

// x_type, type, out_type: ILL_F32 ..; `steps`: workgroups of the step kernel.
hipError_t append_16(int x_type, int type, const PgAppend& a, int D, int R, hipStream_t st);
hipError_t append_mx(int x_type, int type, const PgAppend& a, int D, int R, hipStream_t st);
hipError_t read_16(int out_type, int type, const PgRead& a, int D, int R, hipStream_t st);
hipError_t read_mx(int out_type, const PgRead& a, int D, int R, hipStream_t st);
hipError_t attend_16(int type, int D, const PgBoth& s, int64_t steps, hipStream_t st);
hipError_t attend_mx(int type, int D, const PgBoth& s, int64_t steps, hipStream_t st);

namespace {

template <int TC, int D, bool FINE, bool MX>
hipError_t launch_attend(const PgBoth& s, int64_t steps, hipStream_t st) {
  if (!s.prompts) return launch(pg_step_kernel<TC, D, FINE, MX>, steps, PG_THREADS, 0, st, PgStep{s.a, s.step, s.step_work});
  if (!steps) return launch(pg_prompt_kernel<TC, D, FINE, MX>, s.prompts, PG_THREADS, 0, st, PgStep{s.a, s.prompt, s.prompt_work});
  return launch(pg_both_kernel<TC, D, FINE, MX>, s.prompts + steps, PG_THREADS, 0, st, s);
}
template <int TC, bool MX>
hipError_t launch_attend(int D, const PgBoth& s, int64_t steps, hipStream_t st) {
  if (D == 64) return s.a.out_f32 ? launch_attend<TC, 64, true, MX>(s, steps, st) : launch_attend<TC, 64, false, MX>(s, steps, st);
  return s.a.out_f32 ? launch_attend<TC, 128, true, MX>(s, steps, st) : launch_attend<TC, 128, false, MX>(s, steps, st);
}

template <int TX, int TC, bool MX>
hipError_t launch_append(const PgAppend& a, int D, int R, hipStream_t st) {
  const int64_t blocks = ((int64_t)a.b.rows + R - 1) / R;
  const int lds = R * 8 + (R + 1) / 2 * 8 + R * (a.rot / 2) * 8 + (MX ? R * 4 : 0);
  return D == 64 ? launch(pg_append_kernel<TX, TC, 64, MX>, blocks, 256, lds, st, a, R) : launch(pg_append_kernel<TX, TC, 128, MX>, blocks, 256, lds, st, a, R);
}
template <bool MX>
hipError_t launch_append(int x_type, int type, const PgAppend& a, int D, int R, hipStream_t st) {
  if (type == ILL_F16) return x_type == ILL_F32 ? launch_append<PG_F32, PG_F16, MX>(a, D, R, st) : launch_append<PG_F16, PG_F16, MX>(a, D, R, st);
  return x_type == ILL_F32 ? launch_append<PG_F32, PG_BF16, MX>(a, D, R, st) : launch_append<PG_BF16, PG_BF16, MX>(a, D, R, st);
}

template <int TO, int TC, bool MX>
hipError_t launch_read(const PgRead& a, int D, int R, hipStream_t st) {
  const int64_t blocks = ((int64_t)a.b.rows + R - 1) / R;
  return D == 64 ? launch(pg_read_kernel<TO, TC, MX, 64>, blocks, 256, 12 * R, st, a, R) : launch(pg_read_kernel<TO, TC, MX, 128>, blocks, 256, 12 * R, st, a, R);
}

}  // namespace
}  // namespace illp

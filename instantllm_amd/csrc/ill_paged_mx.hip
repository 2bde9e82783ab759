// The paged-cache kernels of microscaled caches.
#include <hip/hip_runtime.h>

#include "ill_error.h"
#include "ill_paged_launch.h"

namespace illp {

hipError_t append_mx(int x_type, int type, const PgAppend& a, int D, int R, hipStream_t st) { return launch_append<true>(x_type, type, a, D, R, st); }

hipError_t read_mx(int out_type, const PgRead& a, int D, int R, hipStream_t st) {   // (TC says nothing here)
  return out_type == ILL_F32 ? launch_read<PG_F32, PG_F32, true>(a, D, R, st)
                             : out_type == ILL_F16 ? launch_read<PG_F16, PG_F32, true>(a, D, R, st) : launch_read<PG_BF16, PG_F32, true>(a, D, R, st);
}

hipError_t attend_mx(int type, int D, const PgBoth& s, int64_t steps, hipStream_t st) {
  return type == ILL_F16 ? launch_attend<PG_F16, true>(D, s, steps, st) : launch_attend<PG_BF16, true>(D, s, steps, st);
}

}  // namespace illp

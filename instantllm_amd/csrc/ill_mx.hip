// The microscaled operators (ill_mx_* in include/ill_hip.h): entry points and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <optional>

#include "ill_error.h"
#include "ill_launch.h"
#include "ill_mx.h"
#include "ill_mx_check.h"

namespace illm {
namespace {

using illp::launch;

// While this lives the current device is the one that the stream belongs to (a default stream belongs to the current one).
struct OnStream {
  int rc = ILL_OK;
  std::optional<illp::OnDevice> on;
  explicit OnStream(hipStream_t st) {
    if (!st || st == hipStreamLegacy || st == hipStreamPerThread) return;
    int dev = 0;
    if (hipStreamGetDevice(st, &dev) != hipSuccess) {
      rc = fail(ILL_E_HIP, "mx: the stream belongs to no device");
      return;
    }
    on.emplace(dev);
    rc = on->rc;
  }
};

template <int T, int F>
hipError_t launch_rows(bool back, const MxRows& a, hipStream_t st) {
  const int64_t blocks = std::min<int64_t>((a.items + 255ll) / 256, 1 << 16);
  return back ? launch(mx_dequantize_kernel<T, F>, blocks, 256, 0, st, a) : launch(mx_quantize_kernel<T, F>, blocks, 256, 0, st, a);
}
template <int F>
hipError_t launch_rows(bool back, int dtype, const MxRows& a, hipStream_t st) {
  return dtype == ILL_F32 ? launch_rows<PG_F32, F>(back, a, st) : dtype == ILL_F16 ? launch_rows<PG_F16, F>(back, a, st) : launch_rows<PG_BF16, F>(back, a, st);
}

int rows(bool back, int format, int dtype, const void* x, int64_t stride, int64_t rows, int64_t cols, const void* codes, const void* powers, void* stream) {
  if (int rc = check_rows(format, dtype, x, stride, rows, cols, codes, powers)) return rc;
  if (!rows) return ILL_OK;
  hipStream_t st = (hipStream_t)stream;
  OnStream on(st);
  if (on.rc) return on.rc;
  const MxRows a{(uint8_t*)x, (uint8_t*)codes, (uint8_t*)powers, stride, (uint32_t)(rows * cols / 8), (uint32_t)(cols / 8)};
  HCK(format == ILL_MXF8 ? launch_rows<MX_F8>(back, dtype, a, st) : launch_rows<MX_F4>(back, dtype, a, st));
  return ILL_OK;
}

template <int F, bool FINE>
hipError_t launch_few(const MxProduct& p, hipStream_t st) {
  const int tiles = (p.cols + 15) / 16;
  return launch(mx_few_kernel<F, FINE>, (int64_t)((p.rows + 15) / 16) * tiles, 256, 0, st, p, tiles);
}
template <int F, bool FINE, int L>
hipError_t launch_slice(const MxProduct& p, hipStream_t st) {
  using S = MxSlice<FINE, L>;
  const int tiles = (p.cols + 15) / 16, groups = S::WAVES / L;
  return launch(mx_slice_kernel<F, FINE, L>, std::min(256 * S::EACH, (tiles + groups - 1) / groups), 64 * S::WAVES, 0, st, p, tiles);
}
template <int F, bool FINE, int R>   // (for rows that take up to 64 KB of LDS)
hipError_t launch_wide(const MxProduct& p, hipStream_t st) {
  const int tiles = (p.cols + 15) / 16, lds = MxWide<F, FINE, R>::lds(p.inner), each = std::max(1, std::min(4, (160 << 10) / lds));
  return launch(mx_wide_kernel<F, FINE, R>, std::min(256 * each, (tiles + 3) / 4), 256, lds, st, p, tiles);
}
template <int F, bool FINE, int TC, int TR, int S, bool ODD = false, int WR = 2>
hipError_t launch_many(const MxProduct& p, hipStream_t st) {
  using T = MxTile<F, TC, TR, S, WR>;
  const int tiles_c = (p.cols + T::C - 1) / T::C, tiles = tiles_c * ((p.rows + T::R - 1) / T::R);
  return launch(mx_many_kernel<F, FINE, TC, TR, S, ODD, WR>, (tiles + 7) / 8 * 8ll, 128 * WR, 0, st, p, tiles_c, tiles);
}
inline int64_t mx_tiles(const MxProduct& p, int c, int r) { return (int64_t)((p.cols + c - 1) / c) * ((p.rows + r - 1) / r); }
template <int F, bool FINE, bool ODD>
hipError_t launch_tiles(const MxProduct& p, hipStream_t st) {
  auto tiles = [&](int c, int r) { return mx_tiles(p, c, r); };
  // Tiles as large as leave enough of them for 256 CUs, of four waves or (8) eight: two for each SIMD where a CU has one workgroup. Columns x rows, us (the same
  // card for the numbers between two semicolons; the largest ones differ by 15% from card to card). mxf8 rows, 256 x 128 / 128 x 128 / 128 x 64 / 64 x 64: 8192 x 8192 x 8192
  // 449 / 519 / 675 / 927; 3000 x 5000 x 4096 (480 tiles of 256 x 128) 64 / 71 / 88; 512 x 896 x 4864 (112 of 64 x 64) 34 / 24 / 18 / 15. 128 x 128 (8) / 128 x 128 / 128 x 64:
  // 3000 x 3000 x 4096 (576 of 128 x 128) 50 / 59; 2048 x 2048 x 4096 (256) 22.7 / 32 / 25.5; 4096 x 896 x 4864 (224) 25.5 / - / 28.4; 5001 x 896 x 4864 (280) 39 / 41 / 35; against
  // 256 x 128: 3000 x 5000 x 4096 75 / 69, 8192 x 8192 x 8192 659 / 567.
  // mxf4, 256 x 256 (8) / 256 x 256: 8192 x 8192 x 8192 306 / 323; 4096 x 4096 x 4096 43 / 47. 256 x 256 / 128 x 256 / 128 x 128 / 64 x 64: 8192 x 8192 x 8192 312 / 335 / 407 /
  // 768; 3000 x 5000 x 4096 (240) 48 / 50 / 57; 512 x 896 x 4864 - / 27 / 19 / 13.5. 256 x 256 (8) / 128 x 256: 8192 x 8192 x 2048 94 / 95; 8192 x 8192 x 1024 62 / 59. 128 x 128 (8) / 128 x 128:
  // 2048 x 2048 x 4096 (256) 17.7 / 22; 4096 x 896 x 4864 (224) 19.5 / 25; 3000 x 3000 x 4096 (576) 41 / 37; 3000 x 5000 x 1024 (960) 21 / 19.3.
  // ODD, chosen likewise / 128 x 64 (mxf8) and 128 x 128 (mxf4): mxf8 8192 x 8192 x 8160 620 / 876; 3000 x 5000 x 4064 73 / 109; 4096 x 9728 x 928 61.5 / 73.5; 2048 x 2048 x 4064 30.6 / 39.8;
  // mxf4 8192 x 8192 x 8160 412 / 621; 2048 x 2048 x 4064 25 / 37; 4096 x 9728 x 928 57 / 55.
  // The limits between them. mxf8 128 x 128 (8) / 128 x 64, by the number of the former: 2176 x 2176 x 4096 (289) 30.9 / 30.5; 2560 x 2304 x 4096 (360) 33.3 / 33.4; 2560 x 2560 x 1024 (400) 13.0 /
  // 13.9; 2688 x 2688 x 4096 (441) 33.8 / 41.3, over 896 12.6 / 13.9. mxf4 256 x 256 (8) / 128 x 256, 8192 x 8192 over 2048, 2560, 3328 and 3968: 109 / 109, 127 / 130, 153 / 163, 181 / 197;
  // 3000 x 5000 over 3584 (240 of the former) 35 / 40, with 128 x 128 45.
  // Float32 outputs of mxf8 rows, 128 x 64 / 64 x 64: 512 x 896 x 4864 (112 of 64 x 64) 29.1 / 19.3; 4096 x 1152 x 896 (1152) 16.3 / 17.1; 5001 x 896 x 4864 57 / 60; 3000 x 5000 x 4096 128 / 147.
  // No wider than the columns ask for, or products are thrown away: 64 x 64 for up to 64 columns (against the tiles that numbers alone choose: 65536 x 64 x 896 in mxf8 12.8 / 18.9, over
  // 4096 68 / 74; 100000 x 32 x 4096 97 / 118, in mxf4 60 / 77; 65536 x 64 x 4096 in mxf4 43 / 45, with float32 outputs 70 / 81), 256 columns a tile from 129 on (65536 x 128 x 4096 in
  // mxf8 71 / 78, over 896 15.2 / 19.9; in mxf4 42 / 48; 65536 x 100 x 4096 74 / 80 and 48 / 52).
  if (tiles(64, 64) <= 512 || p.rows <= 64 || p.cols <= 64) return launch_many<F, FINE, 1, 1, 3, ODD>(p, st);
  if constexpr (FINE) {
    return launch_many<F, FINE, 2, 1, 2, ODD>(p, st);
  } else if constexpr (F == MX_F8) {
    if (tiles(256, 128) >= 384 && p.cols > 128) return launch_many<F, FINE, 4, 2, 2, ODD>(p, st);
    return tiles(128, 128) >= 384 || tiles(128, 128) <= 256 ? launch_many<F, FINE, 2, 1, 3, ODD, 4>(p, st) : launch_many<F, FINE, 2, 1, 2, ODD>(p, st);
  } else {
    if (tiles(256, 256) >= 240 && p.inner > 16 * 128 && p.cols > 128) return launch_many<F, FINE, 4, 2, 3, ODD, 4>(p, st);
    if (tiles(128, 256) >= 512) return launch_many<F, FINE, 2, 4, 2, ODD>(p, st);
    return tiles(128, 128) <= 256 ? launch_many<F, FINE, 2, 1, 4, ODD, 4>(p, st) : launch_many<F, FINE, 2, 2, 2, ODD>(p, st);
  }
}

template <int F, bool FINE>
hipError_t launch_product(const MxProduct& p, hipStream_t st) {
  const int steps = (p.inner + 127) / 128;
  // Up to 16 rows: slices from 512 tiles of 16 columns on (us, against the four waves of a workgroup that share a tile, mxf8 unless said otherwise: 16 x 9728 x 896
  // 5.2 / 6.3, 16 x 16384 x 4096 14.3 / 19.9, mxf4 16 x 32000 x 8192 37 / 61; but 1 x 896 x 4864 7.8 / 4.7). For float32 outputs, as bf16 values, their rows take too many
  // registers: 1 x 151936 x 896 23.4, with the rows in LDS 18.6. Slices of up to 32 steps: 16 x 16384 x 2048 10.8 / 11.3, 16 x 16384 x 4096 16.3 / 20.0, 16 x 151936 x 1536 40 / 69,
  // 4 x 32000 x 4096 25.1 / 25.7; fewer rows and columns would do without (1 x 16384 x 2048 9.6 / 7.2, 8 rows 10.0 / 9.3, 16 x 8192 x 1152 5.0 / 4.4). Past 32 steps eight waves leave each
  // half the registers, and 118 of them spilled: 16 x 32000 x 8192 92.5 / 73.0, 1 x 32000 x 8192 89 / 41. Up to 32 rows in LDS, against tiles of 64 x 64: 32 x 151936 x 896 22.9 / 28.2.
  if (p.rows <= 16 && p.cols >= 8192 && steps <= (FINE ? 32 : 64)) {
    if constexpr (FINE) {
      if (steps <= 8) return launch_wide<F, FINE, 1>(p, st);
    } else {
      if (steps <= 8) return launch_slice<F, FINE, 1>(p, st);
      if (steps > 32) return launch_slice<F, FINE, 8>(p, st);
    }
    return steps <= 16 ? launch_slice<F, FINE, 2>(p, st) : launch_slice<F, FINE, 4>(p, st);
  }
  if (p.rows <= 16) return launch_few<F, FINE>(p, st);
  if (p.rows <= 32 && p.cols >= 16384 && MxWide<F, FINE, 2>::lds(p.inner) <= 64 << 10) return launch_wide<F, FINE, 2>(p, st);
  // Few tiles over a long inner size: 16 rows at a time, as above (64 x 896 x 4864 6.7 us, 14 tiles of 64 x 64 13).
  if (p.rows <= 64 && mx_tiles(p, 64, 64) < 64 && steps > 16) return launch_few<F, FINE>(p, st);
  return p.inner % 128 ? launch_tiles<F, FINE, true>(p, st) : launch_tiles<F, FINE, false>(p, st);
}

}  // namespace
}  // namespace illm

extern "C" {

int ill_mx_quantize(int format, int dtype, const void* x, int64_t x_stride, int64_t rows, int64_t cols, void* codes, void* powers, void* stream) {
  return illm::rows(false, format, dtype, x, x_stride, rows, cols, codes, powers, stream);
}

int ill_mx_dequantize(int format, int dtype, const void* codes, const void* powers, int64_t rows, int64_t cols, void* y, int64_t y_stride, void* stream) {
  return illm::rows(true, format, dtype, y, y_stride, rows, cols, codes, powers, stream);
}

int ill_mx_product(int x_format, const void* x, const void* x_powers, const void* w, const void* w_powers, int64_t rows, int64_t cols, int64_t inner,
                   const float* bias, int y_dtype, void* y, int64_t y_stride, void* stream) {
  if (int rc = illm::check_product(x_format, x, x_powers, w, w_powers, bias, y, y_stride, y_dtype, rows, cols, inner)) return rc;
  if (!rows) return ILL_OK;
  hipStream_t st = (hipStream_t)stream;
  illm::OnStream on(st);
  if (on.rc) return on.rc;
  const int size = y_dtype == ILL_F32 ? 4 : 2;
  const int wide = y_stride % (16 / size) == 0 && illm::aligned(y, 16) ? 2 : y_stride % 4 == 0 && illm::aligned(y, 4 * size) ? 1 : 0;
  const MxProduct p{(const uint8_t*)x, (const uint8_t*)x_powers, (const uint8_t*)w, (const uint8_t*)w_powers, bias, y, y_stride,
                    (int)rows, (int)cols, (int)inner, y_dtype, wide};
  if (x_format == ILL_MXF4) HCK((illm::launch_product<MX_F4, false>(p, st)));
  else if (y_dtype == ILL_F32) HCK((illm::launch_product<MX_F8, true>(p, st)));
  else HCK((illm::launch_product<MX_F8, false>(p, st)));
  return ILL_OK;
}

}  // extern "C"

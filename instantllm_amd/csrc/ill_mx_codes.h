// Microscaled codes: blocks of 32 values that share a power of two, whose byte e stands for 2^(e - 127), 255 for a block of NaN.
#pragma once
#include "ill_values.h"

enum MxFormat { MX_F8 = 0, MX_F4 = 4 };   // as the matrix instructions name their operands' types: e4m3, e2m1

typedef short v2s __attribute__((ext_vector_type(2)));

// A block's power of two as a float, which the conversions read the exponent of only: 0 is 2^-127, 255 NaN.
__device__ __forceinline__ float mx_power(uint32_t byte) { return __uint_as_float(byte << 23); }

// Bytes of `n` codes.
template <int F>
constexpr int mx_bytes(int n) { return F == MX_F8 ? n : n / 2; }

// The power's byte of a block whose largest size has these bits (0: no value; from 0x7F800000 on: an infinity or NaN).
template <int F>
__device__ __forceinline__ uint32_t mx_power_of(uint32_t most) {
  const int e = (int)(most >> 23);
  return e == 255 ? 255 : (uint32_t)max(e - (F == MX_F8 ? 8 : 2), 0);
}
// Eight values of a block as codes, rounded to nearest, ties to even. The conversion to e4m3 makes what rounds past 448 a NaN: its operands end there.
template <int F>
__device__ __forceinline__ uint2 mx_codes(const float* x, uint32_t byte) {
  const float p = mx_power(byte);
  if constexpr (F == MX_F4) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], p, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], p, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], p, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], p, 3);
    return {byte == 255 ? 0 : c, 0};
  } else {
    const float most = __uint_as_float((byte + 8) << 23 | 0x600000);   // 448 2^(byte - 127)
    v2s c[2] = {};
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = __builtin_amdgcn_fmed3f(x[i], -most, most);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      c[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c[i], y[4 * i], y[4 * i + 1], p, false);
      c[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c[i], y[4 * i + 2], y[4 * i + 3], p, true);
    }
    const uint2 r = __builtin_bit_cast(uint2, c);
    return {byte == 255 ? 0 : r.x, byte == 255 ? 0 : r.y};
  }
}
// Eight values of codes (mxf8: eight bytes, mxf4: the first four).
template <int F>
__device__ __forceinline__ void mx_values(uint2 c, uint32_t byte, float* x) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const float p = mx_power(byte);
  v2f y[4];
  if constexpr (F == MX_F4) {
    y[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, p, 0);
    y[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, p, 1);
    y[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, p, 2);
    y[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, p, 3);
  } else {
    y[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, p, false);
    y[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, p, true);
    y[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, p, false);
    y[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, p, true);
  }
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = y[i / 2][i & 1];
}
// Eight codes as 16-bit values of type T. bf16 has an exact place for every code and power (but below 2^-133 and above its range); f16 for
// values from 2^-14 up to 65504, below it they are off by 2^-25 at most, and infinite above it.
template <int T, int F>
__device__ __forceinline__ uint4 mx_16(uint2 c, uint32_t byte) {
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  const float p = mx_power(byte);
  if constexpr (T == PG_F16) {
    static_assert(F == MX_F8, "e4m3");
    const v2h y[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c.x, p, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c.x, p, true),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c.y, p, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c.y, p, true)};
    return __builtin_bit_cast(uint4, y);
  } else if constexpr (F == MX_F4) {
    const v2bf y[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.x, p, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.x, p, 1),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.x, p, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.x, p, 3)};
    return __builtin_bit_cast(uint4, y);
  } else {
    const v2bf y[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, p, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, p, true),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, p, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, p, true)};
    return __builtin_bit_cast(uint4, y);
  }
}

// Values of the three element types as floats, and back.
#pragma once
#include "ill_device.h"

enum PgType { PG_F32 = 0, PG_F16 = 1, PG_BF16 = 2 };   // ILL_F32, ILL_F16, ILL_BF16

// 16-bit values as floats, and back with one rounding to nearest, ties to even.
template <int T>
__device__ __forceinline__ void pg_unpack2(uint32_t w, float* x) {
  if constexpr (T == PG_BF16) {
    x[0] = __uint_as_float(w << 16);
    x[1] = __uint_as_float(w & 0xFFFF0000u);
  } else {
    x[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)w);
    x[1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  }
}
template <int T>
__device__ __forceinline__ void pg_unpack(const uint4* p, float* x) {   // eight values of type T
  if constexpr (T == PG_F32) {
    *(uint4*)x = p[0];
    *(uint4*)(x + 4) = p[1];
  } else {
    const uint32_t w[4] = {p->x, p->y, p->z, p->w};
#pragma unroll
    for (int i = 0; i < 4; i++) pg_unpack2<T>(w[i], x + 2 * i);
  }
}
template <int T>
__device__ __forceinline__ uint32_t pg_pack2(float a, float b) {   // (as a pair: one instruction)
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  if constexpr (T == PG_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2bf));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2h));
}
template <int T>
__device__ __forceinline__ uint4 pg_pack8(const float* x) {
  return {pg_pack2<T>(x[0], x[1]), pg_pack2<T>(x[2], x[3]), pg_pack2<T>(x[4], x[5]), pg_pack2<T>(x[6], x[7])};
}

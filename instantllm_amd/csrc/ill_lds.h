// Loads from memory straight into LDS, the waits that belong to them, and barriers: for kernels that keep several such loads in flight.
#pragma once
#include <type_traits>
#include <utility>
#include "ill_device.h"

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
#define LAS __attribute__((address_space(3)))   // LDS: named, as GAS is, or an access counts as one to memory too

// 16 bytes from base + each lane's offset into LDS, lane i's at lds + 16 i. In inline assembly, because the
// compiler cannot tell the buffers apart and would wait for every load in flight before each LDS read;
// the kernels wait themselves (PG_WAIT), and extra loads of the compiler's own only make that wait longer.
// `base` may have been written by a vector instruction just before (v_readlane, also from a spill): a load may read it five
// wait states later, which the compiler, not seeing the load, does not ensure.
template <int AT>
__device__ __forceinline__ void pg_dma16(const void* base, uint32_t off, uint32_t lds) {   // to lds + AT + 16 i; base and lds: the same for every lane
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base), "n"(AT) : "memory", "scc", "m0");
}
template <int AT>
__device__ __forceinline__ void pg_dma4(const void* base, uint32_t off, uint32_t lds) {   // four bytes of each lane, to lds + AT + 4 i
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base), "n"(AT) : "memory", "scc", "m0");
}
__device__ __forceinline__ uint32_t pg_lds_at(const void* p) {   // an LDS address, as every lane's
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const LAS uint8_t*)p);
}
// Calls f with the constants 0 .. N - 1.
template <int N, class F>
__device__ __forceinline__ void pg_each(F&& f) {
  [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}
// The compiler's own loads so far have arrived, and it knows it (else it would wait for them, and with them for every later
// load of pg_dma16, where it first uses them inside a loop).
#define PG_WAIT_OWN() __builtin_amdgcn_s_waitcnt(0x0F70)   // vmcnt(0)
#define PG_WAIT(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")
#define PG_TURN()                                                        \
  do { /* a barrier that waits for no loads, and that no work moves over */ \
    __builtin_amdgcn_sched_barrier(0);                                   \
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      \
    __builtin_amdgcn_sched_barrier(0);                                   \
  } while (0)
#define PG_WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

// Loads that go straight to LDS, and the transposing LDS reads.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nvdsa {

// 16 bytes a lane from base + offset straight to LDS at `lds` + 16 * lane (the
// same for the wave).  Counts in vmcnt like a load; has no register to return.
__device__ inline void load_to_lds(const uint8_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ inline void load_to_lds(const uint8_t* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
// The same from base + offset + OFFSET to `lds` + `more` + OFFSET + 16 * lane.
template <int OFFSET>
__device__ inline void load_to_lds(const uint8_t* base, uint32_t offset, uint32_t lds, uint32_t more) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3 offset:%4" ::"s"(lds), "s"(more), "v"(offset),
               "s"(base), "n"(OFFSET)
               : "memory", "m0", "scc");
}
template <int N>
__device__ inline void wait_loads() {  // all but the wave's newest N are done
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ inline uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

// ds_read_b64_tr_b16 (gfx950): within each 16-lane group, lane i reads four
// 16-bit values M[i][0..3] at its address; lane l receives
// M[4j + (l >> 2)][l & 3] for j = 0..3.
__device__ inline uint2 read_tr16(const uint8_t* p) {
  typedef short v4i16 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(const_cast<uint8_t*>(p))));
}
__device__ inline uint2 read_tr16(uint32_t lds) {  // (by address)
  typedef short v4i16 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4i16*>(lds)));
}

}  // namespace nvdsa

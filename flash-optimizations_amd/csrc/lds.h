// Copies from memory to LDS, LDS accesses by plain address, and the vector types around
// them, shared by the decodes that stage records as they are stored.
#pragma once
#include "remnant_device.h"

namespace {

using namespace rm;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

// Copies HBM -> LDS: 16 bytes a lane to lds + 16 lane. The LDS address is a plain number,
// so that the compiler ties the copies to no array; wait_copies() orders them.
__device__ __forceinline__ void copy16(const void* src, uint32_t lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)__builtin_amdgcn_readfirstlane(lds),
                                   16, 0, 0);
}
__device__ __forceinline__ void copy4(const void* src, uint32_t lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)__builtin_amdgcn_readfirstlane(lds),
                                   4, 0, 0);
}
// Until at most kLater vector loads issued since are in flight.
template <int kLater>
__device__ __forceinline__ void wait_copies() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kLater & 15) | ((kLater >> 4) << 14));
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  __builtin_amdgcn_sched_barrier(0);
}
template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)at;
}
template <class T>
__device__ __forceinline__ void lds_write(uint32_t at, T v) {
  *(__attribute__((address_space(3))) T*)(uintptr_t)at = v;
}
// Barrier that orders LDS accesses only: loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
__device__ __forceinline__ uint32_t sub_sat(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, a),
                                                          __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

}  // namespace

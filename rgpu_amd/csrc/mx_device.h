// Device-side helpers shared by the microscaled kernels.
#pragma once

#include <hip/hip_runtime.h>

namespace rt_mx {

typedef unsigned int u2 __attribute__((ext_vector_type(2)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

// 16 bytes that are read or written once, from and to any address that suits
// their element: past the caches (streams of values; 8192 x 4096 bf16 into 8 bits
// from HBM 34.9 us through them, 21.0 past).
typedef unsigned int u4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ inline u4 load_once(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u4_any*>(p));
}
__device__ inline void store_once(void* p, u4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u4_any*>(p)); }

// 2^(byte - 127), or NaN for 255.
__device__ inline float scale_of(unsigned byte) {
  const unsigned bits = byte == 0 ? 0x00400000u : byte << 23;
  return __uint_as_float(byte == 255u ? 0x7fc00000u : bits);
}

// Round to nearest even; a NaN stays one.
__device__ inline unsigned short f32_to_bf16(float x) {
  const unsigned u = __float_as_uint(x);
  const unsigned rne = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
  return (unsigned short)((u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 0x40u : rne);
}

}  // namespace rt_mx

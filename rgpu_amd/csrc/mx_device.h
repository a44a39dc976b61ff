// Device-side helpers shared by the microscaled kernels.
#pragma once

#include <hip/hip_runtime.h>

namespace rt_mx {

typedef unsigned int u2 __attribute__((ext_vector_type(2)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

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

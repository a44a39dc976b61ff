// Microscaled tensors: conversion to and from f32/bf16/f16, and the ReLU mask
// of an 8-bit saved activation.  The layout is rtensor_hip.h's; all HBM-bound.
// Measured, from HBM: 8192 x 4096 bf16 into 8 bits 19.7 us (5.2 TB/s), back 16.3
// (6.2); f32 [4096, 4096] into its transpose in 4 bits 16.7 (4.6); a copy of 1 GiB
// 5.1 TB/s.  Below about 4 MB a launch's 3.2 us.
//
// Quantisation of a block of 32: with m·2^E, 1 <= m < 2, its largest finite
// magnitude, the least e with m·2^E <= MAX·2^e is E - T, plus one if m is
// above MAX's mantissa (MAX = 6 = 1.5·2^2 or 448 = 1.75·2^8), but not below
// -127; so the scale byte is the exponent field of that magnitude less T (plus
// one), and no element can round past MAX.  x·2^-e is exact, so the one
// rounding is the hardware's conversion (round to nearest even).

#include <algorithm>
#include <type_traits>

#include "device_util.h"
#include "mx_device.h"
#include "rt_internal.h"

namespace {

using rt_mx::u2;
using rt_mx::u4;

typedef float f2 __attribute__((ext_vector_type(2)));
typedef short s2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ inline float get(float v) { return v; }
  static __device__ inline float put(float v) { return v; }
};
struct bf16_bits {
  unsigned short u;
};
template <>
struct Elem<bf16_bits> {
  static __device__ inline float get(bf16_bits v) { return __uint_as_float((unsigned)v.u << 16); }
  static __device__ inline bf16_bits put(float v) { return bf16_bits{rt_mx::f32_to_bf16(v)}; }
};
template <>
struct Elem<_Float16> {
  static __device__ inline float get(_Float16 v) { return (float)v; }
  static __device__ inline _Float16 put(float v) { return (_Float16)v; }
};

// The scale byte for the largest magnitude's bits of a block.
template <bool FP4>
__device__ inline unsigned scale_byte(unsigned amax) {
  constexpr unsigned top = FP4 ? 2 : 8, mant = FP4 ? 0x400000 : 0x600000;
  const unsigned e = (amax >> 23) + ((amax & 0x7fffffu) > mant ? 1u : 0u);
  return e > top ? e - top : 0u;
}

// What a value's magnitude counts for in the block's maximum: RT_MXFP8 leaves
// out infinities and NaN (they become NaN codes beside whatever scale the
// others want), RT_MXFP4 keeps them (its block becomes NaN).
template <bool FP4>
__device__ inline unsigned magnitude(float v) {
  const unsigned m = __float_as_uint(v) & 0x7fffffffu;
  return FP4 || m < 0x7f800000u ? m : 0u;
}

// Four values as four 4-bit (low 16 bits of the result) or 8-bit codes.
template <bool FP4>
__device__ inline unsigned encode4(const float* v, float scale) {
  if constexpr (FP4) {
    unsigned w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1) & 0xffffu;
  } else {
    s2 h = {0, 0};
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, v[0], v[1], scale, false);
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, v[2], v[3], scale, true);
    const unsigned w = __builtin_bit_cast(unsigned, h);
    // Zero codes take 0x80 where the value was positive, 0 where it was not.
    const unsigned nonzero = ((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u;
    unsigned pos = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) pos |= v[i] > 0.0f ? 0x80u << (8 * i) : 0u;
    return (w & (0x7f7f7f7fu | nonzero)) | (pos & ~nonzero);
  }
}

// Stores the scale bytes of a 64-row group of one step, gathered in LDS in the
// order of the layout.  Rows past the last one hold zeros.
__device__ inline void store_scales(const unsigned* sc, unsigned char* scales, long long step, long long groups,
                                    long long group) {
  if (threadIdx.x < 64)
    reinterpret_cast<unsigned*>(scales)[(step * groups + group) * 64 + threadIdx.x] = sc[threadIdx.x];
}

// The largest m of LANES (4 or 8) neighbouring lanes, in each of them.
template <int LANES>
__device__ inline unsigned block_max(unsigned m) {
  auto with = [&](auto ctrl) {
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, decltype(ctrl)::value, 0xF, 0xF, false));
  };
  with(std::integral_constant<int, 0xB1>{});                        // quad_perm [1, 0, 3, 2]
  with(std::integral_constant<int, 0x4E>{});                        // quad_perm [2, 3, 0, 1]
  if constexpr (LANES == 8) with(std::integral_constant<int, 0x141>{});  // row_half_mirror: the other four
  return m;
}

// The values of w from the n-th on (0 <= n <= 16 / sizeof(T)), then zeros.
template <typename T>
__device__ inline u4 from_element(u4 w, int n) {
  const int bytes = n * (int)sizeof(T);
  if (bytes & 16) w = u4{0, 0, 0, 0};
  if (bytes & 8) w = u4{w[2], w[3], 0, 0};
  if (bytes & 4) w = u4{w[1], w[2], w[3], 0};
  if constexpr (sizeof(T) == 2) {
    const unsigned sh = 8 * (bytes & 2);
    w = u4{__builtin_amdgcn_alignbit(w[1], w[0], sh), __builtin_amdgcn_alignbit(w[2], w[1], sh),
           __builtin_amdgcn_alignbit(w[3], w[2], sh), w[3] >> sh};
  }
  return w;
}

// A block of threads takes 64 rows of one step (128 columns): lanes hold V
// consecutive values (16 bytes), so 32 / V lanes share a block and find its
// maximum by exchange.
template <typename T, bool FP4>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ src, long long rows, long long cols,
                                                       unsigned char* __restrict__ codes,
                                                       unsigned char* __restrict__ scales, long long steps,
                                                       long long groups, long long block0) {
  constexpr int V = 16 / sizeof(T), LANES = 128 / V, ROWS = 256 / LANES, PASSES = 64 / ROWS;
  __shared__ unsigned sc[64];
  const long long block = block0 + blockIdx.x, step = block % steps, group = block / steps;
  const int lane = threadIdx.x % LANES, row0 = threadIdx.x / LANES;
  const long long col = step * 128 + lane * V;
  if (threadIdx.x < 64) sc[threadIdx.x] = 0;
  __syncthreads();
  T raw[PASSES][V];
  const long long row_bytes = steps * (FP4 ? 64 : 128);
  auto finish = [&](auto whole) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int r = row0 + p * ROWS;
      float v[V];
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = Elem<T>::get(raw[p][i]);
        m = max(m, magnitude<FP4>(v[i]));
      }
      m = block_max<32 / V>(m);
      const unsigned byte = FP4 && m >= 0x7f800000u ? 255u : scale_byte<FP4>(m);
      const float scale = rt_mx::scale_of(min(byte, 254u));
      unsigned w[V / 4];
#pragma unroll
      for (int i = 0; i < V / 4; ++i) w[i] = encode4<FP4>(v + 4 * i, scale);
      if (decltype(whole)::value || group * 64 + r < rows) {
        unsigned char* out = codes + (group * 64 + r) * row_bytes + (step * 128 + lane * V) / (FP4 ? 2 : 1);
        if constexpr (FP4 && V == 4) *reinterpret_cast<unsigned short*>(out) = (unsigned short)w[0];
        else if constexpr (FP4) *reinterpret_cast<unsigned*>(out) = w[0] | (w[1] << 16);
        else if constexpr (V == 4) *reinterpret_cast<unsigned*>(out) = w[0];
        else *reinterpret_cast<u2*>(out) = u2{w[0], w[1]};
        if (lane * V % 32 == 0)
          reinterpret_cast<unsigned char*>(sc)[4 * (16 * (lane * V / 32) + r % 16) + r / 16] = (unsigned char)byte;
      }
    }
  };
  if (group * 64 + 64 <= rows && step * 128 + 128 <= cols) {
    const T* at = src + (group * 64 + row0) * cols + col;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const u4 w = rt_mx::load_once(at + p * ROWS * cols);
      __builtin_memcpy(raw[p], &w, 16);
    }
    finish(std::true_type());
  } else if (cols >= V) {
    // Loads without branches, which would wait for one another (1500 x 1003 f32
    // 4.7 us that way, 3.8 this way): a lane past the row's end, or across it,
    // takes the row's last V values, and of them those from its own column on.
    const int behind = (int)max(0LL, min(col + V - cols, (long long)V));
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const long long row = min(group * 64 + row0 + p * ROWS, rows - 1);
      const u4 w = rt_mx::load_once(src + row * cols + min(col, cols - V));
      __builtin_memcpy(raw[p], &w, 16);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      u4 w;
      __builtin_memcpy(&w, raw[p], 16);
      w = from_element<T>(w, group * 64 + row0 + p * ROWS < rows ? behind : V);
      __builtin_memcpy(raw[p], &w, 16);
    }
    finish(std::false_type());
  } else {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const long long row = group * 64 + row0 + p * ROWS;
#pragma unroll
      for (int i = 0; i < V; ++i)
        raw[p][i] = row < rows && col + i < cols ? src[row * cols + col + i] : Elem<T>::put(0.0f);
    }
    finish(std::false_type());
  }
  __syncthreads();
  store_scales(sc, scales, step, groups, group);
}

// The same of the transpose: src [cols, rows], dst rows of src's columns.  A
// lane takes four bytes of a row of src, one or two (W) rows of dst, a wave 32
// rows of src and 64 W of their values, so a block's maximum needs no exchange.
template <typename T, bool FP4>
__global__ __launch_bounds__(256) void quantize_t_kernel(const T* __restrict__ src, long long rows, long long cols,
                                                         unsigned char* __restrict__ codes,
                                                         unsigned char* __restrict__ scales, long long steps,
                                                         long long groups, long long block0) {
  constexpr int W = 4 / sizeof(T);
  typedef unsigned int any_u1 __attribute__((aligned(2)));
  __shared__ unsigned sc[64 * W];
  const long long block = block0 + blockIdx.x, blocks = (groups + W - 1) / W;
  const long long group = block % blocks * W, step = block / blocks;
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const long long row = group * 64 + W * lane, col = step * 128 + 32 * g;
  if (threadIdx.x < 64 * W) sc[threadIdx.x] = 0;
  __syncthreads();
  if (row < rows) {
    // Every load is made, from inside src: a branch around each would make them
    // wait for one another (1003 x 1500 f16 12.3 us that way, 4.3 this way).
    const bool whole = row + W <= rows;  // else the last of an odd number
    const T* at = src + (whole || rows < W ? row : row - 1);
    T raw[32][W];
    if (W == 2 && rows < W) {  // uniform: one row of dst
#pragma unroll
      for (int i = 0; i < 32; ++i) raw[i][0] = src[min(col + i, cols - 1)];
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const unsigned w =
            __builtin_nontemporal_load(reinterpret_cast<const any_u1*>(at + min(col + i, cols - 1) * rows));
        const unsigned v = whole ? w : w >> 16;
        __builtin_memcpy(raw[i], &v, 4);
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) raw[i][j] = col + i < cols ? raw[i][j] : Elem<T>::put(0.0f);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (j > 0 && !whole) break;
      float v[32];
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[i] = Elem<T>::get(raw[i][j]);
        m = max(m, magnitude<FP4>(v[i]));
      }
      const unsigned byte = FP4 && m >= 0x7f800000u ? 255u : scale_byte<FP4>(m);
      const float scale = rt_mx::scale_of(min(byte, 254u));
      unsigned w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = encode4<FP4>(v + 4 * i, scale);
      if constexpr (FP4) {
        u4* out = reinterpret_cast<u4*>(codes + (row + j) * (steps * 64) + step * 64 + 16 * g);
        *out = u4{w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16)};
      } else {
        u4* out = reinterpret_cast<u4*>(codes + (row + j) * (steps * 128) + step * 128 + 32 * g);
        out[0] = u4{w[0], w[1], w[2], w[3]};
        out[1] = u4{w[4], w[5], w[6], w[7]};
      }
      const int q = W * lane + j, r = q % 64;
      reinterpret_cast<unsigned char*>(sc)[256 * (q / 64) + 4 * (16 * g + r % 16) + r / 16] = (unsigned char)byte;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (group + i < groups) store_scales(sc + 64 * i, scales, step, groups, group + i);
}

// Four codes (a half or a whole word) as values, without their scale.
template <bool FP4>
__device__ inline void decode4(unsigned w, float (&v)[4]) {
  f2 lo, hi;
  if constexpr (FP4) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  } else {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true);
  }
  v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
}

// Back to values, with the lanes of quantize_kernel: 16 bytes of values each, so
// that a store instruction writes whole rows of the step.
template <typename T, bool FP4>
__global__ __launch_bounds__(256) void dequantize_kernel(const unsigned char* __restrict__ codes,
                                                         const unsigned char* __restrict__ scales, T* __restrict__ dst,
                                                         long long rows, long long cols, long long steps,
                                                         long long groups, long long block0) {
  constexpr int V = 16 / sizeof(T), LANES = 128 / V, ROWS = 256 / LANES, PASSES = 64 / ROWS;
  __shared__ unsigned sc[64];
  const long long block = block0 + blockIdx.x, step = block % steps, group = block / steps;
  const int lane = threadIdx.x % LANES, row0 = threadIdx.x / LANES;
  const long long col = step * 128 + lane * V, row_bytes = steps * (FP4 ? 64 : 128);
  if (threadIdx.x < 64)
    sc[threadIdx.x] = reinterpret_cast<const unsigned*>(scales)[(step * groups + group) * 64 + threadIdx.x];
  unsigned w[PASSES][V / 4];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const long long row = min(group * 64 + row0 + p * ROWS, rows - 1);
    const unsigned char* at = codes + row * row_bytes + col / (FP4 ? 2 : 1);
    if constexpr (FP4 && V == 4) w[p][0] = *reinterpret_cast<const unsigned short*>(at);
    else if constexpr (FP4) w[p][0] = *reinterpret_cast<const unsigned*>(at);
    else __builtin_memcpy(w[p], __builtin_assume_aligned(at, V), V);
    if constexpr (FP4 && V == 8) w[p][1] = w[p][0] >> 16;
  }
  __syncthreads();
  if (col >= cols) return;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = row0 + p * ROWS;
    const long long row = group * 64 + r;
    if (row >= rows) break;
    const unsigned byte = (sc[16 * (lane * V / 32) + r % 16] >> (8 * (r / 16))) & 0xffu;
    const float scale = rt_mx::scale_of(byte);
    T out[V];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      float v[4];
      decode4<FP4>(w[p][i], v);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * i + e] = Elem<T>::put(v[e] * scale);
    }
    T* at = dst + row * cols + col;
    if (col + V <= cols) {
      u4 o;
      __builtin_memcpy(&o, out, 16);
      rt_mx::store_once(at, o);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col + i < cols) at[i] = out[i];
    }
  }
}

// v zeroed where the mask is not positive (VJP false), or v = g · 1[mask > 0]
// as a product (VJP true).  A thread takes four values of a row, read, masked and
// written whole where the row has room.
template <bool VJP>
__global__ __launch_bounds__(256) void mask_kernel(const unsigned char* __restrict__ codes, unsigned rows,
                                                   unsigned cols, long long row_bytes, const float* g, float* v) {
  const unsigned chunks = (cols + 3) / 4;
  for (unsigned row = blockIdx.y * blockDim.y + threadIdx.y; row < rows; row += gridDim.y * blockDim.y)
    for (unsigned c = blockIdx.x * blockDim.x + threadIdx.x; c < chunks; c += gridDim.x * blockDim.x) {
      const unsigned col = 4 * c, w = *reinterpret_cast<const unsigned*>(codes + row * row_bytes + col);
      float* at = v + (long long)row * cols + col;
      const float* from = VJP ? g + (long long)row * cols + col : at;
      const int n = min(4u, cols - col);
      float x[4];
      if (n == 4) {
        __builtin_memcpy(x, from, sizeof x);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = e < n ? from[e] : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool on = rt_dev::mx_positive((w >> (8 * e)) & 0xffu);
        if constexpr (VJP) x[e] = x[e] * (on ? 1.0f : 0.0f);
        else x[e] = on ? x[e] : 0.0f;
      }
      if (n == 4) {
        __builtin_memcpy(at, x, sizeof x);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < n) at[e] = x[e];
      }
    }
}

template <bool VJP>
hipError_t mask(hipStream_t s, const rt::MxTensor& m, const float* g, float* v) {
  if (m.rows == 0 || m.cols == 0) return hipSuccess;
  const unsigned chunks = (unsigned)((m.cols + 3) / 4);
  // A block: 256 threads over a row, or over several short ones.
  unsigned bx = 256;
  while (bx > 16 && bx / 2 >= chunks) bx /= 2;
  const unsigned by = 256 / bx, gx = std::min((chunks + bx - 1) / bx, 4096u);
  const unsigned gy = (unsigned)std::min<long long>((m.rows + by - 1) / by, std::max(1u, 32768u / gx));
  rt::launch(mask_kernel<VJP>, dim3(gx, gy), dim3(bx, by), 0, s, m.codes, (unsigned)m.rows, (unsigned)m.cols,
             (long long)rt::mx_layout(m.dtype, m.rows, m.cols).row_bytes, g, v);
  return hipGetLastError();
}

// A grid holds fewer than 2^32 threads: more blocks go in several launches.
template <typename F>
void in_launches(long long blocks, F&& launch) {
  constexpr long long kMost = 1LL << 23;
  for (long long b = 0; b < blocks; b += kMost) launch(b, (unsigned)std::min(kMost, blocks - b));
}

template <typename T>
hipError_t quantize(hipStream_t s, const void* src, bool transposed, const rt::MxTensor& d) {
  const rt::MxLayout l = rt::mx_layout(d.dtype, d.rows, d.cols);
  auto* codes = const_cast<unsigned char*>(d.codes);
  auto* scales = const_cast<unsigned char*>(d.scales);
  const size_t per = transposed ? 4 / sizeof(T) : 1;  // groups a block
  auto go = [&](auto kernel) {
    in_launches((long long)(l.steps * ((l.groups + per - 1) / per)), [&](long long block0, unsigned n) {
      rt::launch(kernel, dim3(n), dim3(256), 0, s, static_cast<const T*>(src), d.rows, d.cols, codes, scales,
                 (long long)l.steps, (long long)l.groups, block0);
    });
  };
  if (d.dtype == RT_MXFP4) transposed ? go(quantize_t_kernel<T, true>) : go(quantize_kernel<T, true>);
  else transposed ? go(quantize_t_kernel<T, false>) : go(quantize_kernel<T, false>);
  return hipGetLastError();
}

template <typename T>
hipError_t dequantize(hipStream_t s, const rt::MxTensor& m, void* dst) {
  const rt::MxLayout l = rt::mx_layout(m.dtype, m.rows, m.cols);
  auto go = [&](auto kernel) {
    in_launches((long long)(l.steps * l.groups), [&](long long block0, unsigned n) {
      rt::launch(kernel, dim3(n), dim3(256), 0, s, m.codes, m.scales, static_cast<T*>(dst), m.rows, m.cols,
                 (long long)l.steps, (long long)l.groups, block0);
    });
  };
  m.dtype == RT_MXFP4 ? go(dequantize_kernel<T, true>) : go(dequantize_kernel<T, false>);
  return hipGetLastError();
}

}  // namespace

namespace rt {

MxTensor mx_tensor(const rt_buf* b) {
  MxTensor m;
  m.dtype = b->dtype;
  m.rows = (long long)b->shape[0];
  m.cols = (long long)b->shape[1];
  m.codes = static_cast<const unsigned char*>(b->ptr);
  m.scales = m.codes + mx_layout(b->dtype, b->shape[0], b->shape[1]).scale_off;
  return m;
}

hipError_t mx_quantize_launch(hipStream_t s, const void* src, int src_dtype, bool transposed, const MxTensor& dst) {
  if (dst.rows == 0 || dst.cols == 0) return hipSuccess;
  switch (src_dtype) {
    case RT_F32: return quantize<float>(s, src, transposed, dst);
    case RT_BF16: return quantize<bf16_bits>(s, src, transposed, dst);
    case RT_F16: return quantize<_Float16>(s, src, transposed, dst);
  }
  return hipErrorInvalidValue;
}

hipError_t mx_dequantize_launch(hipStream_t s, const MxTensor& src, void* dst, int dst_dtype) {
  if (src.rows == 0 || src.cols == 0) return hipSuccess;
  switch (dst_dtype) {
    case RT_F32: return dequantize<float>(s, src, dst);
    case RT_BF16: return dequantize<bf16_bits>(s, src, dst);
    case RT_F16: return dequantize<_Float16>(s, src, dst);
  }
  return hipErrorInvalidValue;
}

hipError_t mx_mask_launch(hipStream_t s, const MxTensor& m, float* v) { return mask<false>(s, m, nullptr, v); }

hipError_t mx_relu_vjp_launch(hipStream_t s, const MxTensor& m, const float* g, float* dx) {
  return mask<true>(s, m, g, dx);
}

}  // namespace rt

// ------------------------------------------------------------------ C ABI
using namespace rt;

extern "C" int rt_convert_t(rt_ctx* c, const rt_buf* src, rt_buf* dst) {
  CHECK_CTX(c);
  if (!src || !dst) return fail(c, RT_ERR_INVALID, "null buffer");
  if (src->dtype == RT_U32 || is_mx(src->dtype) || !is_mx(dst->dtype))
    return fail(c, RT_ERR_DTYPE, "convert_t takes f32, bf16 or f16 into a microscaled tensor");
  if (src->rank != 2 || src->shape[0] != dst->shape[1] || src->shape[1] != dst->shape[0])
    return fail(c, RT_ERR_SHAPE, "convert_t: the source must be [%zu,%zu]", dst->shape[1], dst->shape[0]);
  Launch L(c, "convert_t");
  HIP_TRY(c, mx_quantize_launch(c->stream, src->ptr, src->dtype, true, mx_tensor(dst)), "convert_t");
  return RT_OK;
}

// The weight gradient from an 8-bit saved input: dW = Xᵀ·δ with X RT_MXFP8
// [rows, K] and δ f32, bf16 or f16 [rows, N], on v_mfma_f32_16x16x32_bf16.
//
// A value of X has four significant bits and a power of two, so it is a bf16
// without rounding; δ is one bf16 plane as it stands, two for f16 (11 bits) or
// three for f32 (24 bits, each plane the next eight by truncation).  So every
// product is exact, and the sums are those of a bf16 GEMM in f32.  The scale
// of X varies along the rows that are summed, so it cannot stay outside the
// product: X is decoded on its way into LDS, where a thread holds 16 columns
// of one row, which share a scale.
//
// Tiles.  Both operands are contiguous along the output (rows are summed):
// LDS holds them as [row][columns + 16] and fragments come out by transposed
// reads (ds_read_b64_tr_b16).  Two LDS stages; the loads of stage k + 1 are in
// flight under the MFMAs of stage k, then decoded or split into the other
// stage.  Few output tiles over many rows are cut into slices of rows, whose
// f32 planes splitk_reduce adds in slice order.

#include <algorithm>
#include <type_traits>

#include "device_util.h"
#include "mx_device.h"
#include "rt_internal.h"

namespace {

using rt_dev::static_for;
using rt_mx::u2;
using rt_mx::u4;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Args {
  const unsigned char* x;  // codes
  const unsigned char* x_scales;
  const void* delta;
  float* c;
  long long rows;  // summed
  int K, N;        // of C
  int x_row;       // bytes of a row of codes
  int x_groups;
  long long rows_per_split, split_stride;
  int tiles_m, tiles_n;
};

__device__ inline u2 lds_tr(const unsigned short* p) {
  s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
  return __builtin_bit_cast(u2, r);
}

// The upper halves of two words, lo first.
__device__ inline unsigned pack_hi(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// 16 codes with one scale as 16 bf16 (exact).
__device__ inline void decode16(const u4& w, float scale, u4 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i / 2][2 * (i % 2)] =
        __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, false));
    out[i / 2][2 * (i % 2) + 1] =
        __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, true));
  }
}

// Eight consecutive values of δ and their planes.
template <int DT>
struct Delta;
template <>
struct Delta<RT_BF16> {
  static constexpr int PLANES = 1, ROWS = 64;
  using T = unsigned short;
  struct Raw {
    u4 v;
  };
  __device__ static inline void planes(const Raw& x, u4 (&out)[1]) { out[0] = x.v; }
};
// v in planes of truncated bf16.  An infinity is its first plane alone.
template <int P>
__device__ inline void split8(const float (&v)[8], u4 (&out)[P]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
  for (int p = 0; p < P; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[p][i] = pack_hi(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rest = x[i] - __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u);
      x[i] = p == 0 && fabsf(x[i]) == INFINITY ? 0.0f : rest;
    }
  }
}
template <>
struct Delta<RT_F16> {
  static constexpr int PLANES = 2, ROWS = 32;
  using T = _Float16;
  struct Raw {
    u4 v;
  };
  __device__ static inline void planes(const Raw& x, u4 (&out)[2]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)__builtin_bit_cast(_Float16, (unsigned short)(x.v[i / 2] >> (16 * (i % 2))));
    split8<2>(v, out);
  }
};
template <>
struct Delta<RT_F32> {
  static constexpr int PLANES = 3, ROWS = 32;
  using T = float;
  struct Raw {
    f4 v[2];
  };
  __device__ static inline void planes(const Raw& x, u4 (&out)[3]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x.v[i / 4][i % 4];
    split8<3>(v, out);
  }
};

template <int DT, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN) void mx_dw_kernel(Args p) {
  using D = Delta<DT>;
  using T = typename D::T;
  constexpr int THREADS = 64 * WGM * WGN, ROWS = D::ROWS, P = D::PLANES;
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int SA = BM + 16, SB = BN + 16;  // halves per LDS row
  constexpr int STAGE = ROWS * (SA + P * SB);
  constexpr int XC = ROWS * BM / 16 / THREADS, DC = ROWS * BN / 8 / THREADS;  // chunks a thread
  static_assert(XC * THREADS * 16 == ROWS * BM && DC * THREADS * 8 == ROWS * BN, "chunks split evenly");
  static_assert(2 * STAGE * 2 <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) unsigned short smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;

  // Each XCD takes a contiguous run of (slice, tile) items, the tiles of a
  // slice in bands of 8 tile rows.
  const int nb = p.tiles_m * p.tiles_n, total = gridDim.x;
  int lin = blockIdx.x;
  if ((total & 7) == 0) lin = (lin & 7) * (total >> 3) + (lin >> 3);
  const int slice = lin / nb, bid = lin - slice * nb;
  constexpr int BAND = 8;
  const int band = bid / (BAND * p.tiles_n), first_m = band * BAND;
  const int size = min(p.tiles_m - first_m, BAND), in_band = bid - band * BAND * p.tiles_n;
  const int m0 = (first_m + in_band % size) * BM, n0 = (in_band / size) * BN;
  const long long rb = slice * p.rows_per_split, re = min(p.rows, rb + p.rows_per_split);
  const int stages = (int)((re - rb + ROWS - 1) / ROWS);  // at least one, by the host's plan

  u4 xr[XC];
  unsigned char xs[XC];
  typename D::Raw dr[DC];
  const T* delta = static_cast<const T*>(p.delta);
  auto load = [&](int s) {
    const long long base = rb + (long long)s * ROWS;
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int idx = tid + THREADS * i, col = m0 + 16 * (idx % (BM / 16));
      const long long row = base + idx / (BM / 16);
      xr[i] = u4{0u, 0u, 0u, 0u};
      xs[i] = 0;
      if (row < re && col < p.x_row) {
        xr[i] = *reinterpret_cast<const u4*>(p.x + row * p.x_row + col);
        xs[i] = p.x_scales[((long long)(col / 128) * p.x_groups + row / 64) * 256 + 4 * (16 * (col % 128 / 32) + row % 16) +
                           row % 64 / 16];
      }
    }
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      const int idx = tid + THREADS * i, col = n0 + 8 * (idx % (BN / 8));
      const long long row = base + idx / (BN / 8);
      const T* at = delta + row * p.N + col;
      if (row < re && col + 8 <= p.N) {
        __builtin_memcpy(&dr[i], at, 8 * sizeof(T));
      } else {
        T h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = row < re && col + e < p.N ? at[e] : T(0);
        __builtin_memcpy(&dr[i], h, sizeof h);
      }
    }
  };
  auto store = [&](int buf) {
    unsigned short* a = smem + buf * STAGE;
    unsigned short* b = a + ROWS * SA;
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int idx = tid + THREADS * i;
      u4 h[2];
      decode16(xr[i], rt_mx::scale_of(xs[i]), h);
      u4* at = reinterpret_cast<u4*>(a + (idx / (BM / 16)) * SA + 16 * (idx % (BM / 16)));
      at[0] = h[0];
      at[1] = h[1];
    }
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      const int idx = tid + THREADS * i;
      u4 h[P];
      D::planes(dr[i], h);
#pragma unroll
      for (int q = 0; q < P; ++q)
        *reinterpret_cast<u4*>(b + q * ROWS * SB + (idx / (BN / 8)) * SB + 8 * (idx % (BN / 8))) = h[q];
    }
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int u = 0; u < TN; ++u) acc[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  // Lane (g, r) of 16 columns at c: k = 8 g .. 8 g + 7 of the 32 rows from k0.
  auto frag = [&](const unsigned short* lds, int stride, int k0, int c) {
    const unsigned short* at = lds + (k0 + 8 * g + (r >> 2)) * stride + c + 4 * (r & 3);
    const u2 lo = lds_tr(at), hi = lds_tr(at + 4 * stride);
    return u4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto compute = [&](int buf) {
    const unsigned short* a = smem + buf * STAGE;
    const unsigned short* b = a + ROWS * SA;
#pragma unroll
    for (int kk = 0; kk < ROWS; kk += 32) {
      u4 fa[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) fa[t] = frag(a, SA, kk, wm + 16 * t);
      // The small planes first: their sums keep more of their bits.
#pragma unroll
      for (int q = P - 1; q >= 0; --q) {
        u4 fb[TN];
#pragma unroll
        for (int u = 0; u < TN; ++u) fb[u] = frag(b + q * ROWS * SB, SB, kk, wn + 16 * u);
#pragma unroll
        for (int t = 0; t < TM; ++t)
#pragma unroll
          for (int u = 0; u < TN; ++u)
            acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[u]),
                                                                __builtin_bit_cast(bf16x8, fa[t]), acc[t][u], 0, 0, 0);
      }
    }
  };

  load(0);
  store(0);
  __syncthreads();
  for (int s = 0; s < stages; ++s) {
    if (s + 1 < stages) load(s + 1);
    compute(s & 1);
    if (s + 1 < stages) store((s + 1) & 1);
    __syncthreads();
  }

  float* c = p.c + slice * p.split_stride;
  const bool vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(c) & 15) == 0;
  static_for<0, TM>([&](auto tc) {
    constexpr int t = decltype(tc)::value;
    const int row = m0 + wm + 16 * t + r;
    if (row >= p.K) return;
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      const int col = n0 + wn + 16 * u + 4 * g;
      if (col >= p.N) continue;
      float* at = c + (long long)row * p.N + col;
      if (vec) {
        *reinterpret_cast<f4*>(at) = acc[t][u];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.N) at[e] = acc[t][u][e];
      }
    }
  });
}

constexpr int kTile = 128;

struct Plan {
  long long tiles, rows_per_split;
  int splits;
};

// Slices of rows where the tiles of C alone do not give each CU two blocks:
// about 512 blocks, and at least 256 rows a slice.
Plan plan(long long rows, long long K, long long N) {
  Plan q;
  q.tiles = ((K + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
  const long long want = std::max<long long>(1, std::min(512 / std::max<long long>(q.tiles, 1), rows / 256));
  q.rows_per_split = ((rows + want - 1) / want + 63) / 64 * 64;
  q.splits = (int)((rows + q.rows_per_split - 1) / q.rows_per_split);
  return q;
}

template <int DT>
hipError_t launch(hipStream_t s, const Args& p, const Plan& q) {
  rt::launch(mx_dw_kernel<DT, kTile, kTile, 2, 2>, dim3((unsigned)(q.tiles * q.splits)), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

namespace rt {

size_t mx_dw_scratch_elems(const MxTensor& x, int, long long N) {
  if (x.rows == 0) return 0;
  const Plan q = plan(x.rows, x.cols, N);
  return q.splits > 1 ? (size_t)q.splits * x.cols * N : 0;
}

hipError_t mx_dw_launch(hipStream_t s, const MxTensor& x, const void* delta, int delta_dtype, long long N, float* C,
                        float* scratch) {
  if (x.rows == 0) return fill_i32_launch(s, reinterpret_cast<int*>(C), 0, (size_t)x.cols * N);
  const MxLayout l = mx_layout(x.dtype, x.rows, x.cols);
  const Plan q = plan(x.rows, x.cols, N);
  Args p{};
  p.x = x.codes;
  p.x_scales = x.scales;
  p.delta = delta;
  p.c = q.splits > 1 ? scratch : C;
  p.rows = x.rows;
  p.K = (int)x.cols;
  p.N = (int)N;
  p.x_row = (int)l.row_bytes;
  p.x_groups = (int)l.groups;
  p.rows_per_split = q.rows_per_split;
  p.split_stride = (long long)x.cols * N;
  p.tiles_m = (p.K + kTile - 1) / kTile;
  p.tiles_n = (p.N + kTile - 1) / kTile;
  hipError_t e = delta_dtype == RT_BF16  ? launch<RT_BF16>(s, p, q)
                 : delta_dtype == RT_F16 ? launch<RT_F16>(s, p, q)
                                         : launch<RT_F32>(s, p, q);
  if (e != hipSuccess || q.splits == 1) return e;
  return splitk_reduce_launch(s, scratch, q.splits, p.split_stride, p.K, p.N, C, RT_F32, p.N, RT_EPI_NONE, nullptr,
                              nullptr, RT_F32, nullptr, nullptr);
}

}  // namespace rt

// The weight gradient from an 8-bit saved input: dW = Xᵀ·δ with X RT_MXFP8
// [rows, K] and δ f32, bf16 or f16 [rows, N], on v_mfma_f32_16x16x32_bf16 and
// _f16; and the bias gradient, δ's column sums, from the same tiles.
//
// A value of X has four significant bits and a power of two, so it is a bf16
// without rounding, and an f16 too where its block's scale is from 2^-15 to 2^7.
// bf16 δ is multiplied as it stands; f16 δ as well where the block's part of X
// has only such scales (a block looks its scales over first: 1/32 of its codes'
// bytes), else as two bf16 planes (11 bits); f32 δ as three (24 bits, each plane
// the next eight by truncation).  So every product is exact, and the sums are
// f32.  The scale of X varies along the rows that are summed, so it cannot stay
// outside the product: X is decoded on its way into LDS, where a thread holds 16
// columns of one row, which share a scale.
//
// Tiles.  Both operands are contiguous along the output (rows are summed):
// LDS holds them by rows and fragments come out by transposed reads
// (ds_read_b64_tr_b16).  Few output tiles over many rows are cut into slices of
// rows, whose f32 planes splitk_reduce adds in slice order.

#include <algorithm>
#include <type_traits>

#include "device_util.h"
#include "mx_device.h"
#include "rt_internal.h"

namespace {

using rt_dev::barrier_lds;
using rt_dev::static_for;
using rt_dev::wait_vm;
using rt_mx::u2;
using rt_mx::u4;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Args {
  const unsigned char* x;  // codes
  const unsigned char* x_scales;
  const void* delta;
  float* c;
  float* shares;   // column sums of δ, [slices, tiles_m, N]: of a slice's 64-row pieces tile row t adds those with
                   // index % tiles_m == t (blocks of both bodies share a slice); or null
  long long rows;  // summed
  int K, N;        // of C
  int x_row;       // bytes of a row of codes
  int x_groups;
  long long rows_per_split, split_stride;  // a slice starts on a 64-row group
  int tiles_m, tiles_n;
};

// The (slice, tile) of a block.  Each XCD takes a contiguous run of them, the
// tiles of a slice in bands of 8 tile rows.
struct Place {
  int slice, tile_m, m0, n0;
  long long rb, re;  // its rows of X and δ
};
template <int BM, int BN>
__device__ inline Place place(const Args& p) {
  const int nb = p.tiles_m * p.tiles_n, total = gridDim.x;
  int lin = blockIdx.x;
  if ((total & 7) == 0) lin = (lin & 7) * (total >> 3) + (lin >> 3);
  Place q;
  q.slice = lin / nb;
  const int bid = lin - q.slice * nb;
  constexpr int BAND = 8;
  const int band = bid / (BAND * p.tiles_n), first_m = band * BAND;
  const int size = min(p.tiles_m - first_m, BAND), in_band = bid - band * BAND * p.tiles_n;
  q.tile_m = first_m + in_band % size;
  q.m0 = q.tile_m * BM;
  q.n0 = (in_band / size) * BN;
  q.rb = q.slice * p.rows_per_split;
  q.re = min(p.rows, q.rb + p.rows_per_split);
  return q;
}

__device__ inline u2 lds_tr(const unsigned short* p) {
  s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
  return __builtin_bit_cast(u2, r);
}

// 16 consecutive codes of one row of X and their scale byte.
struct XChunk {
  u4 w;
  unsigned char byte;
  __device__ inline void load(const Args& p, long long row, long long re, int col) {
    w = u4{0u, 0u, 0u, 0u};
    byte = 0;
    if (row < re && col < p.x_row) {
      w = *reinterpret_cast<const u4*>(p.x + row * p.x_row + col);
      byte = p.x_scales[((long long)(col / 128) * p.x_groups + row / 64) * 256 + 4 * (16 * (col % 128 / 32) + row % 16) +
                        row % 64 / 16];
    }
  }
};

// 16 codes as 16 bf16 or f16.
template <bool F16>
__device__ inline void decode16(const u4& w, unsigned byte, u4 (&out)[2]) {
  const float scale = rt_mx::scale_of(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned v;
    if constexpr (F16) {
      v = i % 2 ? __builtin_bit_cast(unsigned, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i / 2], scale, true))
                : __builtin_bit_cast(unsigned, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i / 2], scale, false));
    } else {
      v = i % 2 ? __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i / 2], scale, true))
                : __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i / 2], scale, false));
    }
    out[i / 4][i % 4] = v;
  }
}

// A descriptor of `bytes` bytes from base on: none where that is not positive (a
// stage past the last one), for a negative size would be taken as a huge one.
__device__ inline __amdgpu_buffer_rsrc_t bounded_rsrc(const void* base, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0,
                                           (int)max(0LL, min(bytes, 0x7ffffff0LL)), 0x00020000);
}

// C's tile (or its plane of the slice): lane (g, r) holds four consecutive
// columns of a row.
template <int TM, int TN>
__device__ __forceinline__ void store_c(const Args& p, const f4 (&acc)[TM][TN], const Place& at, int wm, int wn, int g,
                                        int r) {
  float* c = p.c + at.slice * p.split_stride;
  const bool vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(c) & 15) == 0;
  static_for<0, TM>([&](auto tc) {
    constexpr int t = decltype(tc)::value;
    const int row = at.m0 + wm + 16 * t + r;
    if (row >= p.K) return;
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      const int col = at.n0 + wn + 16 * u + 4 * g;
      if (col >= p.N) continue;
      float* o = c + (long long)row * p.N + col;
      if (vec) {
        *reinterpret_cast<f4*>(o) = acc[t][u];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.N) o[e] = acc[t][u][e];
      }
    }
  });
}

// Each thread's sums of 8 columns (chunk tid % CH), over the threads that share
// them, in a fixed order.  smem: THREADS * 8 floats that nothing else uses.
template <int THREADS, int CH>
__device__ __forceinline__ void store_shares(const Args& p, const float (&cs)[8], float* red, const Place& at, int tid) {
#pragma unroll
  for (int e = 0; e < 8; ++e) red[(tid / CH) * CH * 8 + 8 * (tid % CH) + e] = cs[e];
  __syncthreads();
  float* out = p.shares + ((long long)at.slice * p.tiles_m + at.tile_m) * p.N;
  for (int col = tid; col < CH * 8 && at.n0 + col < p.N; col += THREADS) {
    float v = 0.0f;
    for (int j = 0; j < THREADS / CH; ++j) v += red[j * CH * 8 + col];
    out[at.n0 + col] = v;
  }
}

// ---------------------------------------------------------------- δ in bf16 planes
// The upper halves of two words, lo first.
__device__ inline unsigned pack_hi(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// v in planes of truncated bf16.  An infinity is its first plane alone.
template <int P>
__device__ inline void split8(const float (&v)[8], u4 (&out)[P]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
  for (int q = 0; q < P; ++q) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[q][i] = pack_hi(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rest = x[i] - __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u);
      x[i] = q == 0 && fabsf(x[i]) == INFINITY ? 0.0f : rest;
    }
  }
}

// Eight consecutive values of δ: planes P, and rows of a stage (two bf16 k-steps
// of 32 where there is one plane, so that a stage has the same work).
template <int DT>
struct Delta;
template <>
struct Delta<RT_BF16> {
  static constexpr int PLANES = 1, ROWS = 64;
  using T = unsigned short;
  static __device__ inline float get(T v) { return __uint_as_float((unsigned)v << 16); }
};
template <>
struct Delta<RT_F16> {
  static constexpr int PLANES = 2, ROWS = 32;
  using T = _Float16;
  static __device__ inline float get(T v) { return (float)v; }
};
template <>
struct Delta<RT_F32> {
  static constexpr int PLANES = 3, ROWS = 32;
  using T = float;
  static __device__ inline float get(T v) { return v; }
};

// LDS of the planes' two stages: [row][BM + 16] of X, then [row][BN + 16] of
// each plane, in halves.
template <int DT, int BM, int BN>
constexpr int planes_lds() {
  return 2 * Delta<DT>::ROWS * (BM + 16 + Delta<DT>::PLANES * (BN + 16));
}

// Any δ, any alignment: both operands through registers, where X is decoded and
// δ split, into the LDS stage that the MFMAs of the other one do not read.
template <int DT, int BM, int BN, int WGM, int WGN>
__device__ __forceinline__ void planes_body(const Args& p, const Place& at, unsigned short* smem) {
  using D = Delta<DT>;
  using T = typename D::T;
  constexpr int THREADS = 64 * WGM * WGN, ROWS = D::ROWS, P = D::PLANES;
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int SA = BM + 16, SB = BN + 16, STAGE = ROWS * (SA + P * SB);
  constexpr int XC = ROWS * BM / 16 / THREADS, DC = ROWS * BN / 8 / THREADS;  // chunks a thread
  constexpr int CH = BN / 8;
  static_assert(XC * THREADS * 16 == ROWS * BM && DC * THREADS * 8 == ROWS * BN, "chunks split evenly");
  static_assert(THREADS % CH == 0, "a thread's chunks of δ are all of the same columns");
  static_assert(THREADS * 8 * 4 <= 2 * STAGE * 2, "column sums fit in LDS");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;
  const int stages = (int)((at.re - at.rb + ROWS - 1) / ROWS);  // at least one, by the host's plan

  XChunk x[XC];
  T d[DC][8];
  const T* delta = static_cast<const T*>(p.delta);
  const int dcol = at.n0 + 8 * (tid % CH);
  auto load = [&](int s) {
    const long long base = at.rb + (long long)s * ROWS;
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int idx = tid + THREADS * i;
      x[i].load(p, base + idx / (BM / 16), at.re, at.m0 + 16 * (idx % (BM / 16)));
    }
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      const long long row = base + (tid + THREADS * i) / CH;
      const T* src = delta + row * p.N + dcol;
      if (row < at.re && dcol + 8 <= p.N) {
        __builtin_memcpy(d[i], src, sizeof d[i]);  // whatever the alignment
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[i][e] = row < at.re && dcol + e < p.N ? src[e] : T(0);
      }
    }
  };
  const bool do_cs = p.shares != nullptr;
  float cs[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  auto store = [&](int s) {
    unsigned short* a = smem + (s & 1) * STAGE;
    unsigned short* b = a + ROWS * SA;
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int idx = tid + THREADS * i;
      u4 h[2];
      decode16<false>(x[i].w, x[i].byte, h);
      u4* to = reinterpret_cast<u4*>(a + (idx / (BM / 16)) * SA + 16 * (idx % (BM / 16)));
      to[0] = h[0];
      to[1] = h[1];
    }
    const bool add = do_cs && s * ROWS / 64 % p.tiles_m == at.tile_m;
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = D::get(d[i][e]);
      if (add) {
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] += v[e];
      }
      u4 h[P];
      split8<P>(v, h);
#pragma unroll
      for (int q = 0; q < P; ++q)
        *reinterpret_cast<u4*>(b + q * ROWS * SB + ((tid + THREADS * i) / CH) * SB + 8 * (tid % CH)) = h[q];
    }
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int u = 0; u < TN; ++u) acc[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  // Lane (g, r) of 16 columns at c: k = 8 g .. 8 g + 7 of the 32 rows from k0.
  auto frag = [&](const unsigned short* lds, int stride, int k0, int c) {
    const unsigned short* q = lds + (k0 + 8 * g + (r >> 2)) * stride + c + 4 * (r & 3);
    const u2 lo = lds_tr(q), hi = lds_tr(q + 4 * stride);
    return u4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto compute = [&](int s) {
    const unsigned short* a = smem + (s & 1) * STAGE;
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
    compute(s);
    if (s + 1 < stages) store(s + 1);
    __syncthreads();
  }
  if (do_cs) store_shares<THREADS, CH>(p, cs, reinterpret_cast<float*>(smem), at, tid);
  store_c<TM, TN>(p, acc, at, wm, wn, g, r);
}

template <int DT, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN) void mx_dw_planes_kernel(Args p) {
  __shared__ __attribute__((aligned(16))) unsigned short smem[planes_lds<DT, BM, BN>()];
  planes_body<DT, BM, BN, WGM, WGN>(p, place<BM, BN>(p), smem);
}

// ---------------------------------------------------------------- δ as it stands
// bf16 or f16 δ whose rows are whole 16-byte chunks goes straight into LDS; X
// through registers.  LDS rows are unpadded: 32-byte granule G of row k is at
// G ^ hm(k), which gives the eight rows of a transposed read distinct banks.
// Two stages of 64 rows (two MFMA k-steps).  With the first k-step's fragments
// of stage k in registers:
//   the first k-step's MFMAs, under them the reads of the second's fragments;
//   wait for all loads, barrier; start δ's loads of stage k + 2 into stage k's
//   buffer, decode X of stage k + 2 into it (loaded a stage ago), load X of
//   stage k + 3;
//   the second k-step's MFMAs, under them the reads of stage k + 1's first.
template <bool F16, int BM, int BN, int WGM, int WGN>
__device__ __forceinline__ void direct_body(const Args& p, const Place& at, unsigned short* smem) {
  constexpr int WAVES = WGM * WGN, THREADS = 64 * WAVES, ROWS = 64;
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int STAGE = ROWS * (BM + BN);
  constexpr int XC = ROWS * BM / 16 / THREADS;          // chunks of X a thread
  constexpr int LOADS = ROWS * BN * 2 / 1024 / WAVES;   // δ's loads a wave
  constexpr int RPL = 512 / BN;                         // rows a load
  constexpr int CH = BN / 8, KG = THREADS / CH;
  static_assert(XC * THREADS * 16 == ROWS * BM && LOADS * WAVES * 1024 == ROWS * BN * 2, "loads split evenly");
  static_assert(BM % 128 == 0 && BN % 128 == 0 && (RPL * WAVES) % 16 == 0, "swizzle period");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;
  const int stages = (int)((at.re - at.rb + ROWS - 1) / ROWS);
  auto hm = [](int k) { return (k & 3) | ((k >> 3) & 1) << 2; };

  // δ: this lane's chunk of its first load; later ones are RPL * WAVES rows on.
  const int k0 = RPL * wave + lane / CH, slot = lane % CH;
  const int voff = 2 * (k0 * p.N + 16 * ((slot >> 1) ^ hm(k0)) + 8 * (slot & 1)), vstep = 2 * RPL * WAVES * p.N;
  const unsigned smem_at = rt_dev::lds_offset(smem);
  auto issue = [&](int s) {
    const long long row = at.rb + (long long)s * ROWS;
    const unsigned short* src = static_cast<const unsigned short*>(p.delta) + row * p.N + at.n0;
    // The slice's rows end here: what follows arrives as zeros.
    const __amdgpu_buffer_rsrc_t rsrc = bounded_rsrc(src, 2 * ((at.re - row) * p.N - at.n0));
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      rt_dev::dma16_at(rsrc, smem_at + 2 * ((s & 1) * STAGE + ROWS * BM) + 1024 * (i * WAVES + wave), voff + i * vstep);
  };
  // X: a thread's chunks are 32 rows apart (of the 64 of a group), in the same
  // columns, so one dword holds all their scales.  Rows past the slice's end are
  // zeros; columns past X's last come from elsewhere, in rows of C that are not
  // stored.
  constexpr int XR = BM / 16;  // chunks a row
  static_assert(THREADS / XR == 32 && XC == 2, "chunks of X");
  const int xk = tid / XR, xvoff = xk * p.x_row + 16 * (tid % XR);
  const int svoff = (tid % XR) / 8 * (p.x_groups * 256) + 4 * (16 * (tid % 8 / 2) + xk % 16);
  u4 xw[XC];
  unsigned xs;
  auto load_x = [&](int s) {
    const long long row = at.rb + (long long)s * ROWS, group = row / 64;
    const long long first = (long long)(at.m0 / 128) * p.x_groups + group, all = (long long)(p.x_row / 128) * p.x_groups;
    const __amdgpu_buffer_rsrc_t rsrc = bounded_rsrc(p.x + row * p.x_row + at.m0, (at.re - row) * p.x_row - at.m0);
    const __amdgpu_buffer_rsrc_t srsrc = bounded_rsrc(p.x_scales + first * 256, (all - first) * 256);
#pragma unroll
    for (int i = 0; i < XC; ++i) xw[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, xvoff + i * 32 * p.x_row, 0, 0);
    xs = __builtin_amdgcn_raw_buffer_load_b32(srsrc, svoff, 0, 0);
  };
  auto store_x = [&](int s) {
    unsigned short* a = smem + (s & 1) * STAGE + xk * BM + 16 * ((tid % XR) ^ hm(xk));
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      u4 h[2];
      // Absent rows have no scale either (their byte may be any).
      const bool in = at.rb + (long long)s * ROWS + xk + 32 * i < at.re;
      decode16<F16>(xw[i], in ? (xs >> (8 * (xk / 16 + 2 * i))) & 0xffu : 0u, h);
      u4* to = reinterpret_cast<u4*>(a + 32 * i * BM);
      to[0] = h[0];
      to[1] = h[1];
    }
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int u = 0; u < TN; ++u) acc[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  const int kl = 8 * g + (r >> 2);  // hm(kl + 4) == hm(kl)
  auto read_a = [&](int s, int kk, int t) {
    const unsigned short* q = smem + (s & 1) * STAGE + (32 * kk + kl) * BM + 4 * (r & 3) + 16 * ((wm / 16 + t) ^ hm(kl));
    const u2 lo = lds_tr(q), hi = lds_tr(q + 4 * BM);
    return u4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto read_b = [&](int s, int kk, u4 (&fb)[TN]) {
    const unsigned short* b = smem + (s & 1) * STAGE + ROWS * BM + (32 * kk + kl) * BN + 4 * (r & 3);
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      const unsigned short* q = b + 16 * ((wn / 16 + u) ^ hm(kl));
      const u2 lo = lds_tr(q), hi = lds_tr(q + 4 * BN);
      fb[u] = u4{lo[0], lo[1], hi[0], hi[1]};
    }
  };
  // The MFMAs of one k-step (fa, cur), and the reads of the next one's fragments:
  // B's into a second set, a fragment of A over the one that was just used (two
  // sets of both do not fit beside 128 accumulators).
  u4 fa[TM], fb0[TN], fb1[TN];
  auto k_step = [&](const u4 (&cur)[TN], u4 (&next)[TN], int s, int kk) {
    read_b(s, kk, next);
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int u = 0; u < TN; ++u) {
        if constexpr (F16)
          acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, cur[u]),
                                                             __builtin_bit_cast(f16x8, fa[t]), acc[t][u], 0, 0, 0);
        else
          acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, cur[u]),
                                                              __builtin_bit_cast(bf16x8, fa[t]), acc[t][u], 0, 0, 0);
      }
      fa[t] = read_a(s, kk, t);
    }
    // Kept in this order: the scheduler would move the reads up, into new registers.
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * TN, 0);
    static_for<0, TM>([&](auto) {
      __builtin_amdgcn_sched_group_barrier(0x008, TN, 0);  // MFMAs
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // LDS reads
    });
  };
  const bool do_cs = p.shares != nullptr;
  float cs[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  auto colsum = [&](int s) {
    const unsigned short* b = smem + (s & 1) * STAGE + ROWS * BM;
    const int c = tid % CH;
#pragma unroll
    for (int k = tid / CH; k < ROWS; k += KG) {
      const u4 v = *reinterpret_cast<const u4*>(b + k * BN + 16 * ((c >> 1) ^ hm(k)) + 8 * (c & 1));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned short h = (unsigned short)(v[e / 2] >> (16 * (e % 2)));
        if constexpr (F16) cs[e] += (float)__builtin_bit_cast(_Float16, h);
        else cs[e] += __uint_as_float((unsigned)h << 16);
      }
    }
  };

  // Past the last stage rows are zeros: loaded, decoded, never multiplied.
  issue(0);
  load_x(0);
  wait_vm<0>();
  store_x(0);
  issue(1);
  load_x(1);
  wait_vm<0>();
  store_x(1);
  load_x(2);
  barrier_lds();
  read_b(0, 0, fb0);
#pragma unroll
  for (int t = 0; t < TM; ++t) fa[t] = read_a(0, 0, t);
  for (int s = 0; s < stages; ++s) {
    k_step(fb0, fb1, s, 1);
    if (do_cs && s % p.tiles_m == at.tile_m) colsum(s);
    wait_vm<0>();
    barrier_lds();
    if (s + 2 < stages) issue(s + 2);
    store_x(s + 2);
    load_x(s + 3);
    k_step(fb1, fb0, s + 1, 0);
  }
  __syncthreads();
  if (do_cs) store_shares<THREADS, CH>(p, cs, reinterpret_cast<float*>(smem), at, tid);
  store_c<TM, TN>(p, acc, at, wm, wn, g, r);
}

template <bool F16, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN) void mx_dw_kernel(Args p) {
  constexpr int LDS = 2 * 64 * (BM + BN), OTHER = F16 ? planes_lds<RT_F16, BM, BN>() : 0;
  __shared__ __attribute__((aligned(16))) unsigned short smem[LDS > OTHER ? LDS : OTHER];
  const Place at = place<BM, BN>(p);
  if constexpr (F16) {
    // Scales that f16 holds: 448·2^7 and 2^-9·2^-15 are f16 values.  A byte of 0
    // is a block of zeros (or of values below 2^-118, which count as zeros).
    int bad = 0;
    const long long g0 = at.rb / 64, n = (at.re + 63) / 64 - g0;
    for (int step = at.m0 / 128; step < min(at.m0 + BM, p.x_row) / 128; ++step) {
      const unsigned* sc = reinterpret_cast<const unsigned*>(p.x_scales) + ((long long)step * p.x_groups + g0) * 64;
      for (long long i = threadIdx.x; i < n * 64; i += 64 * WGM * WGN) {
        const unsigned w = sc[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned b = (w >> (8 * e)) & 0xffu;
          bad |= b != 0 && (b < 112 || b > 134);
        }
      }
    }
    if (__syncthreads_or(bad)) return planes_body<RT_F16, BM, BN, WGM, WGN>(p, at, smem);
  }
  direct_body<F16, BM, BN, WGM, WGN>(p, at, smem);
}

struct Plan {
  bool direct;  // δ straight into LDS
  int tile;     // 256 or 128, square
  long long tiles_m, tiles_n, rows_per_split;
  int splits;
};

// Slices of rows where the tiles of C alone do not fill the chip: up to 256
// blocks of 256 x 256 (one a CU), 512 of 128 x 128 (two).
Plan plan(const rt::MxTensor& x, const void* delta, int dtype, long long N) {
  Plan q;
  q.direct = dtype != RT_F32 && N % 8 == 0 && (reinterpret_cast<uintptr_t>(delta) & 15) == 0 && N <= (1LL << 23) &&
             x.cols <= (1LL << 23) && x.rows <= (1LL << 28);  // offsets of a stage below 2^31 bytes
  auto tiles = [&](int t) { return ((x.cols + t - 1) / t) * ((N + t - 1) / t); };
  auto splits = [&](int t, long long blocks, long long rows) {
    return std::max<long long>(1, std::min(blocks / std::max<long long>(tiles(t), 1), x.rows / rows));
  };
  q.tile = q.direct && tiles(256) * splits(256, 256, 1024) >= 192 ? 256 : 128;
  const long long want = q.tile == 256 ? splits(256, 256, 1024) : splits(128, 512, 256);
  q.tiles_m = (x.cols + q.tile - 1) / q.tile;
  q.tiles_n = (N + q.tile - 1) / q.tile;
  q.rows_per_split = ((x.rows + want - 1) / want + 63) / 64 * 64;
  q.splits = (int)((x.rows + q.rows_per_split - 1) / q.rows_per_split);
  return q;
}

size_t plane_elems(const Plan& q, long long K, long long N) { return q.splits > 1 ? (size_t)q.splits * K * N : 0; }
size_t share_elems(const Plan& q, long long N) {
  return q.splits * q.tiles_m > 1 ? (size_t)q.splits * q.tiles_m * N : 0;
}

}  // namespace

namespace rt {

size_t mx_dw_scratch_elems(const MxTensor& x, const void* delta, int delta_dtype, long long N, bool colsum) {
  if (x.rows == 0 || x.cols == 0) return 0;
  const Plan q = plan(x, delta, delta_dtype, N);
  size_t n = plane_elems(q, x.cols, N);
  if (colsum) n += share_elems(q, N) + (q.splits == 1 ? colsum_scratch_elems((int)q.tiles_m, (int)N, RT_F32) : 0);
  return n;
}

hipError_t mx_dw_launch(hipStream_t s, const MxTensor& x, const void* delta, int delta_dtype, long long N, float* C,
                        float* colsum, float* scratch, size_t scratch_elems) {
  const MxLayout l = mx_layout(x.dtype, x.rows, x.cols);
  const Plan q = plan(x, delta, delta_dtype, N);
  const size_t planes = plane_elems(q, x.cols, N), shares = share_elems(q, N);
  Args p{};
  p.x = x.codes;
  p.x_scales = x.scales;
  p.delta = delta;
  p.c = q.splits > 1 ? scratch : C;
  p.shares = !colsum ? nullptr : shares ? scratch + planes : colsum;
  p.rows = x.rows;
  p.K = (int)x.cols;
  p.N = (int)N;
  p.x_row = (int)l.row_bytes;
  p.x_groups = (int)l.groups;
  p.rows_per_split = q.rows_per_split;
  p.split_stride = (long long)x.cols * N;
  p.tiles_m = (int)q.tiles_m;
  p.tiles_n = (int)q.tiles_n;
  const dim3 grid((unsigned)(q.tiles_m * q.tiles_n * q.splits));
  if (q.direct && q.tile == 256) {
    if (delta_dtype == RT_F16) rt::launch(mx_dw_kernel<true, 256, 256, 2, 4>, grid, dim3(512), 0, s, p);
    else rt::launch(mx_dw_kernel<false, 256, 256, 2, 4>, grid, dim3(512), 0, s, p);
  } else if (q.direct) {
    if (delta_dtype == RT_F16) rt::launch(mx_dw_kernel<true, 128, 128, 2, 2>, grid, dim3(256), 0, s, p);
    else rt::launch(mx_dw_kernel<false, 128, 128, 2, 2>, grid, dim3(256), 0, s, p);
  } else if (delta_dtype == RT_F32) {
    rt::launch(mx_dw_planes_kernel<RT_F32, 128, 128, 2, 2>, grid, dim3(256), 0, s, p);
  } else if (delta_dtype == RT_F16) {
    rt::launch(mx_dw_planes_kernel<RT_F16, 128, 128, 2, 2>, grid, dim3(256), 0, s, p);
  } else {
    rt::launch(mx_dw_planes_kernel<RT_BF16, 128, 128, 2, 2>, grid, dim3(256), 0, s, p);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (q.splits > 1)
    return splitk_reduce_launch(s, scratch, q.splits, p.split_stride, p.K, p.N, C, RT_F32, p.N, RT_EPI_NONE, nullptr,
                                nullptr, RT_F32, p.shares, colsum, colsum ? p.tiles_m : 0);
  if (colsum && shares)
    return colsum_launch(s, p.shares, RT_F32, p.tiles_m, p.N, colsum, scratch + planes + shares,
                         scratch_elems - planes - shares);
  return hipSuccess;
}

}  // namespace rt

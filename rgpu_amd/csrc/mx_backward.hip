// The weight gradient from an 8-bit saved input: dW = Xᵀ·δ with X RT_MXFP8
// [rows, K] and δ f32, bf16 or f16 [rows, N], on v_mfma_f32_16x16x32_bf16 and
// _f16; and the bias gradient, δ's column sums, from the same tiles.
//
// A value of X has four significant bits and a power of two, so it is a bf16
// without rounding (from 2^-133 on: the last bits of blocks whose scale is 2^-125
// or less are lost), and an f16 too where its block's scale is from 2^-15 to 2^7.
// bf16 δ is multiplied as it stands; f16 δ as well where the scales of the
// workgroup's part of X span no more than those 22 powers of two: X is multiplied
// by a power of two that brings them there, C by its inverse (a workgroup looks
// its scales over first: 1/32 of its codes' bytes).  Else f16 δ goes in as two
// bf16 planes (11 bits; 262144 rows of 512 x 512 521 us, 160 as it stands); f32 δ
// as three (24 bits, each plane the next eight by truncation).  So every product
// is exact, and the sums are f32.  The scale of X varies along the rows that are
// summed, so it cannot stay outside the product: X is decoded on its way into LDS,
// where a thread holds 16 columns of one row, which share a scale.
//
// Tiles.  Both operands are contiguous along the output (rows are summed):
// LDS holds them by rows and fragments come out by transposed reads
// (ds_read_b64_tr_b16).  Few output tiles over many rows are cut into slices of
// rows, whose f32 planes splitk_reduce adds in slice order.
//
// Measured: 8192 rows, 4096 x 4096, bf16 with the bias gradient 246-274 us (1.0 to
// 1.12 PFLOP/s; a library product of 8192^3 1.21); 262144 rows of 512 x 512 158-175
// (2.3-2.6 TB/s); 2048 rows, 1024 x 1024, f32 33 with the sum of its slices.

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
  float* shares;   // column sums of δ, [slices, sharers, N]: of a slice's 64-row pieces tile row t < sharers adds those
                   // with index % sharers == t (blocks of both bodies share a slice); or null
  int sharers;
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
  int shift;         // X is multiplied by 2^shift, C by 2^-shift (f16)
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
  q.shift = 0;
  return q;
}

__device__ inline u2 lds_tr(const unsigned short* p) {
  s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
  return __builtin_bit_cast(u2, r);
}

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

// What is left of an operand from the next stage on.
struct Cursor {
  const char* base;
  long long left, step;  // bytes to the slice's end, bytes a stage
  __device__ inline __amdgpu_buffer_rsrc_t next() {
    const __amdgpu_buffer_rsrc_t r = bounded_rsrc(base, left);
    base += step;
    left -= step;
    return r;
  }
};

// X by stages: a thread's chunks of 16 codes are 32 rows apart, in the same
// columns; the dword that holds the scale of one holds those of all (of the
// 64-row group).  Rows past the slice's end are zeros; columns past X's last come
// from elsewhere, in rows of C that are not stored.
template <int ROWS, int BM, int THREADS>
struct XSide {
  static constexpr int XR = BM / 16, CHUNKS = ROWS * XR / THREADS;
  static_assert(THREADS / XR == 32 && CHUNKS * 32 == ROWS, "chunks 32 rows apart");
  struct Raw {
    u4 w[CHUNKS];
    unsigned scales;
  };
  Cursor codes, scales;
  int k, voff, svoff, vstep, rows;  // row and place of the first chunk; rows of the slice
  int shift;
  __device__ inline void init(const Args& p, const Place& at, int tid) {
    const int c = at.m0 % 128 / 16 + tid % XR;  // chunk of its 128 columns, and beyond
    k = tid / XR;
    voff = k * p.x_row + 16 * (tid % XR);
    vstep = 32 * p.x_row;
    svoff = c / 8 * (p.x_groups * 256) + 4 * (16 * (c % 8 / 2) + k % 16);
    rows = (int)(at.re - at.rb);
    shift = at.shift;
    codes = Cursor{reinterpret_cast<const char*>(p.x + at.rb * p.x_row + at.m0), (long long)rows * p.x_row - at.m0,
                   (long long)ROWS * p.x_row};
    const long long first = (long long)(at.m0 / 128) * p.x_groups + at.rb / 64;
    scales = Cursor{reinterpret_cast<const char*>(p.x_scales + first * 256),
                    ((long long)(p.x_row / 128) * p.x_groups - first) * 256, 256};
  }
  // The next stage; s: its number.
  __device__ inline void load(int s, Raw& x) {
    const __amdgpu_buffer_rsrc_t rsrc = codes.next();
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) x.w[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, voff + i * vstep, 0, 0);
    const __amdgpu_buffer_rsrc_t srsrc = bounded_rsrc(scales.base, scales.left);
    x.scales = __builtin_amdgcn_raw_buffer_load_b32(srsrc, svoff, 0, 0);
    if (ROWS == 64 || (s & 1)) scales.next();  // a group is 64 rows
  }
  // Chunk i as 16 halves.  Absent rows have no scale either (their byte may be any).
  template <bool F16>
  __device__ inline void decode(int s, const Raw& x, int i, u4 (&h)[2]) const {
    const int row = s * ROWS + k + 32 * i;
    unsigned byte = (x.scales >> (8 * (row % 64 / 16))) & 0xffu;
    if constexpr (F16) byte = (unsigned)max((int)byte + shift, 0);
    decode16<F16>(x.w[i], row < rows ? byte : 0u, h);
  }
};

// acc += of 32 rows; the operands swapped (D = δᵀ·X), so that lane (g, r) ends
// with row r and four consecutive columns.
template <bool F16>
__device__ inline f4 mfma(const u4& a, const u4& b, const f4& acc) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0,
                                                   0);
}

// C's tile (or its plane of the slice): lane (g, r) holds four consecutive
// columns of a row.
template <int TM, int TN>
__device__ __forceinline__ void store_c(const Args& p, f4 (&acc)[TM][TN], const Place& at, int wm, int wn, int g,
                                        int r) {
  float* c = p.c + at.slice * p.split_stride;
  const bool vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(c) & 15) == 0;
  if (at.shift != 0) {
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int u = 0; u < TN; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][u][e] = ldexpf(acc[t][u][e], -at.shift);
  }
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

// Whose turn a 64-row piece's column sums are: tile row t's, pieces t, t +
// sharers, ...
struct Turn {
  int left, sharers;  // pieces until the next one of this tile row
  __device__ inline bool take(bool done) {  // done: the piece ends here
    const bool mine = left == 0;
    if (done) left = mine ? sharers - 1 : left - 1;
    return mine;
  }
};

// Each thread's sums of 8 columns (chunk tid % CH), over the threads that share
// them, in a fixed order.  smem: THREADS * 8 floats that nothing else uses.
template <int THREADS, int CH>
__device__ __forceinline__ void store_shares(const Args& p, const float (&cs)[8], float* red, const Place& at, int tid) {
#pragma unroll
  for (int e = 0; e < 8; ++e) red[(tid / CH) * CH * 8 + 8 * (tid % CH) + e] = cs[e];
  __syncthreads();
  float* out = p.shares + ((long long)at.slice * p.sharers + at.tile_m) * p.N;
  for (int col = tid; col < CH * 8 && at.n0 + col < p.N; col += THREADS) {
    float v = 0.0f;
    for (int j = 0; j < THREADS / CH; ++j) v += red[j * CH * 8 + col];
    out[at.n0 + col] = v;
  }
}

// ---------------------------------------------------------------- through registers
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

// What δ is and how it is multiplied: its planes, the rows of a stage (two MFMA
// k-steps of 32 where there is one plane, one else), and a chunk of eight values.
// Halves come as five dwords from the one that holds the first value on, shifted
// to it, so that rows may start on any of them.
enum Kind { kBf16, kF16, kF16Planes, kF32 };
template <int KIND>
struct Delta {
  static constexpr bool F16 = KIND == kF16;
  static constexpr int PLANES = KIND == kF16Planes ? 2 : 1, ROWS = PLANES == 1 ? 64 : 32, SIZE = 2;
  struct Raw {
    u4 w;
    unsigned last;
  };
  static __device__ inline Raw load(__amdgpu_buffer_rsrc_t rsrc, unsigned at) {
    const int a = (int)(at & ~3u);
    return Raw{__builtin_amdgcn_raw_buffer_load_b128(rsrc, a, 0, 0),
               (unsigned)__builtin_amdgcn_raw_buffer_load_b32(rsrc, a + 16, 0, 0)};
  }
  static __device__ inline u4 halves(const Raw& x, unsigned at) {
    const unsigned sh = 8 * (at & 3u);
    u4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbit(i < 3 ? x.w[i + 1] : x.last, x.w[i], sh);
    return v;
  }
  static __device__ inline void values(const Raw& x, unsigned at, float (&v)[8]) {
    const u4 h = halves(x, at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned short b = (unsigned short)(h[e / 2] >> (16 * (e % 2)));
      if constexpr (KIND == kBf16) v[e] = __uint_as_float((unsigned)b << 16);
      else v[e] = (float)__builtin_bit_cast(_Float16, b);
    }
  }
  static __device__ inline void planes(const Raw& x, unsigned at, u4 (&out)[PLANES]) {
    if constexpr (PLANES == 1) {
      out[0] = halves(x, at);
    } else {
      float v[8];
      values(x, at, v);
      split8<PLANES>(v, out);
    }
  }
};
template <>
struct Delta<kF32> {
  static constexpr bool F16 = false;
  static constexpr int PLANES = 3, ROWS = 32, SIZE = 4;
  struct Raw {
    u4 w[2];
  };
  static __device__ inline Raw load(__amdgpu_buffer_rsrc_t rsrc, unsigned at) {
    return Raw{{__builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at, 0, 0),
                __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at + 16, 0, 0)}};
  }
  static __device__ inline void values(const Raw& x, unsigned, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(x.w[e / 4][e % 4]);
  }
  static __device__ inline void planes(const Raw& x, unsigned at, u4 (&out)[3]) {
    float v[8];
    values(x, at, v);
    split8<3>(v, out);
  }
};

// LDS of two stages: [row][BM + 16] of X, then [row][BN + 16] of each plane, in halves.
template <int KIND, int BM, int BN>
constexpr int staged_lds() {
  return 2 * Delta<KIND>::ROWS * (BM + 16 + Delta<KIND>::PLANES * (BN + 16));
}

// Any δ, any alignment: both operands through registers, where X is decoded and
// δ split, into the LDS stage that the MFMAs of the other one do not read.  Loads
// go out two stages ahead of that, three ahead of their MFMAs.
template <int KIND, int BM, int BN, int WGM, int WGN>
__device__ __forceinline__ void staged_body(const Args& p, const Place& at, unsigned short* smem) {
  using D = Delta<KIND>;
  constexpr int THREADS = 64 * WGM * WGN, ROWS = D::ROWS, P = D::PLANES;
  constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int SA = BM + 16, SB = BN + 16, STAGE = ROWS * (SA + P * SB);
  constexpr int CH = BN / 8, KR = THREADS / CH, DC = ROWS / KR;  // chunks a row of δ, rows between a thread's, chunks
  using X = XSide<ROWS, BM, THREADS>;
  static_assert(THREADS % CH == 0 && DC * KR == ROWS, "a thread's chunks of δ are all of the same columns");
  static_assert(THREADS * 8 * 4 <= 2 * STAGE * 2, "column sums fit in LDS");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;
  const int stages = (int)((at.re - at.rb + ROWS - 1) / ROWS);  // at least one, by the host's plan

  X xs;
  xs.init(p, at, tid);
  // δ is addressed from the dword that holds the slice's first value (every
  // stage's then starts at the same place of its dword) to the one that holds its
  // last; columns past N are the next row's.  Half of the last dword may be a
  // value of an absent row, whose chunks are therefore sent past the end.
  const uintptr_t from = reinterpret_cast<uintptr_t>(p.delta) + (unsigned long long)D::SIZE * (at.rb * p.N + at.n0);
  const unsigned odd = (unsigned)(from & 3);
  const unsigned dvoff = odd + (unsigned)D::SIZE * ((unsigned)(tid / CH) * p.N + 8 * (tid % CH));
  const unsigned dstep = D::SIZE * KR * p.N;
  Cursor dc{reinterpret_cast<const char*>(from - odd),
            (D::SIZE * ((at.re - at.rb) * p.N - at.n0) + (long long)odd + 3) & ~3LL, (long long)D::SIZE * ROWS * p.N};
  struct Raw {
    typename X::Raw x;
    typename D::Raw d[DC];
  };
  auto load = [&](int s, Raw& raw) {
    xs.load(s, raw.x);
    const __amdgpu_buffer_rsrc_t rsrc = dc.next();
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      const bool in = D::SIZE == 4 || s * ROWS + tid / CH + KR * i < xs.rows;
      raw.d[i] = D::load(rsrc, in ? dvoff + i * dstep : 0x7fffff00u);
    }
  };
  const bool do_cs = p.shares != nullptr && at.tile_m < p.sharers;
  float cs[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  Turn turn{at.tile_m, p.sharers};
  auto store = [&](int s, const Raw& raw) {
    unsigned short* a = smem + (s & 1) * STAGE;
    unsigned short* b = a + ROWS * SA;
#pragma unroll
    for (int i = 0; i < X::CHUNKS; ++i) {
      u4 h[2];
      xs.template decode<D::F16>(s, raw.x, i, h);
      u4* to = reinterpret_cast<u4*>(a + (xs.k + 32 * i) * SA + 16 * (tid % X::XR));
      to[0] = h[0];
      to[1] = h[1];
    }
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      u4 h[P];
      D::planes(raw.d[i], dvoff + i * dstep, h);
#pragma unroll
      for (int q = 0; q < P; ++q)
        *reinterpret_cast<u4*>(b + q * ROWS * SB + (tid / CH + KR * i) * SB + 8 * (tid % CH)) = h[q];
    }
    const bool mine = turn.take(ROWS == 64 || (s & 1));
    if (do_cs && mine) {
#pragma unroll
      for (int i = 0; i < DC; ++i) {
        float v[8];
        D::values(raw.d[i], dvoff + i * dstep, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] += v[e];
      }
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
          for (int u = 0; u < TN; ++u) acc[t][u] = mfma<D::F16>(fa[t], fb[u], acc[t][u]);
      }
    }
  };

  // Two stages a turn, without a branch between them: after one, the compiler
  // would wait for all loads, not for those it needs.  Past the last stage rows
  // are zeros (their loads have empty descriptors).
  Raw r0, r1;
  load(0, r0);
  load(1, r1);
  store(0, r0);
  load(2, r0);
  __syncthreads();
  auto stage = [&](int s, Raw& next) {
    compute(s);
    store(s + 1, next);
    load(s + 3, next);
    __syncthreads();
  };
  for (int s = 0; s + 1 < stages; s += 2) {
    stage(s, r1);
    stage(s + 1, r0);
  }
  if (stages & 1) compute(stages - 1);
  __syncthreads();
  if (do_cs) store_shares<THREADS, CH>(p, cs, reinterpret_cast<float*>(smem), at, tid);
  store_c<TM, TN>(p, acc, at, wm, wn, g, r);
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
  constexpr int LOADS = ROWS * BN * 2 / 1024 / WAVES;   // δ's loads a wave
  constexpr int RPL = 512 / BN;                         // rows a load
  constexpr int CH = BN / 8, KG = THREADS / CH;
  static_assert(LOADS * WAVES * 1024 == ROWS * BN * 2 && THREADS % CH == 0 && KG * (ROWS / KG) == ROWS, "even split");
  using X = XSide<ROWS, BM, THREADS>;
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
  // The slice's rows end where its bytes do: what follows arrives as zeros.
  Cursor dc{reinterpret_cast<const char*>(static_cast<const unsigned short*>(p.delta) + at.rb * p.N + at.n0),
            2 * ((at.re - at.rb) * p.N - at.n0), 2LL * ROWS * p.N};
  auto issue = [&](int s) {
    const __amdgpu_buffer_rsrc_t rsrc = dc.next();
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      rt_dev::dma16_at(rsrc, smem_at + 2 * ((s & 1) * STAGE + ROWS * BM) + 1024 * (i * WAVES + wave), voff + i * vstep);
  };
  X xs;
  xs.init(p, at, tid);
  typename X::Raw xr;
  auto load_x = [&](int s) { xs.load(s, xr); };
  auto store_x = [&](int s) {
    unsigned short* a = smem + (s & 1) * STAGE + xs.k * BM + 16 * ((tid % X::XR) ^ hm(xs.k));
#pragma unroll
    for (int i = 0; i < X::CHUNKS; ++i) {
      u4 h[2];
      xs.template decode<F16>(s, xr, i, h);
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
      for (int u = 0; u < TN; ++u) acc[t][u] = mfma<F16>(fa[t], cur[u], acc[t][u]);
      fa[t] = read_a(s, kk, t);
    }
    // Kept in this order: the scheduler would move the reads up, into new registers.
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * TN, 0);
    static_for<0, TM>([&](auto) {
      __builtin_amdgcn_sched_group_barrier(0x008, TN, 0);  // MFMAs
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // LDS reads
    });
  };
  const bool do_cs = p.shares != nullptr && at.tile_m < p.sharers;
  float cs[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  Turn turn{at.tile_m, p.sharers};
  auto colsum = [&](int s) {
    const unsigned short* b = smem + (s & 1) * STAGE + ROWS * BM;
    const int c = tid % CH;
#pragma unroll
    for (int i = 0; i < ROWS / KG; ++i) {
      const int k = tid / CH + KG * i;
      const u4 v = *reinterpret_cast<const u4*>(b + k * BN + 16 * ((c >> 1) ^ hm(k)) + 8 * (c & 1));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned short h = (unsigned short)(v[e / 2] >> (16 * (e % 2)));
        if constexpr (F16) cs[e] += (float)__builtin_bit_cast(_Float16, h);
        else cs[e] += __uint_as_float((unsigned)h << 16);
      }
    }
  };

  // Past the last stage rows are zeros: decoded, never multiplied.
  issue(0);
  load_x(0);
  wait_vm<0>();
  store_x(0);
  if (stages > 1) {
    issue(1);
    load_x(1);
    wait_vm<0>();
    store_x(1);
    load_x(2);
  }
  barrier_lds();
  read_b(0, 0, fb0);
#pragma unroll
  for (int t = 0; t < TM; ++t) fa[t] = read_a(0, 0, t);
  for (int s = 0; s < stages; ++s) {
    k_step(fb0, fb1, s, 1);
    const bool mine = turn.take(true);
    if (do_cs && mine) colsum(s);
    wait_vm<0>();
    barrier_lds();
    if (s + 2 < stages) {
      issue(s + 2);
      store_x(s + 2);
      load_x(s + 3);
    }
    k_step(fb1, fb0, s + 1, 0);
  }
  __syncthreads();
  if (do_cs) store_shares<THREADS, CH>(p, cs, reinterpret_cast<float*>(smem), at, tid);
  store_c<TM, TN>(p, acc, at, wm, wn, g, r);
}

// The shift at which f16 holds the values of the workgroup's part of X: one that
// puts its scales between 2^-15 and 2^7 (448·2^7 and 2^-9·2^-15 are f16 values), 0
// where they are; or kNoShift.  A byte of 0 is a block of zeros (or of values up to
// 2^-118, which are zeros where the shift does not bring them up); 255, NaN, is
// left to bf16.  smem: 8 ints.
constexpr int kNoShift = 1 << 20;
template <int BM, int THREADS>
__device__ inline int f16_shift(const Args& p, const Place& at, int* smem) {
  int high = 0, low = 0;  // the largest byte, and 255 - the least that is not 0
  const long long g0 = at.rb / 64, n = (at.re + 63) / 64 - g0;
  for (int step = at.m0 / 128; 128 * step < min(at.m0 + BM, p.x_row); ++step) {
    const unsigned* sc = reinterpret_cast<const unsigned*>(p.x_scales) + ((long long)step * p.x_groups + g0) * 64;
    for (long long i = threadIdx.x; i < n * 64; i += THREADS) {
      const unsigned w = sc[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int b = (int)((w >> (8 * e)) & 0xffu);
        high = max(high, b);
        low = max(low, b != 0 ? 255 - b : 0);
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    high = max(high, __shfl_xor(high, d));
    low = max(low, __shfl_xor(low, d));
  }
  if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = high << 8 | low;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    high = max(high, smem[w] >> 8);
    low = max(low, smem[w] & 0xff);
  }
  __syncthreads();  // the stages overwrite smem
  high = __builtin_amdgcn_readfirstlane(high);
  low = 255 - __builtin_amdgcn_readfirstlane(low);
  if (high == 255 || high - low > 22) return kNoShift;
  return high == 0 || (low >= 112 && high <= 134) ? 0 : 134 - high;
}

constexpr int larger(int a, int b) { return a > b ? a : b; }

// 128 x 128 with four waves, 64 x 64 with two.
template <int KIND, int TILE>
__global__ __launch_bounds__(2 * TILE, 2) void mx_dw_staged_kernel(Args p) {
  constexpr int OTHER = KIND == kF16 ? kF16Planes : KIND, WGN = TILE / 64;
  __shared__ __attribute__((aligned(16))) unsigned short smem[larger(staged_lds<KIND, TILE, TILE>(), staged_lds<OTHER, TILE, TILE>())];
  Place at = place<TILE, TILE>(p);
  if constexpr (KIND == kF16) {
    const int shift = f16_shift<TILE, 2 * TILE>(p, at, reinterpret_cast<int*>(smem));
    if (shift == kNoShift) return staged_body<kF16Planes, TILE, TILE, 2, WGN>(p, at, smem);
    at.shift = shift;
  }
  staged_body<KIND, TILE, TILE, 2, WGN>(p, at, smem);
}

template <bool F16>
__global__ __launch_bounds__(512) void mx_dw_direct_kernel(Args p) {
  __shared__ __attribute__((aligned(16))) unsigned short smem[larger(2 * 64 * 512, staged_lds<kF16Planes, 256, 256>())];
  Place at = place<256, 256>(p);
  if constexpr (F16) {
    const int shift = f16_shift<256, 512>(p, at, reinterpret_cast<int*>(smem));
    if (shift == kNoShift) return staged_body<kF16Planes, 256, 256, 2, 4>(p, at, smem);
    at.shift = shift;
  }
  direct_body<F16, 256, 256, 2, 4>(p, at, smem);
}

struct Plan {
  int tile;  // 256 (δ straight into LDS), 128 or 64 (through registers), square
  long long tiles_m, tiles_n, rows_per_split;
  int splits, sharers;
};

// The tile and the slices of rows, by what they are expected to take.  A block
// alone on its CU takes `alone` a stage (latencies), several share the CU's
// throughput (`each`); slices write and read a plane of C each (4 TB/s, counted
// once each way, and a launch).  Measured, us: 2048 rows, 1024 x 1024, bf16: 64
// tiles unsplit 32.6, 3 slices 23.9, 8 30; 128 tiles 4 slices 25.8, unsplit 41.8;
// f32: 64 tiles 4 slices 33.2, unsplit 62.3.  600 rows, 2000 x 1500, bf16: 64
// tiles 17.9 unsplit, 29 in 2 slices.  5000 rows, 200 x 64, bf16: 64 tiles 69
// unsplit, 9.9 in 32 slices.  8192 rows, 4096 x 4096, bf16: 256 with 256 tiles,
// 399 with 128.
Plan plan(const rt::MxTensor& x, const void* delta, int dtype, long long N) {
  struct Tile {
    int size;
    float alone, each;  // us a stage of a block
  };
  static constexpr Tile kTiles[3] = {{64, 0.9f, 0.35f}, {128, 1.2f, 0.85f}, {256, 1.8f, 1.8f}};
  // 256 tiles take rows of δ by whole 16-byte chunks (and a step's scales below
  // 2^31 bytes).
  const bool direct = dtype != RT_F32 && N % 8 == 0 && (reinterpret_cast<uintptr_t>(delta) & 15) == 0 &&
                      x.rows <= (1LL << 28);
  const int stage_rows = dtype == RT_F32 ? 32 : 64;
  const float plane_us = 4.0f * (float)x.cols * (float)N / 4e6f;
  Plan best{};
  float best_us = 0;
  for (int t = 0; t < (direct ? 3 : 2); ++t) {
    const Tile& tile = kTiles[t];
    const long long tm = (x.cols + tile.size - 1) / tile.size, tn = (N + tile.size - 1) / tile.size;
    for (long long want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128}) {
      if (want > 1 && want * 64 > x.rows) break;
      const long long per = ((x.rows + want - 1) / want + 63) / 64 * 64, splits = (x.rows + per - 1) / per;
      const long long on_cu = (tm * tn * splits + 255) / 256;
      const float us = (float)((per + stage_rows - 1) / stage_rows) * std::max(tile.alone, (float)on_cu * tile.each) +
                       (splits > 1 ? 2.0f + 2.0f * (float)splits * plane_us : plane_us);
      if (best_us == 0 || us < best_us) {
        best_us = us;
        best = Plan{tile.size, tm, tn, per, (int)splits, 0};
      }
    }
  }
  // The bias gradient: over a long slice the tile rows share its pieces, over a
  // short one the first adds them all, which saves the launch that adds shares
  // (37 rows, 1024 x 1000, bf16: 7.2 us and 2.2 for that launch; 4.4 without).
  best.sharers = best.rows_per_split > 1024 ? (int)best.tiles_m : 1;
  return best;
}

template <int KIND>
void launch_staged(hipStream_t s, const Args& p, const Plan& q, dim3 grid) {
  if (q.tile == 128) rt::launch(mx_dw_staged_kernel<KIND, 128>, grid, dim3(256), 0, s, p);
  else rt::launch(mx_dw_staged_kernel<KIND, 64>, grid, dim3(128), 0, s, p);
}

size_t plane_elems(const Plan& q, long long K, long long N) { return q.splits > 1 ? (size_t)q.splits * K * N : 0; }
size_t share_elems(const Plan& q, long long N) {
  return q.splits * q.sharers > 1 ? (size_t)q.splits * q.sharers * N : 0;
}

}  // namespace

namespace rt {

size_t mx_dw_scratch_elems(const MxTensor& x, const void* delta, int delta_dtype, long long N, bool colsum) {
  if (x.rows == 0 || x.cols == 0) return 0;
  const Plan q = plan(x, delta, delta_dtype, N);
  size_t n = plane_elems(q, x.cols, N);
  if (colsum) n += share_elems(q, N) + (q.splits == 1 ? colsum_scratch_elems(q.sharers, (int)N, RT_F32) : 0);
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
  p.sharers = q.sharers;
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
  if (q.tile == 256)
    delta_dtype == RT_F16 ? rt::launch(mx_dw_direct_kernel<true>, grid, dim3(512), 0, s, p)
                          : rt::launch(mx_dw_direct_kernel<false>, grid, dim3(512), 0, s, p);
  else if (delta_dtype == RT_F32) launch_staged<kF32>(s, p, q, grid);
  else if (delta_dtype == RT_F16) launch_staged<kF16>(s, p, q, grid);
  else launch_staged<kBf16>(s, p, q, grid);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (q.splits > 1)
    return splitk_reduce_launch(s, scratch, q.splits, p.split_stride, p.K, p.N, C, RT_F32, p.N, RT_EPI_NONE, nullptr,
                                nullptr, RT_F32, p.shares, colsum, colsum ? p.sharers : 0);
  if (colsum && shares)
    return colsum_launch(s, p.shares, RT_F32, p.sharers, p.N, colsum, scratch + planes + shares,
                         scratch_elems - planes - shares);
  return hipSuccess;
}

}  // namespace rt

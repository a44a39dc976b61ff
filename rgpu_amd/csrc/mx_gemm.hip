// The product of microscaled tensors, C = A·Bᵀ (+ bias, ReLU), A in 4 or 8 bits
// and B in 4, on the scaled matrix instruction
// v_mfma_scale_f32_16x16x128_f8f6f4: a step of K is 128 columns, four blocks of
// 32, each with a scale of its own per row.
//
// What the instruction keeps.  It adds eight neighbouring products first, in a
// window that reaches 2^-13 below the power of two of the largest (measured: of
// 2^16 - 2^16 + 2^s in one eight nothing below s = 3 comes back; between eights
// and against the accumulator 2^-24).  4-bit products span 2^-2 to 36 and fit.
// An 8-bit A does not (its values span 2^-9 to 448).  Each of its fragments
// therefore goes in as two, the codes from 2 up and those below, with zeros in the
// others' places: products then reach from 2^-3 to below 2^12, or from 2^-10 to
// below 2^4, the sums of eight are exact, and what is left are f32 additions.
// Also for a bf16 C, which is the f32 one rounded once: A in one piece (8192 x
// 4096, K 4096: 116 us, 193 in two) changed one value in 500 of 4100 x 1000, K 4000.
//
// What a lane holds.  Lane (g, r), g = lane / 16, r = lane % 16, of an operand
// of 16 rows takes row r: the 4-bit codes of columns 32 g .. 32 g + 31 (16
// bytes), or the 8-bit codes of columns 16 g .. and 64 + 16 g .. (two times 16
// bytes); and the scale byte of row r, columns 32 g .. 32 g + 31.  The scales
// are stored so that one dword a lane serves the four 16-row operands of a
// 64-row group (the instruction picks the byte).  The operands go in swapped
// (D = B·Aᵀ), so that lane (g, r) ends with C(row r, columns 4 g .. 4 g + 3).
//
// Tiles.  Codes and scales go from global memory straight into LDS, a step per
// stage, NS stages in a ring.  A row's codes of a step are 64 or 128 bytes;
// 16-byte granule j of row i is stored at j ^ h((i / 4) % 4), h = 0, 2, 3, 1, or at
// j ^ (i / 2) % 8, which gives the 16 lanes that are served at once different
// banks.  These are not lanes 0 to 15: with h(q) = q, which would do for those,
// every read of a 4-bit fragment took twice its cycles (measured; that fits lanes
// 0-3, 12-15, 20-23 and 24-27 together, which h separates too; 8192 x 16384, K
// 4096: 304 us, 298 so).  With the fragments of step k in registers a step runs
// as: wait for step k + 1, barrier, start the loads of step k + NS into step k's
// buffer, read the fragments of step k + 1 under the MFMAs of step k.  Rows past
// the end of A or B are zeros by the buffer descriptors' range check; K is whole
// steps by the layout.
//
// Measured: 4 bits, 8192 x 16384, K 4096, bf16 C, 298-342 us (3.2-3.7 PFLOP/s, of
// 8.9 that the instruction alone reaches: matrix units busy 38%; the 268 MB of C at
// the copy rate take 52); 8 bits, 8192 x 4096, K 4096, 193-241 us (1.1 to
// 1.4 PFLOP/s); one row by 4096 x 4096 weights 4.4 us, of which a launch is 3.2.

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
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i8 __attribute__((ext_vector_type(8)));

struct Args {
  const unsigned char* a;         // codes
  const unsigned char* b;
  const unsigned char* a_scales;
  const unsigned char* b_scales;
  void* c;
  const float* bias;
  int M, N, steps;
  int a_row, b_row;        // bytes of a row of codes
  int a_groups, b_groups;  // 64-row groups
  int relu, out_bf16;
  int tiles_m, tiles_n;
};

// Fragment of 16 rows of one step: 4 or 8 dwords a lane.
template <int BITS>
struct Frag {
  u4 v[BITS / 4];
  __device__ inline i8 operand() const {
    const i4 lo = __builtin_bit_cast(i4, v[0]);
    if constexpr (BITS == 4) {
      return __builtin_shufflevector(lo, lo, 0, 1, 2, 3, -1, -1, -1, -1);
    } else {
      const i4 hi = __builtin_bit_cast(i4, v[1]);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // The 8-bit codes below 2 (large false) or from 2 up (true): those whose
  // exponent field has its top bit clear or set.
  __device__ inline Frag part(bool large) const {
    Frag f;
#pragma unroll
    for (int h = 0; h < BITS / 4; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // 0xff where the bit is set: selectors 8 to 11 spread bits 15 and 31 of
        // the second and the first word over a byte.
        const unsigned w = v[h][i], mask = __builtin_amdgcn_perm(w << 1, w << 9, 0x0b090a08u);
        f.v[h][i] = w & (large ? mask : ~mask);
      }
    return f;
  }
};

// acc[u] += (B_u·Aᵀ of one step) for TN operands B; SA: which byte of A's scale
// dword (B's: u % 4).
template <int ABITS, int SA, int TN>
__device__ inline void mfma_row(const Frag<ABITS>& a, const Frag<4> (&b)[TN], f4 (&acc)[TN], unsigned sa,
                                const unsigned (&sb)[(TN + 3) / 4]) {
  auto one = [&](const Frag<ABITS>& x) {
    static_for<0, TN>([&](auto uc) {
      constexpr int u = decltype(uc)::value, FA = ABITS == 4 ? 4 : 0;  // e2m1, e4m3
      acc[u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[u].operand(), x.operand(), acc[u], 4, FA, u & 3,
                                                                (int)sb[u / 4], SA, (int)sa);
    });
  };
  if constexpr (ABITS == 8) {
    one(a.part(false));
    one(a.part(true));
  } else {
    one(a);
  }
}

// Four consecutive columns of a row of C: bias, ReLU, rounding, bounds.
__device__ __forceinline__ void store4(const Args& p, f4 v, long long row, int col, const f4& bias, bool vec) {
  if (row >= p.M || col >= p.N) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = v[e] + bias[e];
    if (p.relu) v[e] = fmaxf(v[e], 0.0f);
  }
  const long long off = row * p.N + col;
  const int nv = min(4, p.N - col);
  if (p.out_bf16) {
    unsigned short* c = static_cast<unsigned short*>(p.c) + off;
    unsigned short h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = rt_mx::f32_to_bf16(v[e]);
    if (vec) {
      *reinterpret_cast<u2*>(c) = u2{h[0] | ((unsigned)h[1] << 16), h[2] | ((unsigned)h[3] << 16)};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < nv) c[e] = h[e];
    }
  } else {
    float* c = static_cast<float*>(p.c) + off;
    if (vec) {
      *reinterpret_cast<f4*>(c) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < nv) c[e] = v[e];
    }
  }
}

// Rows of C start on a four-column store's alignment (then N % 4 == 0, and a
// group of four is all inside or all outside).
__device__ inline bool vector_rows(const Args& p) {
  return p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.c) & (p.out_bf16 ? 7 : 15)) == 0;
}

__device__ inline f4 load_bias(const Args& p, int col) {
  f4 b = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = p.bias[min(col + e, p.N - 1)];
  }
  return b;
}

// One operand's side of a tile: ROWS rows, WAVES waves that load it.
template <int BITS, int ROWS, int WAVES>
struct Side {
  static constexpr int RB = 16 * BITS;           // bytes of a row of a step
  static constexpr int BYTES = ROWS * RB;        // codes of a stage
  static constexpr int RPI = 1024 / RB, GR = RB / 16;
  static constexpr int PER_WAVE = BYTES / 1024 / WAVES;
  static_assert(BYTES % (1024 * WAVES) == 0 && ROWS % 64 == 0, "loads split evenly over the waves");
  static_assert((RPI * WAVES) % 16 == 0, "the swizzle of a lane's granule is the same in every load");

  const unsigned char* base;  // of the tile's rows, at the step to be loaded
  int bytes;                  // the rows of a step that exist, from base
  int voff, row_step;

  // The swizzle of a row, which repeats every 16 rows (4 bits: 0, 2, 3, 1 for its quarters).
  __device__ static inline int sw(int row) {
    return BITS == 4 ? (0x78 >> (2 * ((row >> 2) & 3))) & 3 : (row >> 1) & 7;
  }
  __device__ inline void init(const unsigned char* codes, int row_bytes, long long row0, long long rows, int wave,
                              int lane) {
    base = codes + row0 * row_bytes;
    bytes = (int)min((long long)ROWS - 1, rows - row0 - 1) * row_bytes + RB;
    const int row = RPI * wave + lane / GR;
    voff = row * row_bytes + 16 * ((lane % GR) ^ sw(row));
    row_step = RPI * WAVES * row_bytes;
  }
  __device__ inline void issue(int step, unsigned lds, int wave) const {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char*>(base + (long long)step * RB), (short)0, bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i)
      rt_dev::dma16_at(rsrc, lds + 1024 * (i * WAVES + wave), voff + i * row_step);
  }
  // row0: a multiple of 16, so that all fragments of a wave differ by constants.
  __device__ static inline Frag<BITS> frag(const unsigned char* lds, int row0, int g, int r) {
    Frag<BITS> f;
#pragma unroll
    for (int h = 0; h < BITS / 4; ++h)
      f.v[h] = *reinterpret_cast<const u4*>(lds + r * RB + 16 * ((g + 4 * h) ^ sw(r)) + row0 * RB);
    return f;
  }
};

// A wave tile's rows of C as T (f32, or bf16 bits), through the wave's own part
// of LDS; N % 8 == 0 and C on 16 bytes.
template <typename T, int TM, int TN>
__device__ __forceinline__ void store_rows(const Args& p, const f4 (&acc)[TM][TN], const f4 (&bias)[TN],
                                           unsigned char* smem, int wave, int lane, long long row0, int col0) {
  constexpr int ROW = 16 * TN * sizeof(T), STRIDE = ROW + 16;      // bytes of a row of the tile
  constexpr int LPR = ROW / 16, RPI = 64 / LPR;                    // lanes a row, rows an instruction
  unsigned char* stage = smem + wave * 16 * STRIDE;
  const int g = lane >> 4, r = lane & 15, rr = lane / LPR, cc = lane % LPR;
  const int col = col0 + cc * (16 / (int)sizeof(T));
  T* out = static_cast<T*>(p.c) + col;
  static_for<0, TM>([&](auto tc) {
    constexpr int t = decltype(tc)::value;
    if constexpr (t > 0) rt_dev::wave_lds_order();
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      f4 v = acc[t][u];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = v[e] + bias[u][e];
        if (p.relu) v[e] = fmaxf(v[e], 0.0f);
      }
      unsigned char* at = stage + r * STRIDE + (16 * u + 4 * g) * sizeof(T);
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f4*>(at) = v;
      } else {
        unsigned short h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = rt_mx::f32_to_bf16(v[e]);
        *reinterpret_cast<u2*>(at) = u2{h[0] | ((unsigned)h[1] << 16), h[2] | ((unsigned)h[3] << 16)};
      }
    }
    rt_dev::wave_lds_order();  // the wave alone uses its part
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
      const long long row = row0 + 16 * t + i * RPI + rr;
      const u4 v = *reinterpret_cast<const u4*>(stage + (i * RPI + rr) * STRIDE + 16 * cc);
      if (row < p.M && col < p.N) *reinterpret_cast<u4*>(out + row * p.N) = v;
    }
  });
}

// Block tile BM x BN, WGM x WGN waves, NS stages.
template <int ABITS, int BM, int BN, int WGM, int WGN, int NS>
__global__ __launch_bounds__(64 * WGM * WGN) void mx_gemm_kernel(Args p) {
  constexpr int WAVES = WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  using A = Side<ABITS, BM, WAVES>;
  using B = Side<4, BN, WAVES>;
  // Scale dwords: one load of 64 lanes for a group, the groups dealt to the
  // waves in turn (a wave without one of its own repeats another's, so that
  // every wave has the same number of loads in flight).
  constexpr int AG = BM / 64, GROUPS = AG + BN / 64, SPW = (GROUPS + WAVES - 1) / WAVES;
  constexpr int STAGE = A::BYTES + B::BYTES + 256 * GROUPS, PER_STAGE = A::PER_WAVE + B::PER_WAVE + SPW;
  static_assert((NS - 1) * PER_STAGE < 64, "vmcnt range");
  static_assert(NS * STAGE <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) unsigned char smem[NS * STAGE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;

  // Each XCD takes a contiguous run of tiles (workgroups go to the XCDs in
  // turn), in bands of 8 tile rows, so that neighbours share an L2.
  int bid = blockIdx.x;
  const int nb = gridDim.x;
  if ((nb & 7) == 0) bid = (bid & 7) * (nb >> 3) + (bid >> 3);
  constexpr int BAND = 8;
  const int band = bid / (BAND * p.tiles_n), first_m = band * BAND;
  const int size = min(p.tiles_m - first_m, BAND), in_band = bid - band * BAND * p.tiles_n;
  const long long m0 = (long long)(first_m + in_band % size) * BM, n0 = (long long)(in_band / size) * BN;

  A sa;
  B sb;
  sa.init(p.a, p.a_row, m0, p.M, wave, lane);
  sb.init(p.b, p.b_row, n0, p.N, wave, lane);

  const unsigned smem_at = rt_dev::lds_offset(smem);
  auto issue = [&](int step, int buf) {
    const unsigned lds = smem_at + buf * STAGE;
    sa.issue(step, lds, wave);
    sb.issue(step, lds + A::BYTES, wave);
#pragma unroll
    for (int i = 0; i < SPW; ++i) {
      const int grp = (i * WAVES + wave) % GROUPS;
      const bool of_a = grp < AG;
      const int in = of_a ? grp : grp - AG, total = of_a ? p.a_groups : p.b_groups;
      const int at = (int)((of_a ? m0 : n0) / 64) + in;  // a group past the end reads nothing
      const unsigned char* src = (of_a ? p.a_scales : p.b_scales) + 256 * ((long long)step * total + min(at, total - 1));
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<unsigned char*>(src), (short)0, at < total ? 256 : 0, 0x00020000);
      rt_dev::dma4_at(rsrc, lds + A::BYTES + B::BYTES + 256 * grp, 4 * lane);
    }
  };

  struct Set {
    Frag<ABITS> a[TM];
    Frag<4> b[TN];
    unsigned as[(TM + 3) / 4], bs[(TN + 3) / 4];
  };
  auto read = [&](int buf, Set& s) {
    const unsigned char* lds = smem + buf * STAGE;
    const unsigned* sc = reinterpret_cast<const unsigned*>(lds + A::BYTES + B::BYTES);
    // A wave tile of 32 rows starts at byte 0 or 2 of its group's dwords.
#pragma unroll
    for (int i = 0; i < (TM + 3) / 4; ++i) s.as[i] = sc[64 * (wm / 64 + i) + lane] >> (TM < 4 ? 8 * ((wm >> 4) & 3) : 0);
#pragma unroll
    for (int i = 0; i < (TN + 3) / 4; ++i)
      s.bs[i] = sc[64 * (AG + wn / 64 + i) + lane] >> (TN < 4 ? 8 * ((wn >> 4) & 3) : 0);
#pragma unroll
    for (int u = 0; u < TN; ++u) s.b[u] = B::frag(lds + A::BYTES, wn + 16 * u, g, r);
#pragma unroll
    for (int t = 0; t < TM; ++t) s.a[t] = A::frag(lds, wm + 16 * t, g, r);
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int u = 0; u < TN; ++u) acc[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  auto mfmas = [&](const Set& s) {
    static_for<0, TM>([&](auto tc) {
      constexpr int t = decltype(tc)::value;
      mfma_row<ABITS, t & 3, TN>(s.a[t], s.b, acc[t], s.as[t / 4], s.bs);
    });
  };

  if (p.steps > 0) {
    const int last = p.steps - 1;
    static_for<0, NS>([&](auto ic) { issue(min((int)decltype(ic)::value, last), decltype(ic)::value); });
    wait_vm<(NS - 1) * PER_STAGE>();
    barrier_lds();
    Set s0, s1;
    read(0, s0);
    // Past the last step the loads repeat it, into a buffer that nothing reads,
    // so that every step has the same number in flight.
    auto step = [&](int k, int buf, const Set& cur, Set& next) {
      wait_vm<(NS - 2) * PER_STAGE>();
      barrier_lds();
      issue(min(k + NS, last), buf);
      read(buf + 1 == NS ? 0 : buf + 1, next);
      mfmas(cur);
    };
    constexpr int UNROLL = NS % 2 ? 2 * NS : NS;
    for (int k = 0; k < p.steps; k += UNROLL) {
      static_for<0, UNROLL>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (k + i < p.steps) {
          if constexpr (i % 2 == 0) step(k + i, i % NS, s0, s1);
          else step(k + i, i % NS, s1, s0);
        }
      });
    }
  }
  wait_vm<0>();  // the block's LDS is given up only once no load writes it

  const bool vec = vector_rows(p);
  f4 bias[TN];
#pragma unroll
  for (int u = 0; u < TN; ++u) bias[u] = load_bias(p, (int)n0 + wn + 16 * u + 4 * g);
  // Whole rows: 16 rows of the wave's columns at a time go through LDS, so that
  // a store instruction covers a row's 64 to 256 bytes (a lane's own 8 or 16
  // are 32 or 64 consecutive ones for four lanes).
  const bool whole = p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0;
  if (whole) {
    __syncthreads();  // no wave reads its fragments any more
    if (p.out_bf16) store_rows<unsigned short, TM, TN>(p, acc, bias, smem, wave, lane, m0 + wm, (int)n0 + wn);
    else store_rows<float, TM, TN>(p, acc, bias, smem, wave, lane, m0 + wm, (int)n0 + wn);
    return;
  }
  static_for<0, TM>([&](auto tc) {
    static_for<0, TN>([&](auto uc) {
      constexpr int t = decltype(tc)::value, u = decltype(uc)::value;
      store4(p, acc[t][u], m0 + wm + 16 * t + r, (int)n0 + wn + 16 * u + 4 * g, bias[u], vec);
    });
  });
}

// A product of at most 64 rows (tokens of a few requests): bound by reading B
// once and by latency.  A block takes 16 columns of C, its 8 waves deal the
// steps of K among them, four consecutive ones a time (each row of B is then
// read 256 bytes a time), straight from global memory into registers,
// and add their sums in LDS in wave order.
constexpr int kRowWaves = 8, kRowSteps = 4;

template <int ABITS, int TM>
__global__ __launch_bounds__(64 * kRowWaves) void mx_rows_kernel(Args p) {
  __shared__ f4 red[kRowWaves][TM][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int n0 = 16 * blockIdx.x;
  // Rows past the end repeat the last one; what they give is not stored.
  const unsigned char* b = p.b + (long long)min(n0 + r, p.N - 1) * p.b_row + 16 * g;
  const unsigned char* a[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) a[t] = p.a + (long long)min(16 * t + r, p.M - 1) * p.a_row + 16 * g;
  const unsigned* as = reinterpret_cast<const unsigned*>(p.a_scales) + lane;
  const unsigned* bs = reinterpret_cast<const unsigned*>(p.b_scales) + 64LL * (n0 / 64) + lane;
  const int bshift = 8 * ((n0 >> 4) & 3);

  f4 acc[TM][1];
#pragma unroll
  for (int t = 0; t < TM; ++t) acc[t][0] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = kRowSteps * wave; k0 < p.steps; k0 += kRowSteps * kRowWaves) {
    Frag<4> fb[kRowSteps][1];
    Frag<ABITS> fa[kRowSteps][TM];
    unsigned sa[kRowSteps], sb[kRowSteps][1];
#pragma unroll
    for (int i = 0; i < kRowSteps; ++i) {
      const int k = min(k0 + i, p.steps - 1);  // steps past the end are loaded but not used
      fb[i][0].v[0] = *reinterpret_cast<const u4*>(b + (long long)k * 64);
#pragma unroll
      for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int h = 0; h < ABITS / 4; ++h)
          fa[i][t].v[h] = *reinterpret_cast<const u4*>(a[t] + (long long)k * 16 * ABITS + 64 * h);
      sa[i] = as[64LL * k * p.a_groups];
      sb[i][0] = bs[64LL * k * p.b_groups] >> bshift;
    }
#pragma unroll
    for (int i = 0; i < kRowSteps; ++i) {
      if (k0 + i < p.steps) {
        static_for<0, TM>([&](auto tc) {
          constexpr int t = decltype(tc)::value;
          mfma_row<ABITS, t & 3, 1>(fa[i][t], fb[i], acc[t], sa[i], sb[i]);
        });
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TM; ++t) red[wave][t][lane] = acc[t][0];
  __syncthreads();
  if ((int)threadIdx.x < 64 * TM) {
    const int t = threadIdx.x >> 6;
    f4 v = red[0][t][lane];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) v += red[w][t][lane];
    store4(p, v, 16 * t + r, n0 + 4 * g, load_bias(p, n0 + 4 * g), vector_rows(p));
  }
}

template <int ABITS, int BM, int BN, int WGM, int WGN, int NS>
hipError_t launch_tiles(hipStream_t s, Args p) {
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  rt::launch(mx_gemm_kernel<ABITS, BM, BN, WGM, WGN, NS>,
             dim3((unsigned)((long long)p.tiles_m * p.tiles_n)), dim3(64 * WGM * WGN), 0, s, p);
  return hipGetLastError();
}

// Tiles by what fills the chip.  256 x 256 (4 bits) has a CU to itself, so it
// takes whole rounds of 256, or a last one that leaves no more than a third of
// all places idle (us with 256 and 128 tiles: 4096 x 4096, K 1024, 256 blocks,
// 19.0 and 21.1; K 4096: 6912 x 4864, 513 blocks, 104 and 110; 4608 x 4096, 288
// blocks, 66 and 56).  128 x 128, two a CU, from 208 blocks on (8 bits, us with 128
// and 64 tiles: 1800 x 1800, K 2000, 225 blocks, 20.8 and 24.7; 2048 x 4096, K
// 1024, 512 blocks, 23.2 and 30.6; 700 x 4096, K 1000, 192 blocks, 13.1 and 12.0).
template <int ABITS>
hipError_t launch_many(hipStream_t s, const Args& p) {
  auto tiles = [&](int t) { return (long long)((p.M + t - 1) / t) * ((p.N + t - 1) / t); };
  if constexpr (ABITS == 4) {
    const long long t = tiles(256), places = (t + 255) / 256 * 256;
    if (t >= 256 && 2 * places <= 3 * t) return launch_tiles<4, 256, 256, 2, 4, 4>(s, p);
  }
  if (tiles(128) >= 208) return launch_tiles<ABITS, 128, 128, 2, 2, 3>(s, p);
  return launch_tiles<ABITS, 64, 64, 2, 2, 4>(s, p);
}

// Few rows stay with the kernel that reads B once and A again for every 16
// columns, up to 48, or 64 over a short K, or for 8 bits where its blocks are one
// round of the CUs (8 bits, us there and with 64 tiles: N 4096, K 4096, 49 rows 11.1
// and 15.0, 64 rows 12.6 and 15.0; N 1000, K 4000, 64 rows 11.9 and 14.7; N 16384,
// K 4096, 64 rows 43.4 and 16.8.  4 bits, N 4096, 64 rows: K 1024 4.7 with 64 tiles).
template <int ABITS>
hipError_t launch(hipStream_t s, const Args& p) {
  // (A grid holds fewer than 2^32 threads.)
  const bool one_round = ABITS == 8 && p.N <= 16 * 256;
  if ((p.M <= 48 || (p.M <= 64 && (p.steps <= 8 || one_round))) && p.N <= (1 << 26)) {
    const dim3 grid((unsigned)((p.N + 15) / 16)), block(64 * kRowWaves);
    const int tm = (p.M + 15) / 16;
    if (tm == 1) rt::launch(mx_rows_kernel<ABITS, 1>, grid, block, 0, s, p);
    else if (tm == 2) rt::launch(mx_rows_kernel<ABITS, 2>, grid, block, 0, s, p);
    else if (tm == 3) rt::launch(mx_rows_kernel<ABITS, 3>, grid, block, 0, s, p);
    else rt::launch(mx_rows_kernel<ABITS, 4>, grid, block, 0, s, p);
    return hipGetLastError();
  }
  return launch_many<ABITS>(s, p);
}

}  // namespace

namespace rt {

hipError_t mx_gemm_launch(hipStream_t s, const MxTensor& a, const MxTensor& b, void* C, int out_dtype, int epi,
                          const float* bias) {
  const MxLayout la = mx_layout(a.dtype, a.rows, a.cols), lb = mx_layout(b.dtype, b.rows, b.cols);
  Args p{};
  p.a = a.codes;
  p.b = b.codes;
  p.a_scales = a.scales;
  p.b_scales = b.scales;
  p.c = C;
  p.bias = epi == RT_EPI_NONE ? nullptr : bias;
  p.M = (int)a.rows;
  p.N = (int)b.rows;
  p.steps = a.cols > 0 ? (int)la.steps : 0;
  p.a_row = (int)la.row_bytes;
  p.b_row = (int)lb.row_bytes;
  p.a_groups = (int)la.groups;
  p.b_groups = (int)lb.groups;
  p.relu = epi == RT_EPI_BIAS_RELU;
  p.out_bf16 = out_dtype == RT_BF16;
  return a.dtype == RT_MXFP4 ? launch<4>(s, p) : launch<8>(s, p);
}

}  // namespace rt

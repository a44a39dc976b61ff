// Products of the experts that tokens were routed to, over rows in the order
// of their experts (rt_sort_ids: expert e has rows offsets[e] ..
// offsets[e + 1]), and what joins a token's rows again.
//
//   NN  C[p] = A[row(p)] W_e + b_e      p in expert e's rows; row(p) = p, or
//                                       order[p] / k: the token of choice order[p]
//   NT  C[p] = A[p] W_eᵀ
//   TN  C_e  = sum over e's rows p of A[row(p)]ᵀ B[p], and B's column sums
//
// The offsets stay on the device: a launch covers the most tiles that n rows in
// E groups can have (n / BM + E), and a block finds its expert and rows in the
// offsets.  Operands are staged through LDS; 16x16 MFMA tiles with f32 accumulators
// (bf16 and f16: 16x16x32; f32: four 16x16x4 for each 16 of K, in f32).

#include <algorithm>
#include <type_traits>

#include "device_util.h"
#include "dma_operand.h"
#include "elems.h"
#include "experts_dev.h"
#include "rt_internal.h"

namespace {

using rt_dev::barrier_lds;
using rt::ExpertArgs;
using rt::token_of;
using rt_dev::DmaOperand;
using rt_dev::experts_tiles;
using rt_dev::static_for;
using rt_dev::Tile;
using rt_dev::tile_of;
using rt_dev::u2;
using rt_dev::u4;
using rt_dev::wait_vm;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxExperts = 1024;

// Elements of a granule of 16 bytes, from index i of which n exist.
template <int ES>
__device__ inline u4 granule(const void* base, long long i, int n) {
  constexpr int PER = 16 / ES;
  u4 v = {0u, 0u, 0u, 0u};
  const char* p = static_cast<const char*>(base) + i * ES;
  if (n >= PER) {
    __builtin_memcpy(&v, p, 16);
  } else if constexpr (ES == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? reinterpret_cast<const unsigned*>(p)[e] : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e >> 1] |= e < n ? (unsigned)reinterpret_cast<const unsigned short*>(p)[e] << (16 * (e & 1)) : 0u;
  }
  return v;
}

// The results of a wave, lane (g, r) holding columns col0 + 16 u + 4 g .. of rows
// row0 + 16 t + r, through the epilogue into C.  They go 16 rows at a time through
// the wave's own 16 x (16 TN + 4) floats of LDS (stage), so that a store writes
// whole rows of the tile: from the registers it would write 64 bytes a row.
template <int DT, int LAYOUT, int TM, int TN>
__device__ __forceinline__ void write_tile(const ExpertArgs& p, const Tile& tile, const f4 (&acc)[TM][TN], long long row0,
                                           int col0, int lane, float* stage) {
  constexpr int ROW = 16 * TN + 4, LANES = 4 * TN, ROWS = 64 / LANES;  // lanes a row, rows a turn
  const int n_end = LAYOUT == RT_NT ? p.c_K : p.c_N;
  const long long m_end = LAYOUT == RT_TN ? (long long)p.c_K : tile.r1;
  const long long c_base = LAYOUT == RT_TN ? (long long)tile.plane * p.c_K * p.c_N : 0;
  const bool same = DT != RT_F32 && p.c_same;
  const int g = lane >> 4, r = lane & 15, col = col0 + 4 * (lane % LANES), nv = min(4, n_end - col);
  float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.epi == RT_EPI_BIAS || p.epi == RT_EPI_BIAS_RELU) {
    const float* bias = p.bias + (long long)tile.expert * p.c_N;
#pragma unroll
    for (int q = 0; q < 4; ++q) add[q] = bias[min(col + q, n_end - 1)];
  }
  static_for<0, TM>([&](auto tc) {
    constexpr int t = decltype(tc)::value;
    if (row0 + 16 * t >= m_end) return;
    rt_dev::wave_lds_order();
#pragma unroll
    for (int u = 0; u < TN; ++u) *reinterpret_cast<f4*>(stage + r * ROW + 16 * u + 4 * g) = acc[t][u];
    rt_dev::wave_lds_order();
#pragma unroll
    for (int i = 0; i < 16 / ROWS; ++i) {
      const int in = i * ROWS + lane / LANES;
      const long long row = row0 + 16 * t + in;
      if (row >= m_end || nv <= 0) continue;
      const long long at = c_base + row * n_end + col;
      const f4 x = *reinterpret_cast<const f4*>(stage + in * ROW + 4 * (lane % LANES));
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = x[q];
      if (p.epi == RT_EPI_BIAS || p.epi == RT_EPI_BIAS_RELU) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] += add[q];
          if (p.epi == RT_EPI_BIAS_RELU) v[q] = fmaxf(v[q], 0.0f);
        }
      } else if (p.epi == RT_EPI_RELU_MASK) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const long long i = at + min(q, nv - 1);
          const float m = same ? rt_dev::load1<DT>(p.mask, i) : static_cast<const float*>(p.mask)[i];
          v[q] = m > 0.0f ? v[q] : 0.0f;
        }
      }
      if (same) {
        if (nv == 4) {
          unsigned h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = DT == RT_BF16 ? rt_dev::bf16_bits(v[q]) : rt_dev::f16_bits(v[q]);
          const u2 o = {h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
          __builtin_memcpy(static_cast<unsigned short*>(p.C) + at, &o, 8);
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (q < nv) rt_dev::store1<DT>(p.C, at + q, v[q]);
        }
      } else if (nv == 4) {
        __builtin_memcpy(static_cast<float*>(p.C) + at, v, 16);
      } else {
#pragma unroll
        for (int q = 0; q < 3; ++q)
          if (q < nv) static_cast<float*>(p.C)[at + q] = v[q];
      }
    }
  });
}

// The TN layout's column sums of B, by the tiles of the first rows: a thread
// adds up 8 columns of every 16th row of a stage, and the 16 sums of a column
// are added in their order, so the bits do not depend on the tile.
template <int DT, int LAYOUT, int BN, int THREADS, int BK>
struct ColumnSums {
  static constexpr int CH = BN / 8, KG = 16;
  static_assert(LAYOUT != RT_TN || (BK % KG == 0 && KG * CH <= THREADS), "a thread a share");
  const bool on;
  const int tid;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  __device__ inline ColumnSums(const ExpertArgs& p, long long m0, int t)
      : on(LAYOUT == RT_TN && p.colsum != nullptr && m0 == 0), tid(t) {}
  // at(row, c): columns 8 c .. of a row of the stage, in LDS on 16 bytes.
  template <class F>
  __device__ inline void add(F&& at) {
    if constexpr (LAYOUT == RT_TN) {
      if (!on || tid >= KG * CH) return;
#pragma unroll
      for (int k = tid / CH; k < BK; k += KG) {
        float x[8];
        rt_dev::load8<DT>(__builtin_assume_aligned(at(k, tid % CH), 16), 0, 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += x[e];
      }
    }
  }
  // After a barrier; red holds [KG][BN].
  __device__ inline void write(const ExpertArgs& p, const Tile& tile, float* red) {
    if constexpr (LAYOUT == RT_TN) {
      if (!on) return;
      if (tid < KG * CH) {
#pragma unroll
        for (int e = 0; e < 8; ++e) red[(tid / CH) * BN + 8 * (tid % CH) + e] = sum[e];
      }
      __syncthreads();
      for (int col = tid; col < BN && tile.n0 + col < p.c_N; col += THREADS) {
        float v = 0.0f;
        for (int j = 0; j < KG; ++j) v += red[j * BN + col];
        p.colsum[(long long)tile.plane * p.c_N + tile.n0 + col] = v;
      }
      __syncthreads();
    }
  }
};

template <int DT, int LAYOUT, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN) void experts_kernel(ExpertArgs p) {
  constexpr int ES = DT == RT_F32 ? 4 : 2, EPG = 16 / ES, BK = 128 / ES;  // a stage is 128 bytes of K
  constexpr int THREADS = 64 * WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr bool A_KC = LAYOUT != RT_TN, B_KC = LAYOUT == RT_NT;
  // K-contiguous tiles are [row][8 granules], granule g of row r at g ^ ((r >>
  // 1) & 7); the others [k][columns + pad]: 16 halves (the transposing reads) or
  // 4 floats (16 columns of k rows 4 apart) keep the reads off each other's banks.
  constexpr int PAD = ES == 4 ? 4 : 16;
  constexpr int A_ROW = A_KC ? 128 : (BM + PAD) * ES, B_ROW = B_KC ? 128 : (BN + PAD) * ES;  // bytes
  constexpr int A_BYTES = (A_KC ? BM : BK) * A_ROW, B_BYTES = (B_KC ? BN : BK) * B_ROW;
  constexpr int A_PER = (BM * 8 + THREADS - 1) / THREADS, B_PER = (BN * 8 + THREADS - 1) / THREADS;  // granules a thread
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * (A_BYTES + B_BYTES)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, r = lane & 15;
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;

  const Tile rows = tile_of<LAYOUT, BM, BN>(p, lane);
  if (rows.expert < 0) return;
  const long long m0 = rows.m0;
  const int n0 = rows.n0, n_end = LAYOUT == RT_NT ? p.K : p.N;
  const long long m_end = LAYOUT == RT_TN ? (long long)p.K : rows.r1;
  const int a_ld = LAYOUT == RT_NT ? p.N : p.K;  // elements a row of A
  // K of the product: W's K (NN), W's N (NT), the expert's rows (TN).
  const long long k_len = LAYOUT == RT_NN ? p.K : LAYOUT == RT_NT ? p.N : rows.r1 - rows.r0;
  const char* w = static_cast<const char*>(p.B) + (LAYOUT == RT_TN ? 0 : (long long)rows.expert * p.K * p.N * ES);

  auto a_row = [&](long long q) -> long long {  // the row of A of row q, -1 if there is none
    if (!p.order) return q;
    const long long t = token_of(p, p.order[q]);
    return t < p.a_rows ? t : -1;
  };
  // K-contiguous A: the rows of this thread's granules stay the same.
  long long arow[A_PER];
  if constexpr (A_KC) {
#pragma unroll
    for (int i = 0; i < A_PER; ++i) {
      const int row = (tid + THREADS * i) / 8;
      arow[i] = row < BM && m0 + row < m_end ? a_row(m0 + row) : -1;
    }
  }
  u4 va[A_PER], vb[B_PER];
  auto load = [&](long long k0) {
#pragma unroll
    for (int i = 0; i < A_PER; ++i) {
      const int idx = tid + THREADS * i;
      if constexpr (A_KC) {
        const long long k = k0 + (idx % 8) * EPG;
        va[i] = arow[i] >= 0 ? granule<ES>(p.A, arow[i] * a_ld + k, (int)(k_len - k)) : u4{0, 0, 0, 0};
      } else {
        const int kk = idx / (BM / EPG), c = (idx % (BM / EPG)) * EPG;
        const long long q = rows.r0 + k0 + kk, t = kk < BK && q < rows.r1 ? a_row(q) : -1;
        va[i] = t >= 0 ? granule<ES>(p.A, t * a_ld + m0 + c, (int)(p.K - m0 - c)) : u4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int i = 0; i < B_PER; ++i) {
      const int idx = tid + THREADS * i;
      if constexpr (B_KC) {
        const int row = idx / 8;
        const long long k = k0 + (idx % 8) * EPG;
        vb[i] = row < BN && n0 + row < n_end ? granule<ES>(w, (long long)(n0 + row) * p.N + k, (int)(k_len - k))
                                             : u4{0, 0, 0, 0};
      } else {
        const int kk = idx / (BN / EPG), c = (idx % (BN / EPG)) * EPG;
        const bool in = kk < BK && k0 + kk < k_len;
        vb[i] = in ? granule<ES>(w, ((LAYOUT == RT_TN ? rows.r0 : 0) + k0 + kk) * p.N + n0 + c, p.N - n0 - c)
                   : u4{0, 0, 0, 0};
      }
    }
  };
  auto swz = [](int row, int gr) { return 16 * (gr ^ ((row >> 1) & 7)); };
  auto sA = [&](int buf) { return smem + buf * (A_BYTES + B_BYTES); };
  auto sB = [&](int buf) { return smem + buf * (A_BYTES + B_BYTES) + A_BYTES; };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < A_PER; ++i) {
      const int idx = tid + THREADS * i;
      if ((BM * 8) % THREADS != 0 && idx >= BM * 8) continue;
      const int at = A_KC ? (idx / 8) * 128 + swz(idx / 8, idx % 8) : (idx / (BM / EPG)) * A_ROW + 16 * (idx % (BM / EPG));
      *reinterpret_cast<u4*>(sA(buf) + at) = va[i];
    }
#pragma unroll
    for (int i = 0; i < B_PER; ++i) {
      const int idx = tid + THREADS * i;
      if ((BN * 8) % THREADS != 0 && idx >= BN * 8) continue;
      const int at = B_KC ? (idx / 8) * 128 + swz(idx / 8, idx % 8) : (idx / (BN / EPG)) * B_ROW + 16 * (idx % (BN / EPG));
      *reinterpret_cast<u4*>(sB(buf) + at) = vb[i];
    }
  };
  // The 16 bytes of lane (g, r) for rows (columns) base + r and granules 4 kk
  // + g of K: eight halves, or four floats of which the j-th goes to the j-th
  // MFMA (which k a lane's element stands for is the same for A and B).
  auto frag = [&](const unsigned char* lds, auto kc, int row_bytes, int kk, int base) -> u4 {
    if constexpr (decltype(kc)::value) {
      return *reinterpret_cast<const u4*>(lds + (base + r) * 128 + swz(base + r, 4 * kk + g));
    } else if constexpr (ES == 2) {
      const unsigned char* q = lds + (32 * kk + 8 * g + (r >> 2)) * row_bytes + 2 * (base + 4 * (r & 3));
      const u2 a = rt_dev::lds_tr(reinterpret_cast<const unsigned short*>(q));
      const u2 b = rt_dev::lds_tr(reinterpret_cast<const unsigned short*>(q + 4 * row_bytes));
      return u4{a[0], a[1], b[0], b[1]};
    } else {
      u4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = *reinterpret_cast<const unsigned*>(lds + (16 * kk + 4 * g + j) * row_bytes + 4 * (base + r));
      return v;
    }
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int u = 0; u < TN; ++u) acc[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  ColumnSums<DT, LAYOUT, BN, THREADS, BK> cs(p, m0, tid);
  const long long nk = (k_len + BK - 1) / BK;
  if (nk > 0) {
    load(0);
    store(0);
    __syncthreads();
    for (long long k = 0; k < nk; ++k) {
      const int cur = (int)(k & 1);
      if (k + 1 < nk) load((k + 1) * BK);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u4 fb[TN];
#pragma unroll
        for (int u = 0; u < TN; ++u) fb[u] = frag(sB(cur), std::integral_constant<bool, B_KC>{}, B_ROW, kk, wn + 16 * u);
#pragma unroll
        for (int t = 0; t < TM; ++t) {
          const u4 fa = frag(sA(cur), std::integral_constant<bool, A_KC>{}, A_ROW, kk, wm + 16 * t);
#pragma unroll
          for (int u = 0; u < TN; ++u) {
            // Operands swapped: a lane's four results are columns 4 g .. of row r.
            if constexpr (DT == RT_BF16)
              acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[u]),
                                                                  __builtin_bit_cast(bf16x8, fa), acc[t][u], 0, 0, 0);
            else if constexpr (DT == RT_F16)
              acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fb[u]),
                                                                 __builtin_bit_cast(f16x8, fa), acc[t][u], 0, 0, 0);
            else
#pragma unroll
              for (int j = 0; j < 4; ++j)
                acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(fb[u][j]), __uint_as_float(fa[j]),
                                                                 acc[t][u], 0, 0, 0);
          }
        }
      }
      cs.add([&](int row, int c8) { return sB(cur) + row * B_ROW + 8 * ES * c8; });
      if (k + 1 < nk) store(cur ^ 1);
      __syncthreads();
    }
  }
  cs.write(p, rows, reinterpret_cast<float*>(smem));
  write_tile<DT, LAYOUT, TM, TN>(p, rows, acc, m0 + wm, n0 + wn, lane,
                                 reinterpret_cast<float*>(smem) + wave * 16 * (16 * TN + 4));
}

// ------------------------------------------------------------------ direct-to-LDS kernel
// bf16 and f16 operands whose rows are whole granules of 16 bytes: the tiles of
// a stage go from global memory straight into LDS (DmaOperand's layouts), in NS
// stages, and each half of a stage's MFMAs runs while the other half's fragments
// are read.  The schedule is that of gemm_half.hip's kernel; what differs is
// A's rows, whose offsets each lane looks up: for K-contiguous A once, for the
// TN layout, where they are the rows of a stage, a stage ahead, by loads that are
// waited for with the stage's own.
template <int DT, int LAYOUT, int BM, int BN, int WGM, int WGN, int NS>
__global__ __launch_bounds__(64 * WGM * WGN) void experts_dma_kernel(ExpertArgs p) {
  constexpr int THREADS = 64 * WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16, BK = 64;
  constexpr bool A_KC = LAYOUT != RT_TN, B_KC = LAYOUT == RT_NT;
  using OpA = DmaOperand<BM, A_KC, THREADS, BK>;
  using OpB = DmaOperand<BN, B_KC, THREADS, BK>;
  // TN: with a stage's tiles go the choices of the rows of the stage NS after it,
  // into the slot of a ring (a wave's own) that this one's were read from.  They
  // are older than every load that a wait leaves in flight when they are read.
  constexpr int STAGE = OpA::ELEMS + OpB::ELEMS, PER_STAGE = OpA::PER_WAVE + OpB::PER_WAVE + !A_KC;
  constexpr int RING = A_KC ? 0 : NS * BK;  // words a wave
  constexpr int END = 0x7ffffff0;  // past every operand
  static_assert((NS - 1) * PER_STAGE < 64, "vmcnt range");
  __shared__ __attribute__((aligned(16))) unsigned short
      smem[NS * STAGE + WGM * WGN * RING * 2];
  auto sA = [&](int buf) { return smem + buf * STAGE; };
  auto sB = [&](int buf) { return smem + buf * STAGE + OpA::ELEMS; };
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;
  const Tile tile = tile_of<LAYOUT, BM, BN>(p, lane);
  if (tile.expert < 0) return;
  const long long m0 = tile.m0;
  const int n0 = tile.n0, a_ld = LAYOUT == RT_NT ? p.N : p.K;
  const int kn = LAYOUT == RT_NN ? p.K : LAYOUT == RT_NT ? p.N : (int)(tile.r1 - tile.r0);
  const int nk = (kn + BK - 1) / BK;

  const unsigned short* const a = static_cast<const unsigned short*>(p.A);
  OpA oa;
  OpB ob;
  auto sized = [](const unsigned short* at, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(at), (short)0,
                                             (int)min(max(bytes, 0LL), (long long)END), 0x00020000);
  };
  // Byte offset of A's row for row q of all rows, from the descriptor's base.
  const int a_first = p.order ? 0 : LAYOUT == RT_TN ? (int)tile.r0 : (int)m0, r1 = (int)tile.r1;
  auto row_off = [&](int q, unsigned choice) -> int {
    const unsigned t = p.order ? token_of(p, choice) : (unsigned)(q - a_first);
    return q < r1 && t < (unsigned)p.a_rows ? (int)(t * (unsigned)(2 * a_ld)) : END;
  };
  int av[OpA::PER_WAVE];  // this lane's offsets (A_KC: of every stage; TN: of the stage to come)
  bool past = false;      // A_KC: this lane's granule of the last stage is behind K
  int k_row = 0, col_off[2] = {0, 0};
  __amdgpu_buffer_rsrc_t choices = oa.rsrc;
  unsigned* const ring = reinterpret_cast<unsigned*>(smem + NS * STAGE) + wave * RING;
  if constexpr (A_KC) {
    const int row = (512 / BK) * wave + lane / OpA::GR, gr = (lane % OpA::GR) ^ OpA::kc_sw(row);
    past = 8 * gr >= kn - (nk - 1) * BK;
#pragma unroll
    for (int i = 0; i < OpA::PER_WAVE; ++i) {
      const int q = (int)m0 + row + i * OpA::RSTEP;
      const int off = row_off(q, p.order && q < r1 ? p.order[q] : 0u);
      av[i] = off == END ? END : off + 16 * gr;
    }
    oa.rsrc = sized(a + (long long)a_first * a_ld, ((p.order ? p.a_rows : p.n) - a_first) * 2 * a_ld);
  } else {
    constexpr int CH = BM / 8;
    const int s = lane % CH;
    k_row = (512 / BM) * wave + lane / CH;
#pragma unroll
    for (int par = 0; par < 2; ++par)
      col_off[par] = 2 * (16 * ((s >> 1) ^ OpA::hm(k_row + par * OpA::RSTEP)) + 8 * (s & 1));
    oa.rsrc = sized(a + (long long)a_first * a_ld + m0, (((p.order ? p.a_rows : p.n) - a_first) * a_ld - m0) * 2);
    // Without an order the descriptor is empty: the loads are counted all the same.
    choices = sized(reinterpret_cast<const unsigned short*>(p.order + tile.r0), p.order ? (tile.r1 - tile.r0) * 4 : 0);
  }
  auto look_up = [&](int stage) {  // TN: the choices of a stage's rows, into the wave's ring
    if constexpr (!A_KC)
      rt_dev::dma4_at(choices, rt_dev::lds_offset(ring + (stage % NS) * BK), 4 * (stage * BK + lane));
  };
  auto place = [&](int stage) {  // TN: the offsets of a stage's rows
    if constexpr (!A_KC) {
#pragma unroll
      for (int i = 0; i < OpA::PER_WAVE; ++i) {
        const int k = k_row + i * OpA::RSTEP;
        const int off = row_off((int)tile.r0 + stage * BK + k, ring[(stage % NS) * BK + k]);
        av[i] = off == END ? END : off + col_off[OpA::PAR ? (i & 1) : 0];
      }
    }
  };
  auto issue_a = [&](int stage, int buf) {
    const bool last = stage == nk - 1;
#pragma unroll
    for (int i = 0; i < OpA::PER_WAVE; ++i)
      rt_dev::dma16_asm(oa.rsrc, sA(buf) + 512 * (i * OpA::WAVES + wave), A_KC && last && past ? END : av[i],
                        A_KC ? stage * 2 * BK : 0);
  };
  const unsigned short* const b = static_cast<const unsigned short*>(p.B) +
                                  (LAYOUT == RT_TN ? tile.r0 * p.N : (long long)tile.expert * p.K * p.N) +
                                  (B_KC ? (long long)n0 * p.N : n0);
  // TN: the descriptor ends with the expert's rows, whose products the next rows are no part of.
  const long long b_end = LAYOUT == RT_TN ? (tile.r1 - tile.r0) * p.N - n0 : B_KC ? (long long)(p.K - n0) * p.N : (long long)p.K * p.N - n0;
  ob.init(b, p.N, wave, lane);
  ob.rsrc = sized(b, 2 * b_end);
  const bool past_b = B_KC && 8 * ((lane % OpB::GR) ^ OpB::kc_sw((512 / BK) * wave + lane / OpB::GR)) >= kn - (nk - 1) * BK;
  const int b_step = 2 * (B_KC ? BK : BK * p.N);
  auto issue_b = [&](int stage, int buf) {
    const bool last = stage == nk - 1;
#pragma unroll
    for (int i = 0; i < OpB::PER_WAVE; ++i)  // all of it in the vector part, which the range check looks at
      rt_dev::dma16_asm(ob.rsrc, sB(buf) + 512 * (i * OpB::WAVES + wave),
                        rt_dev::past_end_offset(last && past_b ? END : ob.voff[OpB::PAR ? (i & 1) : 0],
                                                (unsigned)(stage * b_step) + (unsigned)(i * OpB::RSTEP * 2 * p.N)),
                        0);
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int u = 0; u < TN; ++u) acc[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  // With two waves a SIMD their addresses are made anew each time, from the lane
  // alone: held through the loop they spill, and a reload waits for every load
  // in flight.
  auto read_frags = [&](int buf, int kk, u4 (&fa)[TM], u4 (&fb)[TN]) {
    int l = lane;
    if constexpr (THREADS > 256) asm volatile("" : "+v"(l));
    const int g = l >> 4, r = l & 15;
#pragma unroll
    for (int u = 0; u < TN; ++u) fb[u] = ob.frag(sB(buf), kk, wn + 16 * u, g, r);
#pragma unroll
    for (int t = 0; t < TM; ++t) fa[t] = oa.frag(sA(buf), kk, wm + 16 * t, g, r);
  };
  auto mfmas = [&](const u4 (&fa)[TM], const u4 (&fb)[TN]) {
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int u = 0; u < TN; ++u) {
        if constexpr (DT == RT_BF16)
          acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[u]),
                                                              __builtin_bit_cast(bf16x8, fa[t]), acc[t][u], 0, 0, 0);
        else
          acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fb[u]),
                                                             __builtin_bit_cast(f16x8, fa[t]), acc[t][u], 0, 0, 0);
      }
  };
  constexpr int N_DS = (A_KC ? TM : 2 * TM) + (B_KC ? TN : 2 * TN), N_MF = TM * TN;
  // One MFMA, one LDS read, ...; one MFMA, one (VG) loads, ...; the other MFMAs.
  auto interleave = [&](auto n_vm) {
    constexpr int N_VM = decltype(n_vm)::value;
    constexpr int VG = N_MF >= 32 && N_DS + N_VM > N_MF ? 2 : 1, GROUPS = (N_VM + VG - 1) / VG;
    if constexpr (N_DS + GROUPS <= N_MF) {
      static_for<0, N_DS>([&](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      });
      static_for<0, GROUPS>([&](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, VG, 0);
      });
      __builtin_amdgcn_sched_group_barrier(0x008, N_MF - N_DS - GROUPS, 0);
    }
  };
  ColumnSums<DT, LAYOUT, BN, THREADS, BK> cs(p, m0, tid);

  if (nk > 0) {
    u4 fa0[TM], fb0[TN], fa1[TM], fb1[TN];
    if constexpr (!A_KC) {
      static_for<0, NS>([&](auto ic) { look_up(decltype(ic)::value); });
      wait_vm<0>();
      __syncthreads();
    }
    // Past the last stage the last one is loaded again, by whatever choices its
    // slot holds, into a buffer that nothing reads.
    static_for<0, NS>([&](auto ic) {
      constexpr int S = decltype(ic)::value;
      place(min(S, nk - 1));
      issue_a(min(S, nk - 1), S);
      look_up(S + NS);  // after the loads that took its slot's choices
      issue_b(min(S, nk - 1), S);
    });
    wait_vm<(NS - 1) * PER_STAGE>();
    barrier_lds();
    read_frags(0, 0, fa0, fb0);
    auto stage = [&](int k, auto bc) {
      constexpr int BUF = decltype(bc)::value, NEXT = (BUF + 1) % NS;
      const int next = min(k + NS, nk - 1);
      read_frags(BUF, 1, fa1, fb1);
      mfmas(fa0, fb0);
      interleave(std::integral_constant<int, 0>{});
      cs.add([&](int row, int c8) {  // OpB::row_chunk's place
        return sB(BUF) + row * BN + 16 * ((c8 >> 1) ^ OpB::hm(row)) + 8 * (c8 & 1);
      });
      wait_vm<(NS - 2) * PER_STAGE>();  // stage k + 1 (TN: and the rows' choices)
      barrier_lds();
      place(next);
      issue_a(next, BUF);
      look_up(k + 2 * NS);
      if constexpr (B_KC) issue_b(next, BUF);
      read_frags(NEXT, 0, fa0, fb0);
      if constexpr (!B_KC) issue_b(next, BUF);
      mfmas(fa1, fb1);
      interleave(std::integral_constant<int, PER_STAGE>{});
    };
    for (int k = 0; k < nk; k += NS) {
      stage(k, std::integral_constant<int, 0>{});
      static_for<1, NS>([&](auto ic) {
        if (k + decltype(ic)::value < nk) stage(k + decltype(ic)::value, ic);
      });
    }
  }
  wait_vm<0>();
  __syncthreads();
  cs.write(p, tile, reinterpret_cast<float*>(smem));
  // The lane once more, so that nothing of it is held through the loop for this.
  int last_lane = threadIdx.x & 63;
  asm volatile("" : "+v"(last_lane));
  write_tile<DT, LAYOUT, TM, TN>(p, tile, acc, m0 + wm, n0 + wn, last_lane,
                                 reinterpret_cast<float*>(smem) + wave * 16 * (16 * TN + 4));
}

// ------------------------------------------------------------------ few rows
// NN for single tokens: what counts is how fast the chosen experts' matrices are
// read.  A block takes 4 rows of an expert and 64 or 32 columns over the whole of K,
// so that few experts still give many loads: its 8 waves deal K among them in runs
// of KB rows of W, of which a lane holds 4 rows of one granule at a time, the next 4
// on their way, and multiplies them, in f32, by A's values from LDS.  The lanes'
// sums of a column are added by shuffles, the waves' in their order.
template <int DT, int BN>
__global__ __launch_bounds__(512, 4) void experts_few_kernel(ExpertArgs p) {
  constexpr int ES = DT == RT_F32 ? 4 : 2, EPG = 16 / ES, BM = 4, WAVES = 8;
  constexpr int R = 4, LPR = BN / EPG, KB = 64 / LPR * R;  // rows of W a lane, lanes a row, rows a wave and turn
  constexpr int KC = 2048;                          // A's columns in LDS at a time
  __shared__ __attribute__((aligned(16))) unsigned char xs[BM * KC * ES];
  __shared__ float part[WAVES][BM][BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Tile tile = tile_of<RT_NN, BM, BN>(p, lane);
  if (tile.expert < 0) return;
  const int rows = (int)min(tile.r1 - tile.m0, (long long)BM);
  const char* w = static_cast<const char*>(p.B) + (long long)tile.expert * p.K * p.N * ES;
  const int col = tile.n0 + (lane % LPR) * EPG, k_lane = (lane / LPR) * R;
  float acc[BM][EPG];
#pragma unroll
  for (int m = 0; m < BM; ++m)
#pragma unroll
    for (int e = 0; e < EPG; ++e) acc[m][e] = 0.0f;
  u4 v[R];
  auto load = [&](int k) {  // rows of W from k on; zeros past K
#pragma unroll
    for (int i = 0; i < R; ++i)
      v[i] = k + i < p.K && col < p.N ? granule<ES>(w, (long long)(k + i) * p.N + col, p.N - col) : u4{0, 0, 0, 0};
  };
  for (int k0 = 0; k0 < p.K; k0 += KC) {
    const int kc = min(KC, p.K - k0);
    int k = wave * KB;
    if (k < kc) load(k0 + k + k_lane);
    __syncthreads();
    for (int i = tid; i < BM * (KC / EPG); i += 64 * WAVES) {  // past K and the rows: zeros
      const int m = i / (KC / EPG), g = i % (KC / EPG) * EPG;
      u4 x = {0, 0, 0, 0};
      if (m < rows && g < kc) {
        const long long q = tile.m0 + m, row = p.order ? token_of(p, p.order[q]) : q;
        if (!p.order || row < p.a_rows) x = granule<ES>(p.A, row * p.K + k0 + g, kc - g);
      }
      *reinterpret_cast<u4*>(xs + (m * KC + g) * ES) = x;
    }
    __syncthreads();
    for (; k < kc; k += WAVES * KB) {
      u4 now[R];
#pragma unroll
      for (int i = 0; i < R; ++i) now[i] = v[i];
      if (k + WAVES * KB < kc) load(k0 + k + WAVES * KB + k_lane);
      float x[BM][R];
#pragma unroll
      for (int m = 0; m < BM; ++m)
#pragma unroll
        for (int i = 0; i < R; ++i) x[m][i] = rt_dev::load1<DT>(xs, m * KC + k + k_lane + i);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float b[8];
        const unsigned one[4] = {now[i][0], now[i][1], now[i][2], now[i][3]};
        if constexpr (ES == 2) rt_dev::load8<DT>(one, 0, 8, b);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] = __uint_as_float(one[e]);
#pragma unroll
        for (int m = 0; m < BM; ++m)
#pragma unroll
          for (int e = 0; e < EPG; ++e) acc[m][e] = fmaf(x[m][i], b[e], acc[m][e]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < BM; ++m)
#pragma unroll
    for (int e = 0; e < EPG; ++e) {
      float s = acc[m][e];
#pragma unroll
      for (int o = LPR; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
      if (lane < LPR) part[wave][m][lane * EPG + e] = s;
    }
  __syncthreads();
  const int m = tid / BN, c = tid % BN, n = tile.n0 + c;
  if (m >= rows || n >= p.N) return;  // rows is at most BM
  float s = part[0][m][c];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) s += part[i][m][c];
  if (p.bias) s += p.bias[(long long)tile.expert * p.N + n];
  if (p.epi == RT_EPI_BIAS_RELU) s = fmaxf(s, 0.0f);
  const long long at = (tile.m0 + m) * p.N + n;
  if (DT != RT_F32 && p.c_same) {
    if (p.mask && !(rt_dev::load1<DT>(p.mask, at) > 0.0f)) s = 0.0f;
    rt_dev::store1<DT>(p.C, at, s);
  } else {
    if (p.mask && !(static_cast<const float*>(p.mask)[at] > 0.0f)) s = 0.0f;
    static_cast<float*>(p.C)[at] = s;
  }
}

template <int DT, int LAYOUT, int BM, int BN, int WGM, int WGN>
hipError_t experts_regs(hipStream_t s, const ExpertArgs& p) {
  return experts_tiles<LAYOUT, BM, BN>(s, p, experts_kernel<DT, LAYOUT, BM, BN, WGM, WGN>, 64 * WGM * WGN);
}
template <int DT, int LAYOUT, int BM, int BN, int WGM, int WGN, int NS>
hipError_t experts_dma(hipStream_t s, const ExpertArgs& p) {
  return experts_tiles<LAYOUT, BM, BN>(s, p, experts_dma_kernel<DT, LAYOUT, BM, BN, WGM, WGN, NS>, 64 * WGM * WGN);
}

// Whether the direct-to-LDS kernel takes the operands: whole granules on 16
// bytes, and offsets from a tile's (TN: an expert's) first byte below 2^31.
template <int LAYOUT>
bool dma_ok(const ExpertArgs& p) {
  const long long lim = 1LL << 31, k = p.K, n = p.N;
  auto on16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  if (p.K % 8 != 0 || p.N % 8 != 0 || !on16(p.A) || !on16(p.B)) return false;
  if (p.order && p.a_rows * k * 2 >= lim) return false;
  if (LAYOUT == RT_TN) return p.n * std::max(k, n) * 2 < lim;
  return k * n * 2 < lim && std::max(k, n) <= 1 << 21;  // rows of a whole tile
}

// A's rows in the order of the experts, for the f32 kernel (gemm_f32.hip), which
// takes them one after the other: a pass of 8 bytes an element beside 12 N
// operations on it.
__global__ __launch_bounds__(256) void gather_kernel(ExpertArgs p, float* out, int tpr) {
  const int per = 256 / tpr, t = threadIdx.x & (tpr - 1);
  for (long long q = (long long)blockIdx.x * per + threadIdx.x / tpr; q < p.n; q += (long long)gridDim.x * per) {
    const long long row = token_of(p, p.order[q]);
    for (int c = 8 * t; c < p.K; c += 8 * tpr) {
      float v[8] = {};
      if (row < p.a_rows) rt_dev::load8<RT_F32>(p.A, row * p.K + c, p.K - c, v);
      rt_dev::store8<RT_F32>(out, q * p.K + c, p.K - c, v);
    }
  }
}

// TN operands of 16 bits whose rows are no whole granules, as the direct-to-LDS
// kernel takes them: A's rows in the order of the experts and B's, each padded to
// a_ld and b_ld elements.  Rows behind the last expert's are left alone.
struct PadArgs {
  ExpertArgs p;
  unsigned short *a, *b;
  int a_ld, b_ld;
  unsigned a_blocks;
};
__global__ __launch_bounds__(256) void pad_kernel(PadArgs t) {
  const ExpertArgs& p = t.p;
  const long long end = min((long long)p.offsets[p.experts], p.n);
  const bool first = blockIdx.x < t.a_blocks;
  const int cols = first ? p.K : p.N, ld = first ? t.a_ld : t.b_ld, lane = threadIdx.x & 63;
  const long long from = (first ? blockIdx.x : blockIdx.x - t.a_blocks) * 4LL + (threadIdx.x >> 6);
  const long long step = 4LL * (first ? t.a_blocks : gridDim.x - t.a_blocks);
  for (long long q = from; q < end; q += step) {  // a wave a row
    const long long row = first && p.order ? token_of(p, p.order[q]) : q;
    const bool there = row < (first ? p.a_rows : p.n);
    for (int c = 8 * lane; c < ld; c += 512)
      *reinterpret_cast<u4*>((first ? t.a : t.b) + q * ld + c) =
          there ? granule<2>(first ? p.A : p.B, row * cols + c, cols - c) : u4{0, 0, 0, 0};
  }
}

// Whether a TN product goes through padded copies: where it has rows enough for
// them, and work.  f16, us with copies and without, by multiply-adds: 2^29.9 (2
// experts 1003 x 333 over 3000 rows) 27.1 and 26.4, 2^30.0 (5 of 1003 x 777 over
// 1400) 25.1 and 23.8, 2^30.4 (over 1800) 27.4 and 27.9, 2^30.5 (1 of 1003 x 1001
// over 1500) 28.5 and 30.5, 2^30.7 (16 of 333 x 333 over 16000) 39.7 and 48.9,
// 2^31.0 (8 of 515 x 1027 over 4000) 31.5 and 37.4, 2^33.9 (8 of 1001 x 2003 over
// 8000) 81 and 153; of 128 rows an expert (64 of 513 x 1025 over 8192) 78 and 76.
bool pads(const ExpertArgs& p, int dtype) {
  if (dtype == RT_F32 || dma_ok<RT_TN>(p) || p.n / p.experts < 256) return false;
  return (double)p.n * p.K * p.N >= 0x1.4p30 && p.n * (std::max(p.K, p.N) + 7LL) * 2 < 1LL << 31;
}

// f32 products of many rows go to the split kernel of gemm_f32.hip, whose tiles
// are addressed by offsets below 2^31 over rows of at most 2^21 elements.
template <int LAYOUT>
bool split_takes(const ExpertArgs& p) {
  return p.n / p.experts > 32 && p.K <= 1 << 21 && p.N <= 1 << 21 && p.K > 0 && p.N > 0;
}

template <int DT, int LAYOUT>
hipError_t experts_launch(hipStream_t s, const ExpertArgs& args, float* rows) {
  ExpertArgs p = args;
  const long long mean = p.n / p.experts;
  if constexpr (DT == RT_F32) {
    if (split_takes<LAYOUT>(p)) {
      if (p.order) {
        int tpr = 1;
        while (tpr < 256 && 8 * tpr < p.K) tpr *= 2;
        rt::launch(gather_kernel, dim3((unsigned)std::min((p.n * tpr + 255) / 256, 8192LL)), dim3(256), 0, s, p, rows, tpr);
        if (hipError_t e = hipGetLastError()) return e;
        p.A = rows;
        p.a_rows = p.n;
        p.order = nullptr;
      }
      return rt::experts_f32_launch(s, LAYOUT, p);
    }
  }
  if constexpr (LAYOUT == RT_TN && DT != RT_F32) {
    if (pads(p, DT)) {
      PadArgs t{p, reinterpret_cast<unsigned short*>(rows), nullptr, (p.K + 7) & ~7, (p.N + 7) & ~7, 0};
      t.b = t.a + p.n * t.a_ld;
      t.a_blocks = (unsigned)std::min((p.n + 3) / 4, 4096LL);
      rt::launch(pad_kernel, dim3(2 * t.a_blocks), dim3(256), 0, s, t);
      if (hipError_t e = hipGetLastError()) return e;
      p.A = t.a;
      p.B = t.b;
      p.a_rows = p.n;
      p.order = nullptr;
      p.K = t.a_ld;
      p.N = t.b_ld;
    }
  }
  if constexpr (LAYOUT == RT_NN) {
    // Half types where the tiles of 32 x 64 below would leave the chip idle over a
    // long K (8 rows, K 4096, N 1024 bf16 18.3 us, 41.3 in tiles; K 1024, N 4096 15.9
    // and 15.3, of 32 rows 30.7 and 20.0), f32 always (16.9 and 80.4 for 2 rows, 47.8
    // and 81.3 for 64, K 1024, N 4096 47.9 and 51.5).
    const long long blocks = std::min<long long>(p.experts, p.n) * ((p.N + 63) / 64);
    if (p.n <= 64 && (DT == RT_F32 || (p.K >= 2048 && blocks <= 512))) {
      // Half the columns a block where that leaves no more than one a CU (K 4096, N 1024,
      // bf16 2 rows 14.8 us, 19.3 in 64 columns; 8 rows 18.3 and 20.3; 16 rows, 256
      // blocks of 64, 26.1 and 22.4; f32 16.9 and 24.0, 20.1 and 26.4, 31.9 and 30.4).
      if (blocks <= 128) return experts_tiles<RT_NN, 4, 32>(s, p, experts_few_kernel<DT, 32>, 512);
      return experts_tiles<RT_NN, 4, 64>(s, p, experts_few_kernel<DT, 64>, 512);
    }
  }
  if constexpr (LAYOUT != RT_TN) {
    if (mean <= 32) return experts_regs<DT, LAYOUT, 32, 64, 1, 4>(s, p);
  }
  if constexpr (DT != RT_F32) {
    // Tiles of C; an expert's rows leave half a tile over on average.
    auto tiles = [&](long long b) {
      const long long n = ((LAYOUT == RT_NT ? p.K : p.N) + b - 1) / b;
      return n * (LAYOUT == RT_TN ? (long long)p.experts * p.slices * ((p.K + b - 1) / b)
                                  : p.n / b + (std::min<long long>(p.experts, p.n) + 1) / 2);
    };
    if (dma_ok<LAYOUT>(p)) {
      // 256x256 tiles read least, and have a CU to themselves: where they fill
      // the chip, TN once (32 experts 2048 x 2048 over 32768 rows 387 us, 501 in
      // 128x128 tiles; 16 over 8192 140 and 182; 64 of 512 x 512 over 8192 27.4 and
      // 30.4; 8 of 1024 x 1024, 128 tiles, 36.5 and 28.7), the others twice and with
      // rows for most of a tile (the 32 experts NN 347 and 392, NT 324 and 362; 16 over
      // 8192, 320 tiles, 120 and 108).  Experts drawn with probabilities e^(g / 2), g
      // normal.
      if (LAYOUT == RT_TN ? tiles(256) >= 256 : tiles(256) >= 512 && mean >= 256)
        return experts_dma<DT, LAYOUT, 256, 256, 2, 4, 2>(s, p);
      // Where a 128x128 tile has a CU to itself, four stages (8 experts 1024 x
      // 1024 over 1024 rows NN 17.2 us, 18.7 in two; over 4096 34.2 and 26.3).
      if constexpr (LAYOUT != RT_TN) {
        if (tiles(128) <= 256) return experts_dma<DT, LAYOUT, 128, 128, 2, 2, 4>(s, p);
      }
      return experts_dma<DT, LAYOUT, 128, 128, 2, 2, 2>(s, p);
    }
    // Through registers smaller tiles, where few, keep more loads on their way (5
    // experts 1003 x 777 over 3000 rows NN 28.7 us, 46.0 in 128x128 tiles; 8 of
    // 1001 x 2003 over 8000 122 and 104), TN, which is short here, always (35.5 and 54.0).
    if constexpr (LAYOUT == RT_TN) {
      return experts_regs<DT, LAYOUT, 64, 64, 2, 2>(s, p);
    } else {
      if (tiles(128) <= 256) return experts_regs<DT, LAYOUT, 64, 64, 2, 2>(s, p);
      return experts_regs<DT, LAYOUT, 128, 128, 2, 2>(s, p);
    }
  } else {
    return experts_regs<DT, LAYOUT, 128, 128, 2, 2>(s, p);
  }
}

// Slices of the TN product's rows: where its tiles leave half the chip idle (f32:
// where they are one round of it or less, which experts with most of the rows
// would draw out) and every slice has 256 (512) rows or more.  8 experts 512 x 512
// over 32768 rows bf16 49 us, 101 in one slice; f32 156 and 196.
int tn_slices(const ExpertArgs& p, int dtype) {
  const bool f32 = dtype == RT_F32;
  const long long n = f32 ? 64 : 128, mean = p.n / p.experts;
  const long long tiles = p.experts * ((p.K + 127) / 128) * ((p.N + n - 1) / n);
  if (tiles > (f32 ? 256 : 192)) return 1;
  return (int)std::max(1LL, std::min({(f32 ? 1024 : 512) / tiles, mean / (f32 ? 512 : 256), 32LL}));
}

// The planes of a sliced TN product added up in their order: C in eights by the
// first blocks, the column sums by the others.
struct JoinArgs {
  const float *part, *cs_part;
  void* C;
  float* colsum;
  long long n, cs_n, blocks;
  int slices;
};
template <int OUT>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs p) {
  if ((long long)blockIdx.x < p.blocks) {
    for (long long i = 8 * ((long long)blockIdx.x * 256 + threadIdx.x); i < p.n; i += 8 * p.blocks * 256) {
      const int left = (int)min(p.n - i, 8LL);
      float v[8], w[8];
      rt_dev::load8<RT_F32>(p.part, i, left, v);
#pragma unroll 4
      for (int s = 1; s < p.slices; ++s) {
        rt_dev::load8<RT_F32>(p.part, s * p.n + i, left, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += w[e];
      }
      rt_dev::store8<OUT>(p.C, i, left, v);
    }
    return;
  }
  const long long i = ((long long)blockIdx.x - p.blocks) * 256 + threadIdx.x;
  if (i >= p.cs_n) return;
  float v = p.cs_part[i];
  for (int s = 1; s < p.slices; ++s) v += p.cs_part[s * p.cs_n + i];
  p.colsum[i] = v;
}

// ------------------------------------------------------------------ joining a token's rows
struct CombineArgs {
  const void* rows;
  const unsigned* rank;
  const float* weights;
  void* y;         // dy in the backward pass
  void* drows;
  float* dweights;
  long long n, tokens;
  int dim, k, tpr;
};

template <int R, int Y>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs p) {
  const int per = 256 / p.tpr;
  for (long long token = (long long)blockIdx.x * per + threadIdx.x / p.tpr; token < p.tokens;
       token += (long long)gridDim.x * per)
  for (int c = 8 * (threadIdx.x & (p.tpr - 1)); c < p.dim; c += 8 * p.tpr) {
    float y[8] = {};
    for (int j = 0; j < p.k; ++j) {
      const unsigned at = p.rank[token * p.k + j];
      if (at >= p.n) continue;  // a choice without a row
      const float w = p.weights ? p.weights[token * p.k + j] : 1.0f;
      float v[8];
      rt_dev::load8<R>(p.rows, (long long)at * p.dim + c, p.dim - c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(w, v[e], y[e]);
    }
    rt_dev::store8<Y>(p.y, token * p.dim + c, p.dim - c, y);
  }
}

// A wave a token: drows[rank] = w dy, dweights = <dy, rows[rank]>.
template <int R, int Y>
__global__ __launch_bounds__(256) void combine_grad_kernel(CombineArgs p) {
  const int lane = threadIdx.x & 63;
  for (long long token = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); token < p.tokens; token += (long long)gridDim.x * 4)
  for (int j = 0; j < p.k; ++j) {
    const unsigned at = p.rank[token * p.k + j];
    const bool on = at < p.n;
    const float w = p.weights ? p.weights[token * p.k + j] : 1.0f;
    float dot = 0.0f;
    if (on) {
      for (int c = 8 * lane; c < p.dim; c += 512) {
        float d[8], v[8];
        rt_dev::load8<Y>(p.y, token * p.dim + c, p.dim - c, d);
        if (p.dweights) {
          rt_dev::load8<R>(p.rows, (long long)at * p.dim + c, p.dim - c, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = fmaf(d[e], v[e], dot);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = w * d[e];
        rt_dev::store8<R>(p.drows, (long long)at * p.dim + c, p.dim - c, v);
      }
    }
    if (p.dweights) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
      if (lane == 0) p.dweights[token * p.k + j] = dot;
    }
  }
}

int check_combine(rt_ctx* c, const rt_buf* rows, const rt_buf* rank, const rt_buf* weights, const rt_buf* y, CombineArgs* p) {
  if (rows->rank != 2 || rank->rank != 2 || y->rank != 2)
    return rt::fail(c, RT_ERR_SHAPE, "combine: rows [n, columns], rank [tokens, k], y [tokens, columns]");
  if (!rt::is_float(rows->dtype) || !rt::is_float(y->dtype)) return rt::fail(c, RT_ERR_DTYPE, "combine: f32, bf16 or f16");
  if (rank->dtype != RT_U32) return rt::fail(c, RT_ERR_DTYPE, "combine: rank is u32");
  if (y->shape[0] != rank->shape[0] || y->shape[1] != rows->shape[1])
    return rt::fail(c, RT_ERR_SHAPE, "combine: y must be [%zu,%zu]", rank->shape[0], rows->shape[1]);
  if (weights && (weights->dtype != RT_F32 || weights->n != rank->n))
    return rt::fail(c, RT_ERR_SHAPE, "combine: weights must be f32, %zu elements", rank->n);
  const size_t lim = size_t(1) << 30;
  if (rows->shape[0] > lim || rank->n > lim || y->shape[0] > lim || rows->shape[1] > (size_t(1) << 24))
    return rt::fail(c, RT_ERR_SHAPE, "combine: at most 2^30 rows of 2^24 columns");
  p->rows = rows->ptr;
  p->rank = static_cast<const unsigned*>(rank->ptr);
  p->weights = weights ? static_cast<const float*>(weights->ptr) : nullptr;
  p->y = y->ptr;
  p->n = (long long)rows->shape[0];
  p->tokens = (long long)y->shape[0];
  p->dim = (int)y->shape[1];
  p->k = (int)rank->shape[1];
  p->tpr = 1;
  while (p->tpr < 256 && 8 * p->tpr < p->dim) p->tpr *= 2;
  return RT_OK;
}

}  // namespace

using namespace rt;

extern "C" {

int rt_experts_gemm(rt_ctx* c, rt_layout layout, const rt_buf* a, const rt_buf* b, rt_buf* out, const rt_buf* offsets,
                    const rt_buf* order, rt_epilogue epi, const rt_buf* aux, rt_buf* colsum) {
  CHECK_CTX(c);
  if (!a || !b || !out || !offsets) return fail(c, RT_ERR_INVALID, "null buffer");
  if (layout != RT_NN && layout != RT_NT && layout != RT_TN) return fail(c, RT_ERR_INVALID, "unknown layout %d", (int)layout);
  const bool tn = layout == RT_TN;
  const rt_buf* w = tn ? out : b;    // [experts, K, N]
  const rt_buf* r = tn ? b : out;    // rows in the order of the experts
  if (a->rank != 2 || w->rank != 3 || r->rank != 2)
    return fail(c, RT_ERR_SHAPE, "experts: rows are rank 2, the experts' matrices [experts, K, N]");
  const size_t E = w->shape[0], K = w->shape[1], N = w->shape[2], n = r->shape[0];
  if (E < 1 || E > (size_t)kMaxExperts) return fail(c, RT_ERR_SHAPE, "experts: between 1 and %d", kMaxExperts);
  if (K > (size_t(1) << 24) || N > (size_t(1) << 24) || n > (size_t(1) << 29) || a->shape[0] > (size_t(1) << 29))
    return fail(c, RT_ERR_SHAPE, "experts: at most 2^29 rows, matrices of at most 2^24 a side");
  if (a->shape[1] != (layout == RT_NT ? N : K) || r->shape[1] != (layout == RT_NT ? K : N))
    return fail(c, RT_ERR_SHAPE, "experts: rows of %zu and %zu with matrices [%zu,%zu] (layout %d)", a->shape[1], r->shape[1], K,
                N, (int)layout);
  if (!is_float(a->dtype) || a->dtype != b->dtype) return fail(c, RT_ERR_DTYPE, "experts: A and B share f32, bf16 or f16");
  if (out->dtype != RT_F32 && out->dtype != a->dtype) return fail(c, RT_ERR_DTYPE, "experts: C is f32 or of the operands' type");
  if (offsets->dtype != RT_U32 || offsets->n != E + 1) return fail(c, RT_ERR_SHAPE, "experts: offsets must be u32 [%zu]", E + 1);
  ExpertArgs p{};
  if (order) {
    if (layout == RT_NT) return fail(c, RT_ERR_INVALID, "experts: the NT layout takes A's rows in the order of the experts");
    if (order->dtype != RT_U32 || order->n != n) return fail(c, RT_ERR_SHAPE, "experts: order must be u32 [%zu]", n);
    const size_t t = a->shape[0];
    if (t == 0 ? n != 0 : n % t != 0) return fail(c, RT_ERR_SHAPE, "experts: %zu rows of %zu tokens", n, t);
    p.order = static_cast<const unsigned*>(order->ptr);
    // With l the bits of k - 1, ceil(2^(31 + l) / k) divides every number below
    // 2^31 exactly (the error of the quotient stays below 1 / k), in 32 bits.
    const unsigned long long k = t && n ? n / t : 1;
    int l = 0;
    while ((1ull << l) < k) ++l;
    p.per_mul = (unsigned)(((1ull << (31 + l)) + k - 1) / k);
    p.per_shift = 31 + l;
  } else if (a->shape[0] != n) {
    return fail(c, RT_ERR_SHAPE, "experts: A has %zu rows, not %zu", a->shape[0], n);
  }
  if (epi == RT_EPI_BIAS || epi == RT_EPI_BIAS_RELU) {
    if (layout != RT_NN) return fail(c, RT_ERR_INVALID, "experts: a bias goes with the NN layout");
    if (!aux || aux->dtype != RT_F32 || aux->n != E * N) return fail(c, RT_ERR_SHAPE, "experts: the bias must be f32 [%zu,%zu]", E, N);
    p.bias = static_cast<const float*>(aux->ptr);
  } else if (epi == RT_EPI_RELU_MASK) {
    if (tn) return fail(c, RT_ERR_INVALID, "experts: the TN layout has no epilogue");
    if (!aux || aux->dtype != out->dtype || aux->n != out->n)
      return fail(c, RT_ERR_SHAPE, "experts: the mask must match C in type and size");
    p.mask = aux->ptr;
  } else if (epi != RT_EPI_NONE) {
    return fail(c, RT_ERR_INVALID, "unknown epilogue %d", (int)epi);
  }
  if (colsum) {
    if (!tn) return fail(c, RT_ERR_INVALID, "fused colsum is only for the TN layout");
    if (colsum->dtype != RT_F32 || colsum->n != E * N) return fail(c, RT_ERR_SHAPE, "experts: colsum must be f32 [%zu,%zu]", E, N);
    p.colsum = static_cast<float*>(colsum->ptr);
  }
  if (out->n == 0 && !(colsum && colsum->n)) return RT_OK;
  if (tn && K == 0) return fail(c, RT_ERR_SHAPE, "experts: column sums alone");
  p.A = a->ptr;
  p.B = b->ptr;
  p.C = out->ptr;
  p.offsets = static_cast<const unsigned*>(offsets->ptr);
  p.n = (long long)n;
  p.a_rows = (long long)a->shape[0];
  p.experts = (int)E;
  p.K = p.c_K = (int)K;
  p.N = p.c_N = (int)N;
  p.epi = epi;
  p.c_same = out->dtype == a->dtype;
  // Scratch: f32's gathered rows or padded ones of 16 bits, then the planes of a sliced
  // TN product.
  const size_t gathered = a->dtype == RT_F32 ? (order && split_takes<RT_NN>(p) ? (n * K + 3) & ~size_t(3) : 0)
                          : tn && pads(p, a->dtype) ? n * (((K + 7) & ~size_t(7)) + ((N + 7) & ~size_t(7))) / 2 : 0;
  p.slices = tn ? tn_slices(p, a->dtype) : 1;
  const size_t planes = p.slices > 1 ? p.slices * E * (K * N + (colsum ? N : 0)) : 0;
  if (int rc = ensure_scratch(c, gathered + planes)) return rc;
  JoinArgs j{};
  if (p.slices > 1) {
    j.part = c->scratch + gathered;
    j.cs_part = j.part + p.slices * E * K * N;
    j.C = p.C;
    j.colsum = p.colsum;
    j.n = (long long)(E * K * N);
    j.cs_n = colsum ? (long long)(E * N) : 0;
    j.blocks = std::min((j.n + 2047) / 2048, 4096LL);
    j.slices = p.slices;
    p.C = const_cast<float*>(j.part);
    if (colsum) p.colsum = const_cast<float*>(j.cs_part);
    p.c_same = 0;
  }
  Launch L(c, layout == RT_NN ? "experts_nn" : tn ? "experts_tn" : "experts_nt");
  HIP_TRY(c, for_float(a->dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            return layout == RT_NN ? experts_launch<DT, RT_NN>(c->stream, p, c->scratch)
                   : tn            ? experts_launch<DT, RT_TN>(c->stream, p, c->scratch)
                                   : experts_launch<DT, RT_NT>(c->stream, p, c->scratch);
          }),
          "experts gemm");
  if (p.slices > 1) {
    HIP_TRY(c, for_float(out->dtype, [&](auto o) {
              launch(join_kernel<decltype(o)::value>, dim3((unsigned)(j.blocks + (j.cs_n + 255) / 256)), dim3(256), 0,
                     c->stream, j);
              return hipGetLastError();
            }),
            "experts gemm join");
  }
  return RT_OK;
}

int rt_combine(rt_ctx* c, const rt_buf* rows, const rt_buf* rank, const rt_buf* weights, rt_buf* y) {
  CHECK_CTX(c);
  if (!rows || !rank || !y) return fail(c, RT_ERR_INVALID, "null buffer");
  CombineArgs p{};
  if (int rc = check_combine(c, rows, rank, weights, y, &p)) return rc;
  if (y->n == 0) return RT_OK;
  Launch L(c, "combine");
  HIP_TRY(c, for_float(rows->dtype, [&](auto r) {
            return for_float(y->dtype, [&](auto t) {
              launch(combine_kernel<decltype(r)::value, decltype(t)::value>,
                     dim3(grid_of((p.tokens * p.tpr + 255) / 256)), dim3(256), 0, c->stream, p);
              return hipGetLastError();
            });
          }),
          "combine");
  return RT_OK;
}

int rt_combine_backward(rt_ctx* c, const rt_buf* dy, const rt_buf* rows, const rt_buf* rank, const rt_buf* weights,
                        rt_buf* drows, rt_buf* dweights) {
  CHECK_CTX(c);
  if (!dy || !rank || !drows) return fail(c, RT_ERR_INVALID, "null buffer");
  CombineArgs p{};
  if (int rc = check_combine(c, drows, rank, weights, dy, &p)) return rc;
  if (dweights) {
    if (!rows) return fail(c, RT_ERR_INVALID, "combine backward: the gradient of the weights needs the rows");
    if (rows->dtype != drows->dtype || rows->rank != 2 || rows->shape[0] != drows->shape[0] || rows->shape[1] != drows->shape[1])
      return fail(c, RT_ERR_SHAPE, "combine backward: rows and drows must match in type and shape");
    if (dweights->dtype != RT_F32 || dweights->n != rank->n)
      return fail(c, RT_ERR_SHAPE, "combine backward: dweights must be f32, %zu elements", rank->n);
    p.dweights = static_cast<float*>(dweights->ptr);
    p.rows = rows->ptr;
  }
  p.drows = drows->ptr;
  if (rank->n == 0) return RT_OK;
  Launch L(c, "combine_bwd");
  HIP_TRY(c, for_float(drows->dtype, [&](auto r) {
            return for_float(dy->dtype, [&](auto t) {
              launch(combine_grad_kernel<decltype(r)::value, decltype(t)::value>, dim3(grid_of((p.tokens + 3) / 4)),
                     dim3(256), 0, c->stream, p);
              return hipGetLastError();
            });
          }),
          "combine backward");
  return RT_OK;
}

}  // extern "C"

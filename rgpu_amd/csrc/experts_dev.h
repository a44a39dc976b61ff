// What the kernels of the experts' products share (experts.hip, and
// gemm_f32.hip for f32): their arguments, and how a block finds its tile.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "rt_internal.h"

namespace rt {

struct ExpertArgs {
  const void* A;
  const void* B;
  void* C;
  const unsigned* offsets;
  const unsigned* order;  // null: A's rows are in the order of the experts
  const float* bias;
  const void* mask;
  float* colsum;
  long long n, a_rows;    // rows in the order of the experts; rows of A
  unsigned per_mul;       // order[p] / k = order[p] * per_mul >> per_shift
  int per_shift;
  int experts;
  int K, N;               // W is [experts, K, N]
  int c_K, c_N;           // experts.hip: C's and the aux operands' K and N (K and N are those of padded copies)
  int epi;
  int c_same;             // C is of the operands' type, else f32
  // TN: each expert's rows in so many slices, whose sums are planes [slices]
  // of C and of the column sums (joined by a launch of experts.hip).
  int slices;
  int vec_c;              // f32: C's rows, the bias's and the mask's are on 16 bytes
};

__device__ inline unsigned token_of(const ExpertArgs& p, unsigned choice) {
  return (unsigned)(((unsigned long long)choice * p.per_mul) >> p.per_shift);
}

// gemm_f32.hip: f32 products over rows that are in the order of the experts, K and
// N above 0 and at most 2^21.
hipError_t experts_f32_launch(hipStream_t s, int layout, ExpertArgs p);

}  // namespace rt

namespace rt_dev {

using rt::ExpertArgs;
using rt::token_of;

// The tile of C that a block computes: its expert (-1: none), the expert's
// rows, and the first row (NN, NT: among all rows; TN: of the matrix) and column.
struct Tile {
  int expert;
  int plane;  // of C and the column sums, each [experts, ..]: expert, or slice * experts + expert
  long long r0, r1, m0;
  int n0;
};

__device__ inline void expert_rows(const ExpertArgs& p, int e, long long& r0, long long& r1) {
  r0 = min((long long)p.offsets[e], p.n);
  r1 = max(r0, min((long long)p.offsets[e + 1], p.n));
}

// Consecutive blocks go to the 8 XCDs in turn.  Tiles are ordered in bands of 8
// tiles of rows by all columns, and dealt to the XCDs in runs, so blocks that read
// the same matrix and rows share an L2: NN and NT in one run an XCD; TN, whose
// tiles cost as much as their expert has rows, in runs of 8 (32 experts 2048 x 2048
// drawn with probabilities e^(g / 2), g normal, 32768 rows: 461 us in eight runs, 387
// this way; 16 over 8192 rows 191 and 140).  How many tiles of rows there are
// only the offsets say: each wave adds them up, 64 experts a turn.
constexpr int BAND = 8;
template <int LAYOUT, int BM, int BN>
__device__ inline Tile tile_of(const ExpertArgs& p, int lane) {
  const int tiles_n = ((LAYOUT == RT_NT ? p.K : p.N) + BN - 1) / BN;
  Tile o{-1, 0, 0, 0, 0, 0};
  int total, each = 0;  // tiles of rows: of all experts, of one (TN)
  auto tiles = [&](int e, long long& r0, long long& r1) -> int {
    r0 = r1 = 0;
    if (e < p.experts) expert_rows(p, e, r0, r1);
    return (int)((r1 - r0 + BM - 1) / BM);
  };
  auto scan = [&](int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int w = __shfl_up(v, d, 64);
      if (lane >= d) v += w;
    }
    return v;
  };
  if constexpr (LAYOUT == RT_TN) {
    each = (p.K + BM - 1) / BM;
    total = p.experts * p.slices * each;
  } else {
    total = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
      long long r0, r1;
      total += __builtin_amdgcn_readlane(scan(tiles(e0 + lane, r0, r1)), 63);
    }
  }
  const long long all = (long long)total * tiles_n, j = blockIdx.x >> 3;
  long long t;
  if constexpr (LAYOUT == RT_TN) {
    t = (j / BAND * 8 + (blockIdx.x & 7)) * BAND + j % BAND;
    if (t >= all) return o;
  } else {
    const long long per = (all + 7) / 8;
    t = (blockIdx.x & 7) * per + j;
    if (j >= per || t >= all) return o;
  }
  const long long band = (long long)BAND * tiles_n, b = t / band, in = t - b * band;
  const int first = (int)b * BAND, rows = min(total - first, BAND);
  int m = first + (int)(in % rows);
  o.n0 = (int)(in / rows) * BN;
  if constexpr (LAYOUT == RT_TN) {
    const int part = m / each, slice = part % p.slices;
    o.expert = part / p.slices;
    o.plane = slice * p.experts + o.expert;
    o.m0 = (long long)(m % each) * BM;
    expert_rows(p, o.expert, o.r0, o.r1);
    if (p.slices > 1) {
      const long long rows = ((o.r1 - o.r0 + p.slices - 1) / p.slices + 63) / 64 * 64;
      o.r0 = min(o.r0 + slice * rows, o.r1);
      o.r1 = min(o.r0 + rows, o.r1);
    }
    o.r0 = (unsigned)__builtin_amdgcn_readfirstlane((int)o.r0);  // rows are counted below 2^31
    o.r1 = (unsigned)__builtin_amdgcn_readfirstlane((int)o.r1);
  } else {
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
      long long r0, r1;
      const int mine = tiles(e0 + lane, r0, r1), s = scan(mine);
      const unsigned long long past = __ballot(s > m);
      if (past) {
        const int l = __builtin_ctzll(past);
        o.expert = o.plane = __builtin_amdgcn_readfirstlane(e0 + l);
        o.r0 = (unsigned)__builtin_amdgcn_readlane((int)r0, l);  // rows are counted below 2^31
        o.r1 = (unsigned)__builtin_amdgcn_readlane((int)r1, l);
        o.m0 = o.r0 + (long long)(m - __builtin_amdgcn_readlane(s - mine, l)) * BM;
        break;
      }
      m -= __builtin_amdgcn_readlane(s, 63);
    }
  }
  return o;
}

// As many blocks as tiles that the rows can have, in whole runs.
template <int LAYOUT, int BM, int BN, class K>
hipError_t experts_tiles(hipStream_t s, const ExpertArgs& p, K kernel, int threads) {
  const long long tiles_n = ((LAYOUT == RT_NT ? p.K : p.N) + BN - 1) / BN;
  const long long tiles_m = LAYOUT == RT_TN ? (long long)p.experts * p.slices * ((p.K + BM - 1) / BM)
                                            : p.n / BM + std::min<long long>(p.experts, p.n);
  const long long run = LAYOUT == RT_TN ? 8 * BAND : 8, blocks = (tiles_m * tiles_n + run - 1) / run * run;
  if (blocks * threads > 0xffffffffLL) return hipErrorInvalidValue;  // a grid's threads are counted in 32 bits
  rt::launch(kernel, dim3((unsigned)blocks), dim3(threads), 0, s, p);
  return hipGetLastError();
}
}  // namespace rt_dev

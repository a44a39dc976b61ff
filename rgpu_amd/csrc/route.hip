// Routing of tokens to experts, and its gradient.
//
// Scores s_e = softmax or sigmoid of a token's logits; the choice goes by
// c_e = s_e + bias_e among the experts of the kept groups (a group's rank is the
// sum of its two greatest c); the k greatest c are chosen, the lowest index of
// equal ones first; weights are the chosen s, over their sum if renormalised,
// times a scale.  c decides by comparison, and two experts' c are often next to
// each other, so s and c are held in 64 bits: in 32, about one token in ten
// thousand would go by the rounding of its exponentials.
//
// A group of LANES lanes takes a token, VPL experts a lane, expert VPL-major
// (coalesced), and meets in DPP rotations.  route_exact has every c as a 64-bit
// whole number of the same order and takes their maximum k times.  That costs an
// exponential and a division in 64 bits an expert: 16384 tokens of 256 experts
// (16.8 MB of logits, 4 us at a copy's rate) 36 us.  So route_fast chooses in
// 32 bits first: whatever comes within the error of its arithmetic of the k-th
// greatest c is a candidate, and only the candidates, a lane each, are computed in
// 64 bits and ranked.  Where it cannot tell (more candidates than lanes, groups
// that close, NaN) the wave goes through route_exact.  17 us; 25 with a bias and 4
// of 8 groups kept.  Both are bound by vector instructions, of two waves a SIMD:
// route_exact's registers count in route_kernel too (216 at 16 experts a lane).

#include <cmath>
#include <type_traits>

#include "device_util.h"
#include "elems.h"
#include "rt_internal.h"

namespace {

constexpr int kMaxExperts = 1024, kMaxChoices = 64, kMaxGroups = 64;

struct RouteArgs {
  const void* logits;
  const float* bias;
  unsigned* ids;
  float* weights;
  const float* dweights;
  void* dlogits;
  long long tokens;
  int experts, k, groups, kept, sigmoid, renorm, fast;
  int per;           // experts a group
  unsigned per_mul;  // e / per = e * per_mul >> 32 for e below 2^10, per above 1
  float scale;
};

// A double as a whole number of the same order, above 1 for every value; a NaN
// is 1, below them all.  0 stands for an expert that is out.
__device__ inline unsigned long long order_key(double c) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(c);
  if (c != c) return 1;
  return (u >> 63) ? ~u : u | (1ull << 63);
}

template <int CTRL>
__device__ inline unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

// f over the lanes of a group of LANES (16: a DPP row; 64: the wave), the
// result in every lane.  step(o) gives a lane another's value, at distance o.
template <int LANES, class F>
__device__ inline void over_lanes(F&& f) {
  f([](unsigned v) { return dpp<0x128>(v); });  // row_ror:8
  f([](unsigned v) { return dpp<0x124>(v); });
  f([](unsigned v) { return dpp<0x122>(v); });
  f([](unsigned v) { return dpp<0x121>(v); });
  if constexpr (LANES == 64) {
    f([](unsigned v) { return (unsigned)__shfl_xor((int)v, 16, 64); });
    f([](unsigned v) { return (unsigned)__shfl_xor((int)v, 32, 64); });
  }
}

template <class F>
__device__ inline double of_lane(double v, F&& from) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v);
  return __longlong_as_double((long long)(((unsigned long long)from((unsigned)(u >> 32)) << 32) | from((unsigned)u)));
}
template <int LANES>
__device__ inline double lanes_sum(double v) {
  over_lanes<LANES>([&](auto from) { v += of_lane(v, from); });
  return v;
}
template <int LANES>
__device__ inline float lanes_sum(float v) {
  over_lanes<LANES>([&](auto from) { v += __uint_as_float(from(__float_as_uint(v))); });
  return v;
}
template <int LANES>
__device__ inline float lanes_max(float v) {
  over_lanes<LANES>([&](auto from) { v = fmaxf(v, __uint_as_float(from(__float_as_uint(v)))); });
  return v;
}

__device__ inline double sigmoid64(double x) { return 1.0 / (1.0 + exp(-x)); }

// Divided before it is scaled: the reciprocal of a sum below 2^-1024 is infinite.
__device__ inline float weight_of(const RouteArgs& p, double score, double sum) {
  const double w = !p.renorm ? score : sum == 0.0 ? 0.0 : score / sum;
  return (float)(w * (double)p.scale);
}

// A token's LDS: its group's c (kept groups only) and its choices.
template <int LANES, int VPL>
struct RouteRow {
  double c[LANES * VPL];
  unsigned chosen[kMaxChoices];
};

template <int DT, int LANES, int VPL>
__device__ void route_exact(const RouteArgs& p, long long token, int lane, RouteRow<LANES, VPL>& lds) {
  const long long row = min(token, p.tokens - 1) * p.experts;  // lanes past the end repeat the last token
  const int E = p.experts;

  float x[VPL];
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = v * LANES + lane;
    x[v] = e < E ? rt_dev::load1<DT>(p.logits, row + e) : -INFINITY;
    top = fmaxf(top, x[v]);
  }
  top = lanes_max<LANES>(top);
  if (top == -INFINITY) top = 0.0f;
  double c[VPL], total = 0.0;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    c[v] = p.sigmoid ? sigmoid64((double)x[v]) : exp((double)x[v] - (double)top);
    total += c[v];
  }
  total = p.sigmoid ? 1.0 : lanes_sum<LANES>(total);
  if (total == 0.0) total = 1.0;
  unsigned long long key[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = v * LANES + lane;
    c[v] /= total;
    if (p.bias && e < E) c[v] += (double)p.bias[e];
    key[v] = e < E ? order_key(c[v]) : 0;
  }
  if (p.kept < p.groups) {
    // Each lane ranks every LANES-th group, starting at another expert of it
    // than its neighbours (banks).
    const int per = E / p.groups;
#pragma unroll
    for (int v = 0; v < VPL; ++v) lds.c[v * LANES + lane] = c[v];
    rt_dev::wave_lds_order();
    unsigned long long mine[kMaxGroups / LANES], on = 0;
#pragma unroll
    for (int t = 0; t < kMaxGroups / LANES; ++t) {
      const int g = t * LANES + lane;
      mine[t] = 0;
      if (g < p.groups) {
        unsigned long long a = 0, b = 0;
        double va = 0.0, vb = 0.0;
        int j = g % per;
        for (int i = 0; i < per; ++i) {
          const double v = lds.c[g * per + j];
          const unsigned long long u = order_key(v);
          if (u > a) b = a, vb = va, a = u, va = v;
          else if (u > b) b = u, vb = v;
          j = j + 1 == per ? 0 : j + 1;
        }
        mine[t] = order_key(per > 1 ? va + vb : va);
      }
    }
    // The kept best groups, the first of equal ones: taken one by one.
    for (int r = 0; r < p.kept; ++r) {
      unsigned long long best = 0;
      unsigned at = 0;
#pragma unroll
      for (int t = 0; t < kMaxGroups / LANES; ++t)
        if (mine[t] > best) best = mine[t], at = t * LANES + lane;
      over_lanes<LANES>([&](auto from) {
        const unsigned long long o = ((unsigned long long)from((unsigned)(best >> 32)) << 32) | from((unsigned)best);
        const unsigned oa = from(at);
        if (o > best || (o == best && oa < at)) best = o, at = oa;
      });
      on |= 1ull << at;
#pragma unroll
      for (int t = 0; t < kMaxGroups / LANES; ++t)
        if ((unsigned)(t * LANES + lane) == at) mine[t] = 0;
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int e = v * LANES + lane;
      if (e < E && !((on >> (e / per)) & 1)) key[v] = 0;
    }
  }
  for (int r = 0; r < p.k; ++r) {
    unsigned long long best = 0;
    unsigned at = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (key[v] > best) best = key[v], at = v * LANES + lane;
    over_lanes<LANES>([&](auto from) {
      const unsigned long long o = ((unsigned long long)from((unsigned)(best >> 32)) << 32) | from((unsigned)best);
      const unsigned oa = from(at);
      if (o > best || (o == best && oa < at)) best = o, at = oa;
    });
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if ((unsigned)(v * LANES + lane) == at) key[v] = 0;
    if (lane == 0) lds.chosen[r] = at;
  }
  rt_dev::wave_lds_order();
  double s[kMaxChoices / LANES], sum = 0.0;
#pragma unroll
  for (int t = 0; t < kMaxChoices / LANES; ++t) {
    const int j = t * LANES + lane;
    s[t] = 0.0;
    if (j < p.k) {
      const double z = (double)rt_dev::load1<DT>(p.logits, row + lds.chosen[j]);
      s[t] = p.sigmoid ? sigmoid64(z) : exp(z - (double)top) / total;
    }
    sum += s[t];
  }
  sum = lanes_sum<LANES>(sum);
#pragma unroll
  for (int t = 0; t < kMaxChoices / LANES; ++t) {
    const int j = t * LANES + lane;
    if (j < p.k && token < p.tokens) {
      p.ids[token * p.k + j] = lds.chosen[j];
      p.weights[token * p.k + j] = weight_of(p, s[t], sum);
    }
  }
}

// Sets `slow` where the choice could not be told in 32 bits; otherwise the token
// is done.  For sigmoid scores, and for softmax without a bias and renormalised,
// whose sum over all experts then cancels (scores are the exponentials).
template <int DT, int VPL>
__device__ bool route_fast(const RouteArgs& p, long long token, int lane, RouteRow<16, VPL>& lds) {
  constexpr int LANES = 16;
  const long long row = min(token, p.tokens - 1) * p.experts;
  const int E = p.experts;
  float* const cf = reinterpret_cast<float*>(lds.c);
  float c[VPL], top = -INFINITY;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = v * LANES + lane;
    c[v] = e < E ? rt_dev::load1<DT>(p.logits, row + e) : -INFINITY;
    top = fmaxf(top, c[v]);
  }
  top = lanes_max<LANES>(top);
  bool slow = !(fabsf(top) < INFINITY);
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = v * LANES + lane;
    const float power = __builtin_amdgcn_exp2f((p.sigmoid ? -c[v] : c[v] - top) * 0x1.715476p+0f);
    c[v] = p.sigmoid ? __builtin_amdgcn_rcpf(1.0f + power) : power;
    if (p.bias && e < E) c[v] += p.bias[e];
    slow |= c[v] != c[v];
    if (e >= E) c[v] = -INFINITY;
  }
  // Scores are at most 1 and off by less than 2^-22, c by half a step of it more:
  // values further apart than `far` are in the order of their exact ones.  (The
  // power 2^(a log2 e) has a relative error of 2^-23 of its own and |a| 2^-24 for
  // each rounding of its exponent: the constant's, the product's and, of softmax, the
  // difference's.  That is at most (1.5 |a| + 1) e^a 2^-23 < 1.1 2^-23 for e^a, a <= 0.
  // A sigmoid has s (1 - s) (|a| + 1) 2^-23 < 0.5 2^-23 of it, 2^-24 of the sum and
  // 2^-23 of the reciprocal.)
  auto far = [](float v) { return 0x1p-20f + 0x1p-22f * fabsf(v); };
  if (p.kept < p.groups) {
    // The two greatest of each group, lane g the g-th's.
    float a = -INFINITY, b = -INFINITY;
    auto merge = [](auto& a, auto& b, auto oa, auto ob) {
      b = max(min(a, oa), max(b, ob));
      a = max(a, oa);
    };
    if (p.per % LANES == 0) {  // a group is whole turns of the lanes
      float ta = -INFINITY, tb = -INFINITY;
      int group = 0, left = p.per / LANES;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        merge(ta, tb, c[v], -INFINITY);
        if (--left == 0) {
          over_lanes<LANES>([&](auto from) {
            merge(ta, tb, __uint_as_float(from(__float_as_uint(ta))), __uint_as_float(from(__float_as_uint(tb))));
          });
          if (lane == group) a = ta, b = tb;
          ta = tb = -INFINITY;
          left = p.per / LANES;
          ++group;
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v) cf[v * LANES + lane] = c[v];
      rt_dev::wave_lds_order();
      if (lane < p.groups) {
        int j = lane % p.per;  // another bank than the neighbour's
#pragma unroll 4
        for (int i = 0; i < p.per; ++i) {
          merge(a, b, cf[lane * p.per + j], -INFINITY);
          j = j + 1 == p.per ? 0 : j + 1;
        }
      }
    }
    const bool some = lane < p.groups;
    const float rank = some ? a + b : -INFINITY;
    // Sums of two, so off by twice as much.
    const float apart = 2.0f * far(lanes_max<LANES>(some ? fabsf(a) + fabsf(b) : 0.0f));
    int before = 0;  // groups that come before this lane's
    rt_dev::static_for<1, LANES>([&](auto oc) {
      constexpr int CTRL = 0x120 + decltype(oc)::value;  // row_ror: from the lane that many before
      const float o = __uint_as_float(dpp<CTRL>(__float_as_uint(rank)));
      before += o > rank || (o == rank && ((lane - decltype(oc)::value) & (LANES - 1)) < lane);
    });
    bool keep = before < p.kept;
    const float worst = -lanes_max<LANES>(keep ? -rank : -INFINITY), best = lanes_max<LANES>(keep ? -INFINITY : rank);
    // Groups that close to the border are ranked in 64 bits: 16384 tokens nearly
    // always hold some, and the launch waits for their wave (through route_exact 6 us
    // longer than with every group in 64 bits here, 26.5; with those groups alone 24.9).
    const bool close = !(worst - best > apart);
    slow |= rank != rank;  // a group of both infinities, by its bias
    if (p.per % LANES != 0) {
      slow |= close;
    } else if (__any(close)) {
      const bool open = some && !(rank - best > apart) && !(worst - rank > apart);
      const unsigned open_row = (unsigned)(__ballot(open) >> (threadIdx.x & 48));
      double da = -INFINITY, db = -INFINITY, ta = -INFINITY, tb = -INFINITY;
      int group = 0, left = p.per / LANES;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        if (v * LANES >= E) break;  // whole turns: E is a multiple of LANES
        if (__any((open_row >> group) & 1)) {
          const double z = (double)rt_dev::load1<DT>(p.logits, row + v * LANES + lane);
          const double s = p.sigmoid ? sigmoid64(z) : exp(z - (double)top);
          merge(ta, tb, p.bias ? s + (double)p.bias[v * LANES + lane] : s, -(double)INFINITY);
        }
        if (--left == 0) {
          over_lanes<LANES>([&](auto from) { merge(ta, tb, of_lane(ta, from), of_lane(tb, from)); });
          if (lane == group) da = ta, db = tb;
          ta = tb = -INFINITY;
          left = p.per / LANES;
          ++group;
        }
      }
      const double exact = open ? da + db : some && keep ? INFINITY : -INFINITY;
      before = 0;
      rt_dev::static_for<1, LANES>([&](auto oc) {
        constexpr int CTRL = 0x120 + decltype(oc)::value;
        const double o = of_lane(exact, [](unsigned v) { return dpp<CTRL>(v); });
        before += o > exact || (o == exact && ((lane - decltype(oc)::value) & (LANES - 1)) < lane);
      });
      keep = before < p.kept;
    }
    const unsigned on = (unsigned)(__ballot(keep) >> (threadIdx.x & 48));
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const unsigned group = __umulhi((unsigned)(v * LANES + lane), p.per_mul);
      if (!((on >> (group & 31)) & 1)) c[v] = -INFINITY;
    }
  }
  // The k-th greatest of the token's values m (of different ones, so never above
  // the k-th of all c where m are some of them), and the candidates above it.  Fewer
  // than k different numbers say nothing of the k-th of all c, unless m are all c.
  float least = 0.0f;
  unsigned count = 0, upto = 0, all = 0;  // candidates of this lane, with those of the lanes before it, of the token
  auto choose = [&](auto nc, const float* m) {
    float kth = INFINITY;
    bool short_of_k = false;
    for (int r = 0; r < p.k; ++r) {
      float best = -INFINITY;
#pragma unroll
      for (int v = 0; v < decltype(nc)::value; ++v) best = fmaxf(best, m[v] < kth ? m[v] : -INFINITY);
      best = lanes_max<LANES>(best);
      if (best == -INFINITY) {  // the wave's other tokens may go on
        short_of_k = decltype(nc)::value < VPL;
        break;
      }
      kth = best;
    }
    least = kth - far(kth);
    count = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) count += c[v] >= least;
    upto = count;
    upto += dpp<0x111>(upto);
    upto += dpp<0x112>(upto);
    upto += dpp<0x114>(upto);
    upto += dpp<0x118>(upto);
    all = (unsigned)__shfl((int)upto, (threadIdx.x & 48) + 15, 64);
    return short_of_k || !(fabsf(kth) < INFINITY) || all > LANES || all < (unsigned)p.k;
  };
  // First by the greatest of each half of a lane's values: the k-th of those 32 is a
  // little low, and seldom so low that 16 lanes do not hold what is above it.
  bool again = true;
  if constexpr (VPL > 4) {
    float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int v = 0; v < VPL; ++v) m[v & 1] = fmaxf(m[v & 1], c[v]);
    again = choose(std::integral_constant<int, 2>{}, m);
  }
  if (__any(again)) slow |= choose(std::integral_constant<int, VPL>{}, c);
  if (__any(slow)) return false;
  unsigned at = upto - count;
#pragma unroll
  for (int v = 0; v < VPL; ++v)
    if (c[v] >= least) lds.chosen[at++] = v * LANES + lane;
  rt_dev::wave_lds_order();
  // The candidates, a lane each.
  const bool in = (unsigned)lane < all;
  const unsigned e = in ? lds.chosen[lane] : 0;
  const double z = (double)rt_dev::load1<DT>(p.logits, row + e);
  const double score = p.sigmoid ? sigmoid64(z) : exp(z - (double)top);
  const unsigned long long key = in ? order_key(p.bias ? score + (double)p.bias[e] : score) : 0;
  const unsigned hi = (unsigned)(key >> 32), lo = (unsigned)key;
  int rank = 0;  // candidates that come before this one
  rt_dev::static_for<1, LANES>([&](auto oc) {
    constexpr int CTRL = 0x120 + decltype(oc)::value;  // row_ror
    const unsigned long long o = ((unsigned long long)dpp<CTRL>(hi) << 32) | dpp<CTRL>(lo);
    const unsigned oe = dpp<CTRL>(e);
    rank += o > key || (o == key && oe < e);
  });
  const bool chosen = in && rank < p.k;
  const double sum = lanes_sum<LANES>(chosen ? score : 0.0);
  if (chosen && token < p.tokens) {
    p.ids[token * p.k + rank] = e;
    p.weights[token * p.k + rank] = weight_of(p, score, sum);
  }
  return true;
}

template <int DT, int LANES, int VPL>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs p) {
  constexpr int ROWS = 256 / LANES;
  __shared__ RouteRow<LANES, VPL> rows[ROWS];
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  for (long long t0 = (long long)blockIdx.x * ROWS; t0 < p.tokens; t0 += (long long)gridDim.x * ROWS) {
    rt_dev::wave_lds_order();
    if constexpr (LANES == 16 && VPL >= 4) {
      if (p.fast && route_fast<DT, VPL>(p, t0 + slot, lane, rows[slot])) continue;
      rt_dev::wave_lds_order();
    }
    route_exact<DT, LANES, VPL>(p, t0 + slot, lane, rows[slot]);
  }
}

// dlogits from the gradient of the weights.  With w = scale s_j / Z and g_j
// its gradient, ds_j = (scale / Z) (g_j - sum_i g_i s_i / Z) (Z = 1 and no
// second term without renormalising), and
//   sigmoid: dx_j = s_j (1 - s_j) ds_j for the chosen, 0 for the others;
//   softmax: dx_e = s_e (ds_e [e chosen] - sum_j s_j ds_j), whose second term
//            is 0 when renormalised (the weights are then a softmax of the
//            chosen logits alone).
// So a chosen expert's is s_j (g_j - sum_i w_i g_i), of weights w that add up to
// 1 with those of g = 0 (the experts that softmax did not choose).  Where one
// weight is nearly 1 that is a small difference of large numbers, so with
// m the chosen of the greatest logit it is added up as
//   s_j (g_j U + sum_i w_i (g_m - g_i) + (g_j - g_m) sum_i w_i),
// i over the chosen and U what the others' weights add up to; 1 - sigmoid(x) is
// likewise exp(-x) sigmoid(x).
// The chosen s are held in 64 bits: a bias or the groups may choose experts whose
// scores are all below what 32 bits hold, and their quotients are still weights.
// A lane has every LANES-th choice and writes it to its expert's place in LDS; one
// that another choice has named is added in a turn of its own.  16384 tokens of 256
// experts, 8 chosen: sigmoid 8.0 us (17 MB written), softmax not renormalised 12.5.
template <int DT, int LANES, int VPL>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteArgs p) {
  constexpr int ROWS = 256 / LANES, T = kMaxChoices / LANES;
  __shared__ unsigned slots[ROWS][LANES * VPL];  // of each expert: its first choice, then its gradient
  const int lane = threadIdx.x % LANES;
  unsigned* const of = slots[threadIdx.x / LANES];
  const bool whole = !p.sigmoid && !p.renorm;  // weights of all experts add up to 1, not of the chosen
  for (long long t0 = (long long)blockIdx.x * ROWS; t0 < p.tokens; t0 += (long long)gridDim.x * ROWS) {
  const long long token = t0 + threadIdx.x / LANES;
  const long long row = min(token, p.tokens - 1) * p.experts, ch = min(token, p.tokens - 1) * p.k;
  const int E = p.experts;
#pragma unroll
  for (int v = 0; v < VPL; ++v) of[v * LANES + lane] = kMaxChoices;
  float x[VPL], top = -INFINITY, total = 0.0f;
  if (!p.sigmoid) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int e = v * LANES + lane;
      x[v] = e < E ? rt_dev::load1<DT>(p.logits, row + e) : -INFINITY;
      top = fmaxf(top, x[v]);
    }
    top = lanes_max<LANES>(top);
    if (top == -INFINITY) top = 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      x[v] = expf(x[v] - top);
      total += x[v];
    }
    total = lanes_sum<LANES>(total);
    if (total == 0.0f) total = 1.0f;
  }
  // The choices: score, 1 - score (sigmoid), gradient; the logit and the gradient of the greatest.
  double s[T], rest1[T], g[T];
  unsigned id[T];
  float most = -INFINITY, gm = 0.0f;
  auto greater = [&](float l, float gl) {  // of equal logits the greater gradient: the same in every lane
    const bool other = l > most || (l == most && gl > gm);
    most = other ? l : most;
    gm = other ? gl : gm;
  };
  rt_dev::wave_lds_order();
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int j = t * LANES + lane;
    s[t] = g[t] = 0.0;
    rest1[t] = 1.0;
    id[t] = 0xffffffffu;
    if (j < p.k) {
      id[t] = p.ids[ch + j];
      if (id[t] < (unsigned)E) {
        const float l = rt_dev::load1<DT>(p.logits, row + id[t]), gl = p.dweights[ch + j];
        if (p.sigmoid) {
          const double power = exp(-(double)l);
          s[t] = 1.0 / (1.0 + power);
          if (power < INFINITY) rest1[t] = power * s[t];
        } else {
          s[t] = exp((double)l - (double)top) / (double)total;
        }
        g[t] = (double)gl;
        greater(l, gl);
        atomicMin(&of[id[t]], (unsigned)j);
      }
    }
  }
  over_lanes<LANES>([&](auto from) {
    const float l = __uint_as_float(from(__float_as_uint(most))), gl = __uint_as_float(from(__float_as_uint(gm)));
    greater(l, gl);
  });
  rt_dev::wave_lds_order();
  bool first[T], again = false;  // whether a choice is the first of its expert (a program's own may repeat one)
  double z = 0.0, gs = 0.0, apart = 0.0, others = 0.0;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    first[t] = id[t] < (unsigned)E && of[id[t]] == (unsigned)(t * LANES + lane);
    again |= id[t] < (unsigned)E && !first[t];
    const bool once = !whole || first[t];
    z += once ? s[t] : 0.0;
    apart += s[t] * ((once ? (double)gm : 0.0) - g[t]);
    gs += s[t] * g[t];
  }
  z = lanes_sum<LANES>(z);
  apart = lanes_sum<LANES>(apart);
  float rest = 0.0f;  // of the experts that were not chosen: -sum_j s_j ds_j
  if (whole) {
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) sum += of[v * LANES + lane] == kMaxChoices ? x[v] : 0.0f;
    others = (double)lanes_sum<LANES>(sum) / (double)total;
    rest = -p.scale * (float)lanes_sum<LANES>(gs);
  }
  rt_dev::wave_lds_order();
#pragma unroll
  for (int v = 0; v < VPL; ++v) of[v * LANES + lane] = __float_as_uint(rest == 0.0f ? 0.0f : rest * (x[v] / total));
  rt_dev::wave_lds_order();
  float add[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    add[t] = 0.0f;
    if (t * LANES + lane >= p.k) continue;
    double d = g[t], w = s[t];
    if (p.renorm) {
      w = z == 0.0 ? 0.0 : s[t] / z;  // no chosen score: the weights were zeros
      d = z == 0.0 ? 0.0 : apart / z + (g[t] - (double)gm);
    } else if (whole && first[t]) {
      d = g[t] * others + (apart + (g[t] - (double)gm) * z);
    }
    add[t] = (float)(w * (double)p.scale * d * rest1[t]);
    if (first[t]) of[id[t]] = __float_as_uint(add[t]);
  }
  rt_dev::wave_lds_order();
  if (__any(again)) {
#pragma unroll
    for (int t = 0; t < T; ++t)
      for (int l = 0; l < LANES; ++l) {  // in their order
        if (lane == l && id[t] < (unsigned)E && !first[t])
          of[id[t]] = __float_as_uint(__uint_as_float(of[id[t]]) + add[t]);
        rt_dev::wave_lds_order();
      }
  }
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const int e = v * LANES + lane;
    if (e < E && token < p.tokens) rt_dev::store1<DT>(p.dlogits, row + e, __uint_as_float(of[e]));
  }
  rt_dev::wave_lds_order();
  }
}

template <bool GRAD, int DT>
hipError_t route_launch(hipStream_t s, const RouteArgs& p) {
  auto go = [&](auto lanes, auto vpl) {
    constexpr int L = decltype(lanes)::value, V = decltype(vpl)::value;
    const dim3 grid(rt::grid_of((p.tokens + 256 / L - 1) / (256 / L)));
    if constexpr (GRAD) rt::launch(route_grad_kernel<DT, L, V>, grid, dim3(256), 0, s, p);
    else rt::launch(route_kernel<DT, L, V>, grid, dim3(256), 0, s, p);
    return hipGetLastError();
  };
  using std::integral_constant;
  const integral_constant<int, 16> row;
  const integral_constant<int, 64> wave;
  if (p.experts <= 16) return go(row, integral_constant<int, 1>{});
  if (p.experts <= 32) return go(row, integral_constant<int, 2>{});
  if (p.experts <= 64) return go(row, integral_constant<int, 4>{});
  if (p.experts <= 128) return go(row, integral_constant<int, 8>{});
  if (p.experts <= 256) return go(row, integral_constant<int, 16>{});
  if (p.experts <= 512) return go(wave, integral_constant<int, 8>{});
  return go(wave, integral_constant<int, 16>{});
}

int check_route(rt_ctx* c, const rt_buf* logits, int score, const rt_buf* ids, const rt_buf* weights, RouteArgs* p) {
  if (logits->rank != 2 || ids->rank != 2) return rt::fail(c, RT_ERR_SHAPE, "route: logits [tokens, experts], ids [tokens, k]");
  if (!rt::is_float(logits->dtype)) return rt::fail(c, RT_ERR_DTYPE, "route: logits are f32, bf16 or f16");
  if (ids->dtype != RT_U32 || weights->dtype != RT_F32) return rt::fail(c, RT_ERR_DTYPE, "route: ids are u32, weights f32");
  const size_t n = logits->shape[0], e = logits->shape[1], k = ids->shape[1];
  if (ids->shape[0] != n || weights->n != n * k || weights->rank != 2 || weights->shape[0] != n)
    return rt::fail(c, RT_ERR_SHAPE, "route: ids and weights must be [%zu, k]", n);
  if (e < 1 || e > (size_t)kMaxExperts) return rt::fail(c, RT_ERR_SHAPE, "route: between 1 and %d experts", kMaxExperts);
  if (k < 1 || k > e || k > (size_t)kMaxChoices)
    return rt::fail(c, RT_ERR_SHAPE, "route: k between 1 and the experts, at most %d", kMaxChoices);
  if (n > (size_t(1) << 30)) return rt::fail(c, RT_ERR_SHAPE, "route: at most 2^30 tokens");
  if (score != RT_SCORE_SOFTMAX && score != RT_SCORE_SIGMOID) return rt::fail(c, RT_ERR_INVALID, "route: unknown score %d", score);
  p->logits = logits->ptr;
  p->tokens = (long long)n;
  p->experts = (int)e;
  p->k = (int)k;
  p->sigmoid = score == RT_SCORE_SIGMOID;
  return RT_OK;
}

}  // namespace

using namespace rt;

extern "C" {

int rt_route(rt_ctx* c, const rt_buf* logits, const rt_buf* bias, int score, size_t groups, size_t kept, int renormalise,
             float scale, rt_buf* ids, rt_buf* weights) {
  CHECK_CTX(c);
  if (!logits || !ids || !weights) return fail(c, RT_ERR_INVALID, "null buffer");
  RouteArgs p{};
  if (int rc = check_route(c, logits, score, ids, weights, &p)) return rc;
  const size_t e = logits->shape[1];
  if (bias && (bias->dtype != RT_F32 || bias->n != e)) return fail(c, RT_ERR_SHAPE, "route: the bias must be f32 [%zu]", e);
  if (groups < 1 || groups > (size_t)kMaxGroups || e % groups != 0)
    return fail(c, RT_ERR_SHAPE, "route: %zu experts in %zu groups (at most %d, of equal size)", e, groups, kMaxGroups);
  if (kept < 1 || kept > groups) return fail(c, RT_ERR_SHAPE, "route: %zu of %zu groups", kept, groups);
  if ((size_t)p.k > e / groups * kept)
    return fail(c, RT_ERR_SHAPE, "route: %d choices among the %zu experts of %zu groups", p.k, e / groups * kept, kept);
  if (p.tokens == 0) return RT_OK;
  p.bias = bias ? static_cast<const float*>(bias->ptr) : nullptr;
  p.ids = static_cast<unsigned*>(ids->ptr);
  p.weights = static_cast<float*>(weights->ptr);
  p.groups = (int)groups;
  p.kept = (int)kept;
  p.renorm = renormalise != 0;
  p.per = (int)(e / groups);
  p.per_mul = p.per > 1 ? (unsigned)(((1ull << 32) + p.per - 1) / p.per) : 0;
  // route_fast ranks choices and groups a lane each.
  p.fast = p.k <= 16 && (kept == groups || (groups <= 16 && p.per > 1)) && (p.sigmoid || (p.renorm && !bias));
  p.scale = scale;
  Launch L(c, "route");
  HIP_TRY(c, for_float(logits->dtype, [&](auto dt) { return route_launch<false, decltype(dt)::value>(c->stream, p); }), "route");
  return RT_OK;
}

int rt_route_backward(rt_ctx* c, const rt_buf* logits, int score, int renormalise, float scale, const rt_buf* ids,
                      const rt_buf* dweights, rt_buf* dlogits) {
  CHECK_CTX(c);
  if (!logits || !ids || !dweights || !dlogits) return fail(c, RT_ERR_INVALID, "null buffer");
  RouteArgs p{};
  if (int rc = check_route(c, logits, score, ids, dweights, &p)) return rc;
  if (dlogits->dtype != logits->dtype) return fail(c, RT_ERR_DTYPE, "route backward: dlogits are of the logits' type");
  if (dlogits->rank != 2 || dlogits->shape[0] != logits->shape[0] || dlogits->shape[1] != logits->shape[1])
    return fail(c, RT_ERR_SHAPE, "route backward: dlogits must be [%zu,%zu]", logits->shape[0], logits->shape[1]);
  if (p.tokens == 0) return RT_OK;
  p.ids = static_cast<unsigned*>(ids->ptr);
  p.dweights = static_cast<const float*>(dweights->ptr);
  p.dlogits = dlogits->ptr;
  p.renorm = renormalise != 0;
  p.scale = scale;
  Launch L(c, "route_bwd");
  HIP_TRY(c, for_float(logits->dtype, [&](auto dt) { return route_launch<true, decltype(dt)::value>(c->stream, p); }),
          "route backward");
  return RT_OK;
}

}  // extern "C"

// Routing to experts with softmax or sigmoid scores, a balance bias, groups and scaled
// weights (qmm_moe_route_scored), into the lists that qmm_moe_route makes.
//
//   score  s = softmax(logits) or 1 / (1 + exp(-logit)); a NaN logit counts as -inf
//          (score 0), +inf as the largest finite value; with no finite logit all are 0
//   choice c = s + bias (a NaN sum comes last; cut to +-1e300)
//   group  the sum of a group's group_top (1 or 2) largest choices; the topk_groups
//          best groups stay, ties to the lower group
//   top-k  of the choices in those groups, ties to the lower expert
//   weight s, over the selection's sum (0 where that is 0) if renormalize, times scale
//
// Scores are formed in 64 bits. Experts' scores are close together (256 of them in
// [0, 1]), a token in a few thousand has two within an f32 rounding of each other at
// its top-k border, and the list must not hang on which exponential made them; the
// f64 work is a few microseconds of a few thousand tokens'.
#pragma once

#include "qmm_mx_common.h"

namespace qmm {

struct RouteArgs {
  int T, E, k, sigmoid, groups, topk_groups, group_top, renorm;
  float scale;
};

__device__ __forceinline__ double route_wave_max(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = fmax(v, __shfl_xor(v, d));
  return v;
}
__device__ __forceinline__ double route_wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// One token by one wave, expert e = 64 i + lane in register i. Lane j < k returns the
// token's j-th expert in increasing order, and its weight. `ch`: E doubles of LDS, this
// wave's own.
template <int R>
__device__ __forceinline__ void route_token(const float* __restrict__ logits, const float* __restrict__ bias,
                                            const RouteArgs& a, double* ch, int& expert, float& weight) {
  const int lane = threadIdx.x & 63;
  double s[R], c[R];
  double mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = 64 * i + lane;
    float l = e < a.E ? logits[e] : -INFINITY;
    l = l != l ? -INFINITY : fminf(l, 3.40282347e38f);
    s[i] = l;
    mx = fmax(mx, s[i]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = 1.0 / (1.0 + exp(-s[i]));
  } else {
    mx = route_wave_max(mx);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[i] = mx == -INFINITY ? 0.0 : exp(s[i] - mx);
      sum += s[i];
    }
    sum = route_wave_sum(sum);
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = 64 * i + lane;
    c[i] = s[i];
    if (bias != nullptr && e < a.E) {
      const double v = s[i] + (double)bias[e];
      c[i] = v != v ? -1e300 : fmin(fmax(v, -1e300), 1e300);
    }
    if (e >= a.E) c[i] = -INFINITY;
  }
  if (a.groups > 1 && a.topk_groups < a.groups) {
    const int gs = a.E / a.groups;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (64 * i + lane < a.E) ch[64 * i + lane] = c[i];
    // (one wave writes and reads its own part: the LDS keeps the order)
    __builtin_amdgcn_wave_barrier();
    double best = -INFINITY, second = -INFINITY;
    if (lane < a.groups)
      for (int j = 0; j < gs; ++j) {
        const double v = ch[lane * gs + j];
        second = fmax(second, fmin(best, v));
        best = fmax(best, v);
      }
    const double score = a.group_top == 2 ? best + second : best;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double o = __shfl(score, g);
      rank += o > score || (o == score && g < lane);
    }
    const unsigned long long kept = __ballot(lane < a.groups && rank < a.topk_groups);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = 64 * i + lane;
      if (e < a.E && !(kept >> (e / gs) & 1)) c[i] = -INFINITY;
    }
    __builtin_amdgcn_wave_barrier();
  }
  // top-k: the largest choice, then the lowest expert that has it
  int mine = 0x7fffffff;  // lane j < k: the j-th selected expert
  double ms = 0.0;        // its score
  for (int j = 0; j < a.k; ++j) {
    double top = c[0];
#pragma unroll
    for (int i = 1; i < R; ++i) top = fmax(top, c[i]);
    top = route_wave_max(top);
    int e = -1;
    double sc = 0.0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const unsigned long long b = __ballot(c[i] == top);
      if (e < 0 && b) {
        const int l = __builtin_ctzll(b);
        e = 64 * i + l;
        sc = __shfl(s[i], l);
        if (lane == l) c[i] = -INFINITY;
      }
    }
    if (lane == j) {
      mine = e;
      ms = sc;
    }
  }
  const double sum = route_wave_sum(ms);
  double w = ms;
  if (a.renorm) w = sum > 0.0 ? ms / sum : 0.0;
  const float wf = (float)(w * (double)a.scale);
  int place = 0;  // increasing expert order
  for (int j = 0; j < a.k; ++j) place += __shfl(mine, j) < mine;
  // lane p takes the selection whose place is p
  expert = 0;
  weight = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    const int p = __shfl(place, j), e = __shfl(mine, j);
    const float v = __shfl(wf, j);
    if (lane == p) {
      expert = e;
      weight = v;
    }
  }
}

constexpr int kRouteMaxE = 1024, kRouteMaxK = 32;

// The lists of one group of up to 64 tokens [t0, t0 + nt), of which sel_e / sel_w (LDS)
// hold the selections in expert order: `before` and `total` are the counts of each
// expert over the tokens before t0 and over all of them. A pair's place is its expert's
// offset, plus `before`, plus the number of the group's earlier tokens that selected it
// (a bit mask of tokens per expert: any order of the ORs gives the same mask).
template <int NT>
__device__ __forceinline__ void route_lists(const RouteArgs& a, int t0, int nt, const uint16_t* sel_e,
                                            const float* sel_w, const int* before, const int* total, int* offs,
                                            unsigned long long* mask, int* __restrict__ counts,
                                            int* __restrict__ offsets, int* __restrict__ pair_token,
                                            float* __restrict__ pair_weight, int* __restrict__ token_pairs) {
  const int t = threadIdx.x;
  for (int e = t; e < a.E; e += NT) mask[e] = 0;
  if (t < 64) {  // exclusive prefix of the totals
    int base = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + t, v = e < a.E ? total[e] : 0;
      int sum = v;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        if (t >= d) sum += o;
      }
      if (e < a.E) offs[e] = base + sum - v;
      base += __shfl(sum, 63);
    }
    if (t == 0) offs[a.E] = base;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = t; e <= a.E; e += NT) {
      offsets[e] = offs[e];
      if (e < a.E) counts[e] = total[e];
    }
  const int np = nt * a.k;
  for (int p = t; p < np; p += NT) atomicOr(&mask[sel_e[p]], 1ull << (p / a.k));
  __syncthreads();
  for (int p = t; p < np; p += NT) {
    const int i = p / a.k, e = sel_e[p];
    const int at = offs[e] + before[e] + __popcll(mask[e] & ((1ull << i) - 1ull));
    pair_token[at] = t0 + i;
    pair_weight[at] = sel_w[p];
    token_pairs[(long long)t0 * a.k + p] = at;
  }
}

}  // namespace qmm

// Up to 16 tokens of up to 256 experts: one launch, a wave a token.
#define QMM_ROUTE_SMALL(R)                                                                                             \
  extern "C" __global__ void __launch_bounds__(1024) qmm_route_small_r##R(                                        \
      const float* __restrict__ logits, const float* __restrict__ bias, qmm::RouteArgs a, int* __restrict__ counts,  \
      int* __restrict__ offsets, int* __restrict__ pair_token, float* __restrict__ pair_weight,                   \
      int* __restrict__ token_pairs) {                                                                            \
    __shared__ double ch[16][64 * R];                                                                             \
    __shared__ uint16_t sel_e[16 * qmm::kRouteMaxK];                                                              \
    __shared__ float sel_w[16 * qmm::kRouteMaxK];                                                                 \
    __shared__ int before[64 * R], total[64 * R], offs[64 * R + 1];                                               \
    __shared__ unsigned long long mask[64 * R];                                                                   \
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;                                                   \
    for (int e = threadIdx.x; e < a.E; e += 1024) before[e] = total[e] = 0;                                       \
    __syncthreads();                                                                                              \
    if (wave < a.T) {                                                                                             \
      int e;                                                                                                      \
      float w;                                                                                                    \
      qmm::route_token<R>(logits + (long long)wave * a.E, bias, a, ch[wave], e, w);                               \
      if (lane < a.k) {                                                                                           \
        sel_e[wave * a.k + lane] = (uint16_t)e;                                                                   \
        sel_w[wave * a.k + lane] = w;                                                                             \
        atomicAdd(&total[e], 1);                                                                                  \
      }                                                                                                           \
    }                                                                                                             \
    __syncthreads();                                                                                              \
    qmm::route_lists<1024>(a, 0, a.T, sel_e, sel_w, before, total, offs, mask, counts, offsets, pair_token,       \
                           pair_weight, token_pairs);                                                             \
  }
QMM_ROUTE_SMALL(1)
QMM_ROUTE_SMALL(2)
QMM_ROUTE_SMALL(4)

// Any number of tokens: their selections, a wave a token; the lists follow.
#define QMM_ROUTE_TOKENS(R)                                                                                       \
  extern "C" __global__ void __launch_bounds__(256) qmm_route_tokens_r##R(                                        \
      const float* __restrict__ logits, const float* __restrict__ bias, qmm::RouteArgs a,                         \
      uint16_t* __restrict__ ids, float* __restrict__ wts) {                                                      \
    __shared__ double ch[4][64 * R];                                                                              \
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;                                                   \
    const int t = 4 * blockIdx.x + wave;                                                                          \
    if (t >= a.T) return;                                                                                         \
    int e;                                                                                                        \
    float w;                                                                                                      \
    qmm::route_token<R>(logits + (long long)t * a.E, bias, a, ch[wave], e, w);                                    \
    if (lane < a.k) {                                                                                             \
      ids[(long long)t * a.k + lane] = (uint16_t)e;                                                               \
      wts[(long long)t * a.k + lane] = w;                                                                         \
    }                                                                                                             \
  }
QMM_ROUTE_TOKENS(1)
QMM_ROUTE_TOKENS(2)
QMM_ROUTE_TOKENS(4)
QMM_ROUTE_TOKENS(16)

// The lists from all tokens' selections, 64 tokens a workgroup. Every workgroup counts
// the selections before its tokens and the rest by itself (LDS counters, eight copies
// by lane where experts are few, so that a wave's adds fall on distinct words); integer
// adds, so their order does not matter.
extern "C" __global__ void __launch_bounds__(1024) qmm_route_lists(
    qmm::RouteArgs a, const uint16_t* __restrict__ ids, const float* __restrict__ wts, int* __restrict__ counts,
    int* __restrict__ offsets, int* __restrict__ pair_token, float* __restrict__ pair_weight,
    int* __restrict__ token_pairs) {
  __shared__ uint16_t sel_e[64 * qmm::kRouteMaxK];
  __shared__ float sel_w[64 * qmm::kRouteMaxK];
  __shared__ int cnt[2][qmm::kRouteMaxE];
  __shared__ int before[qmm::kRouteMaxE], total[qmm::kRouteMaxE], offs[qmm::kRouteMaxE + 1];
  __shared__ unsigned long long mask[qmm::kRouteMaxE];
  const int t = threadIdx.x, t0 = 64 * blockIdx.x, nt = min(64, a.T - t0);
  const int copies = a.E <= 128 ? 8 : 1;
  for (int i = t; i < a.E * copies; i += 1024) cnt[0][i] = cnt[1][i] = 0;
  __syncthreads();
  const long long first = (long long)t0 * a.k, all = (long long)a.T * a.k;
  for (long long p = t; p < all; p += 1024)
    atomicAdd(&cnt[p < first ? 0 : 1][ids[p] * copies + (t & (copies - 1))], 1);
  for (int p = t; p < nt * a.k; p += 1024) {
    sel_e[p] = ids[first + p];
    sel_w[p] = wts[first + p];
  }
  __syncthreads();
  for (int e = t; e < a.E; e += 1024) {
    int b = 0, r = 0;
    for (int c = 0; c < copies; ++c) {
      b += cnt[0][e * copies + c];
      r += cnt[1][e * copies + c];
    }
    before[e] = b;
    total[e] = b + r;
  }
  __syncthreads();
  qmm::route_lists<1024>(a, t0, nt, sel_e, sel_w, before, total, offs, mask, counts, offsets, pair_token, pair_weight,
                         token_pairs);
}

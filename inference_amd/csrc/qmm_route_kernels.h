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
// f64 work is a few microseconds of a few thousand tokens'. Sigmoid scores of logits
// above 53 ln 2 = 36.74 are 1 in 64 bits as well, and tie.
#pragma once

#include "qmm_mx_common.h"

namespace qmm {

struct RouteArgs {
  int T, E, k, sigmoid, groups, topk_groups, group_top, renorm;
  float scale;
};

// A lane's value as a scalar, and a value of another lane of a row of 16 by its pattern:
// a wave's maximum and sum are chains of these, a tenth of the latency of a shuffle each.
__device__ __forceinline__ int route_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ float route_lane(float v, int l) { return __int_as_float(route_lane(__float_as_int(v), l)); }
__device__ __forceinline__ double route_lane(double v, int l) {
  return __hiloint2double(route_lane(__double2hiint(v), l), route_lane(__double2loint(v), l));
}
template <int P>
__device__ __forceinline__ double route_row(double v) {
  const int lo = __double2loint(v), hi = __double2hiint(v);
  return __hiloint2double(__builtin_amdgcn_update_dpp(hi, hi, P, 0xf, 0xf, true),
                          __builtin_amdgcn_update_dpp(lo, lo, P, 0xf, 0xf, true));
}
template <int P>
__device__ __forceinline__ int route_row(int v) {
  return __builtin_amdgcn_update_dpp(v, v, P, 0xf, 0xf, true);
}
template <typename T, typename F>
__device__ __forceinline__ T route_wave(T v, F f) {
  v = f(v, route_row<0xb1>(v));   // lanes 1 0 3 2 of four
  v = f(v, route_row<0x4e>(v));   // 2 3 0 1
  v = f(v, route_row<0x141>(v));  // eight, mirrored
  v = f(v, route_row<0x140>(v));  // sixteen, mirrored
  return f(f(route_lane(v, 0), route_lane(v, 16)), f(route_lane(v, 32), route_lane(v, 48)));
}
__device__ __forceinline__ int route_wave_max(int v) {
  return route_wave(v, [](int a, int b) { return max(a, b); });
}
__device__ __forceinline__ double route_wave_sum(double v) {
  return route_wave(v, [](double a, double b) { return a + b; });
}
// A word whose order as a signed integer is that of a float's bits (its own inverse).
__device__ __forceinline__ int route_order(int bits) { return bits ^ (bits >> 31 & 0x7fffffff); }

// One token by one wave, expert e = 64 i + lane in register i. Lane j < k returns the
// token's j-th expert in increasing order, and its weight. `ch`: E doubles of LDS, this
// wave's own.
//
// What bounds it: instruction issue, of the f64 exponentials and quotients of all experts,
// the groups' scores and the k maxima over the wave. 4096 tokens of 256 experts, 8 of 8
// groups' 4 with sigmoid scores: 12.7 us; 13.5 with 64-bit maxima, 16.4 with maxima, sums
// and group scores by shuffles.
template <int R>
__device__ __forceinline__ void route_token(const float* __restrict__ logits, const float* __restrict__ bias,
                                            const RouteArgs& a, double* ch, int& expert, float& weight) {
  const int lane = threadIdx.x & 63;
  double s[R], c[R];
  float add[R];  // (asked for together with the logits)
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = 64 * i + lane;
    float l = e < a.E ? logits[e] : -INFINITY;
    add[i] = bias != nullptr && e < a.E ? bias[e] : 0.0f;
    l = l != l ? -INFINITY : fminf(l, 3.40282347e38f);
    s[i] = l;
    mx = fmaxf(mx, l);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = 1.0 / (1.0 + exp(-s[i]));
  } else {
    mx = __int_as_float(route_order(route_wave_max(route_order(__float_as_int(mx)))));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[i] = mx == -INFINITY ? 0.0 : exp(s[i] - (double)mx);
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
      const double v = s[i] + (double)add[i];
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
    // `sub` lanes a group, then lane g has group g's score
    int sub = 64;
    while (sub * a.groups > 64) sub /= 2;
    const int mine = lane / sub;
    double best = -INFINITY, second = -INFINITY;
    if (mine < a.groups)
      for (int j = lane % sub; j < gs; j += sub) {
        const double v = ch[mine * gs + j];
        second = fmax(second, fmin(best, v));
        best = fmax(best, v);
      }
    for (int d = 1; d < sub; d *= 2) {
      const double b = __shfl_xor(best, d), n = __shfl_xor(second, d);
      second = fmax(fmax(second, n), fmin(best, b));
      best = fmax(best, b);
    }
    const double part = a.group_top == 2 ? best + second : best;
    const double score = __shfl(part, lane * sub & 63);
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double o = route_lane(part, g * sub);
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
  // top-k: the largest choice, then the lowest expert that has it. The choices as two words
  // that are ordered like them: the maximum of the high ones decides but for close choices.
  int hi[R];
  unsigned lo[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int b = __double2hiint(c[i]), sign = b >> 31;
    hi[i] = route_order(b);
    lo[i] = (unsigned)(__double2loint(c[i]) ^ sign);
  }
  int mine = 0x7fffffff;  // lane j < k: the j-th selected expert
  double ms = 0.0;        // its score
  for (int j = 0; j < a.k; ++j) {
    int high = hi[0];
#pragma unroll
    for (int i = 1; i < R; ++i) high = max(high, hi[i]);
    high = route_wave_max(high);
    unsigned long long b[R];
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      b[i] = __ballot(hi[i] == high);
      n += __popcll(b[i]);
    }
    if (n > 1) {
      int low = INT_MIN;  // (unsigned words, their top bit flipped)
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (hi[i] == high) low = max(low, (int)(lo[i] ^ 0x80000000u));
      low = route_wave_max(low);
#pragma unroll
      for (int i = 0; i < R; ++i) b[i] = __ballot(hi[i] == high && (int)(lo[i] ^ 0x80000000u) == low);
    }
    int e = -1;
    double sc = 0.0;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (e < 0 && b[i]) {
        const int l = __builtin_ctzll(b[i]);
        e = 64 * i + l;
        sc = route_lane(s[i], l);
        if (lane == l) {  // below every choice
          hi[i] = INT_MIN;
          lo[i] = 0;
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
  // lane p takes the selection whose place in increasing expert order is p
  int place = 0;
  for (int j = 0; j < a.k; ++j) place += route_lane(mine, j) < mine;
  expert = 0;
  weight = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    const int p = route_lane(place, j), e = route_lane(mine, j);
    const float v = route_lane(wf, j);
    if (lane == p) {
      expert = e;
      weight = v;
    }
  }
}

constexpr int kRouteMaxK = 32;

// The lists of up to 16 tokens, by one workgroup: sel_e / sel_w (LDS) hold the selections
// in expert order, `total` each expert's count. A pair's place is its expert's offset plus
// the number of earlier tokens that selected it (a bit mask of tokens per expert: any
// order of the ORs gives the same mask).
__device__ __forceinline__ void route_lists(const RouteArgs& a, const uint16_t* sel_e, const float* sel_w,
                                            const int* total, int* offs, int (&sums)[4], unsigned* mask,
                                            int* __restrict__ counts,
                                            int* __restrict__ offsets, int* __restrict__ pair_token,
                                            float* __restrict__ pair_weight, int* __restrict__ token_pairs) {
  const int t = threadIdx.x;
  if (t < a.E) mask[t] = 0;
  int sum = 0, cnt = 0;  // prefix of the totals: of 64 experts a wave, then of the waves
  if (t < 256) {
    sum = cnt = t < a.E ? total[t] : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(sum, d);
      if ((t & 63) >= d) sum += o;
    }
    if ((t & 63) == 63) sums[t >> 6] = sum;
  }
  __syncthreads();
  if (t < a.E) {
    for (int i = 0; i < t >> 6; ++i) sum += sums[i];
    offs[t] = sum - cnt;
    offsets[t] = sum - cnt;
    counts[t] = cnt;
    if (t == a.E - 1) offsets[a.E] = sum;
  }
  const int i = t / a.k, e = i < a.T ? sel_e[t] : 0;
  if (i < a.T) atomicOr(&mask[e], 1u << i);
  __syncthreads();
  if (i < a.T) {
    const int at = offs[e] + __popc(mask[e] & ((1u << i) - 1u));
    pair_token[at] = i;
    pair_weight[at] = sel_w[t];
    token_pairs[t] = at;
  }
}

}  // namespace qmm

// Up to 16 tokens, and fewer of more experts (route_is_small): one launch, a wave a token.
#define QMM_ROUTE_SMALL(R)                                                                                             \
  extern "C" __global__ void __launch_bounds__(1024) qmm_route_small_r##R(                                        \
      const float* __restrict__ logits, const float* __restrict__ bias, qmm::RouteArgs a, int* __restrict__ counts,  \
      int* __restrict__ offsets, int* __restrict__ pair_token, float* __restrict__ pair_weight,                   \
      int* __restrict__ token_pairs) {                                                                            \
    __shared__ double ch[16][64 * R];                                                                             \
    __shared__ uint16_t sel_e[16 * qmm::kRouteMaxK];                                                              \
    __shared__ float sel_w[16 * qmm::kRouteMaxK];                                                                 \
    __shared__ int total[64 * R], offs[64 * R], sums[4];                                                          \
    __shared__ unsigned mask[64 * R];                                                                             \
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;                                                   \
    for (int e = threadIdx.x; e < a.E; e += 1024) total[e] = 0;                                                   \
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
    qmm::route_lists(a, sel_e, sel_w, total, offs, sums, mask, counts, offsets, pair_token, pair_weight,          \
                     token_pairs);                                                                                \
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

// The lists from all tokens' selections, a workgroup an expert: it counts the selections
// of lower experts (its offset) and its own, each thread over a run of the list, and
// writes its own pairs in the list's order. Every workgroup reads the whole list (2 bytes
// a selection), 64 selections a thread in flight; no atomics and no other launch. 32768
// selections of 256 experts: 6.9 us (11.8 by workgroups of 64 tokens that count every
// expert in LDS; 11.5 with one load of 8 selections after another; 14.4 with ranks by
// ballots over a wave's neighbouring selections, which is faster only where one expert has
// nearly all of them).
extern "C" __global__ void __launch_bounds__(1024) qmm_route_lists(
    qmm::RouteArgs a, const uint16_t* __restrict__ ids, const float* __restrict__ wts, int* __restrict__ counts,
    int* __restrict__ offsets, int* __restrict__ pair_token, float* __restrict__ pair_weight,
    int* __restrict__ token_pairs) {
  __shared__ int wave_eq[16], wave_lt[16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, e = blockIdx.x;
  const int all = a.T * a.k, run = ((all + 1023) / 1024 + 7) & ~7;  // runs of 16-byte pieces
  const int p0 = min(t * run, all), p1 = min(p0 + run, all);
  // 64 selections of a run at a time: bit j of the masks is selection j's
  auto masks = [&](int p, unsigned long long& is, unsigned long long& less) {
    qmm::mx_u32x4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (p + 8 * i < p1) v[i] = *reinterpret_cast<const qmm::mx_u32x4*>(ids + p + 8 * i);
    is = less = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (p + 8 * i < p1) {
        unsigned a8 = 0, b8 = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int id = (int)(v[i][j >> 1] >> (16 * (j & 1)) & 0xffff);
          a8 |= (unsigned)(id == e) << j;
          b8 |= (unsigned)(id < e) << j;
        }
        is |= (unsigned long long)a8 << (8 * i);
        less |= (unsigned long long)b8 << (8 * i);
      }
    if (p1 - p < 64) {  // (the list's last piece may be read past its end, within its workspace)
      is &= (1ull << (p1 - p)) - 1;
      less &= (1ull << (p1 - p)) - 1;
    }
  };
  unsigned long long is = 0, less = 0;
  int eq = 0, lt = 0;
  for (int p = p0; p < p1; p += 64) {
    masks(p, is, less);
    eq += __popcll(is);
    lt += __popcll(less);
  }
  int pre = eq, low = lt;  // inclusive prefix of eq, sum of lt, over the wave
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(pre, d);
    if (lane >= d) pre += o;
    low += __shfl_xor(low, d);
  }
  if (lane == 63) {
    wave_eq[wave] = pre;
    wave_lt[wave] = low;
  }
  __syncthreads();
  int at = pre - eq, total = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    at += wave_lt[i] + (i < wave ? wave_eq[i] : 0);
    total += wave_eq[i];
  }
  if (t == 0) {  // (its own run is empty before it: `at` is the expert's offset)
    counts[e] = total;
    offsets[e] = at;
    if (e == a.E - 1) offsets[a.E] = at + total;
  }
  if (eq == 0) return;
  for (int p = p0; p < p1; p += 64) {
    if (run > 64) masks(p, is, less);
    for (; is; is &= is - 1) {
      const int q = p + __builtin_ctzll(is);
      pair_token[at] = q / a.k;
      pair_weight[at] = wts[q];
      token_pairs[q] = at++;
    }
  }
}

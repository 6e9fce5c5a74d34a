// A beam search's selection (qmm_beam_select) and the reordering of what its beams hold.
//
// A continuation's score is beam score + logit - lse, lse = log sum exp(logits of the
// beam). Within a beam the order is the logits', so the first launch takes the largest
// `count` logits of each slice of a beam's row, with the slice's maximum and sum, in one
// pass over the logits; the second joins the slices' sums and takes the best of all lists,
// which are sorted, by their heads.
//
// Scores of different beams are compared in 64 bits: two of them lie within an f32
// rounding of each other (2^-20 at a score of -16) once in a few thousand selections, and
// the list must not hang on which order a sum was taken in. An f64 multiply-add costs what
// an f32 one does here, so the exponentials are f64 polynomials.
#pragma once

#include "qmm_kv_common.h"

namespace qmm {

constexpr int kBeamSlice = 4096;             // logits of a slice: 16 a thread
constexpr int kBeamMaxLists = 64 * 256;      // 64 beams of 2^20 logits

struct BeamArgs {
  const void* logits;
  long long ld;
  const float* scores;
  const int32_t* finished;
  int32_t *tokens, *parents, *out_finished;
  float* out_scores;
  // workspace, by row and slice: sum, maximum, sorted keys
  double* sums;
  float* maxima;
  uint64_t* lists;
  int type, beams, vocab, count, eos, slices, wide;
};

// 2^x for x <= 0, to 2^-31 of its value: the Taylor series of 2^f, |f| <= 1/2, to the
// eighth power (its ninth term is 0.3466^9 / 9! = 2.0e-10).
__device__ __forceinline__ double exp2_neg(double x) {
  x = fmax(x, -1080.0);
  const double n = rint(x), y = (x - n) * 0.69314718055994530942;
  double r = 1.0 / 40320.0;
  r = fma(r, y, 1.0 / 5040.0);
  r = fma(r, y, 1.0 / 720.0);
  r = fma(r, y, 1.0 / 120.0);
  r = fma(r, y, 1.0 / 24.0);
  r = fma(r, y, 1.0 / 6.0);
  r = fma(r, y, 0.5);
  r = fma(r, y, 1.0);
  r = fma(r, y, 1.0);
  return ldexp(r, (int)n);
}

// A logit as the search takes it (NaN: -inf, +inf: the largest finite value, -0: 0), and
// as the high half of a key: keys order by value, then the lower token, and 0 is none.
__device__ __forceinline__ float beam_logit(float x) {
  return x != x ? -INFINITY : fminf(x, 3.402823466e38f) + 0.0f;
}
__device__ __forceinline__ uint64_t beam_key(float x, int token) {
  if (x == -INFINITY) return 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const uint32_t u = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float beam_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int beam_token(uint64_t key) { return (int)~(uint32_t)key; }
// A beam that goes on with its logits.
__device__ __forceinline__ bool beam_live(const BeamArgs& a, int row) {
  const float s = a.scores[row];
  return s == s && s != -INFINITY && !(a.finished && a.finished[row]);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max32(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
}  // namespace qmm

// Grid slices x rows. A thread holds 16 logits. The count-th largest of the threads' own
// maxima is a bound that the slice's count largest logits pass: `count` threads have a
// logit at or above it and no other thread has one, so at most 16 count keys pass, and a
// key's place is the number of larger ones among them.
extern "C" __global__ void __launch_bounds__(256) qmm_beam_slices(qmm::BeamArgs a) {
  using namespace qmm;
  __shared__ uint64_t top[256];
  __shared__ uint64_t pass[16 * 128];
  __shared__ uint64_t bound;
  __shared__ int passed;
  __shared__ float wmax[4];
  __shared__ double wsum[4];
  const int row = blockIdx.y, sl = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (!beam_live(a, row)) return;
  const int first = sl * kBeamSlice;
  float x[16];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = first + 1024 * u + 4 * t;
    float v[4];
    if (i + 4 <= a.vocab) {
      load4_typed(v, a.logits, row * a.ld + i, a.type, a.wide);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < a.vocab ? load_typed(a.logits, row * a.ld + i + e, a.type) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * u + e] = beam_logit(v[e]);
  }
  float m = x[0];
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    m = fmaxf(m, x[i]);
    const uint64_t k = beam_key(x[i], first + 1024 * (i / 4) + 4 * t + i % 4);
    best = k > best ? k : best;
  }
  m = wave_max32(m);
  if (lane == 0) wmax[wave] = m;
  top[t] = best;
  if (t == 0) passed = 0;
  __syncthreads();
  m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  // (threads without a key have the key 0: the lower thread first)
  int place = 0;
  for (int i = 0; i < 256; ++i) place += top[i] > best || (top[i] == best && i < t) ? 1 : 0;
  if (place == a.count - 1) bound = best;
  double z = 0.0;
  if (m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < 16; ++i) z += exp2_neg(((double)x[i] - (double)m) * 1.44269504088896340736);
  }
  z = wave_sum64(z);
  if (lane == 0) wsum[wave] = z;
  __syncthreads();
  const uint64_t least = bound ? bound : 1;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t k = beam_key(x[i], first + 1024 * (i / 4) + 4 * t + i % 4);
    if (k >= least) pass[atomicAdd(&passed, 1)] = k;
  }
  __syncthreads();
  const long long slot = (long long)row * a.slices + sl;
  uint64_t* list = a.lists + slot * a.count;
  const int n = passed;
  for (int i = t; i < n; i += 256) {
    const uint64_t k = pass[i];
    int at = 0;
    for (int j = 0; j < n; ++j) at += pass[j] > k;
    if (at < a.count) list[at] = k;
  }
  for (int i = n + t; i < a.count; i += 256) list[i] = 0;
  if (t == 0) {
    a.maxima[slot] = m;
    a.sums[slot] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
  }
}

// One workgroup a search: the beams' lse, then `count` times the best head of its lists
// (beams x slices of them, list l = beam * slices + slice; a finished beam's first list is
// its end). A thread holds the best head of its lists.
extern "C" __global__ void __launch_bounds__(256) qmm_beam_merge(qmm::BeamArgs a) {
  using namespace qmm;
  __shared__ double lse[64];
  __shared__ double wbest[2][4];
  __shared__ uint64_t wtie[2][4];
  __shared__ uint8_t taken[kBeamMaxLists];  // entries that each list has given
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, row0 = b * a.beams;
  for (int w = wave; w < a.beams; w += 4) {
    const int row = row0 + w;
    if (!beam_live(a, row)) continue;
    float m = -INFINITY;
    for (int i = lane; i < a.slices; i += 64) m = fmaxf(m, a.maxima[(long long)row * a.slices + i]);
    m = wave_max32(m);
    double z = 0.0;
    if (m != -INFINITY)
      for (int i = lane; i < a.slices; i += 64) {
        const long long at = (long long)row * a.slices + i;
        if (a.maxima[at] != -INFINITY)
          z += a.sums[at] * exp2_neg(((double)a.maxima[at] - (double)m) * 1.44269504088896340736);
      }
    z = wave_sum64(z);
    if (lane == 0) lse[w] = (double)m + log(z);
  }
  const int lists = a.beams * a.slices;
  for (int l = t; l < lists; l += 256) taken[l] = 0;
  __syncthreads();
  // the head of list l past its first `skip` entries: score, and what orders equal ones
  auto head = [&](int l, int skip, double& s, uint64_t& tie) {
    s = -INFINITY;
    tie = ~0ull;
    const int w = l / a.slices, row = row0 + w;
    const float score = a.scores[row];
    if (!(score > -INFINITY)) return;
    if (a.finished && a.finished[row]) {
      if (l % a.slices == 0 && skip == 0) {
        s = score;
        tie = (uint64_t)w << 32 | (uint32_t)a.eos;
      }
      return;
    }
    if (skip >= a.count) return;
    const uint64_t k = a.lists[((long long)row * a.slices + l % a.slices) * a.count + skip];
    if (k == 0) return;
    s = (double)score + ((double)beam_value(k) - lse[w]);
    tie = (uint64_t)w << 32 | (uint32_t)beam_token(k);
  };
  double s = -INFINITY;
  uint64_t tie = ~0ull;
  int mine = 0;  // the best head of this thread's lists, and its list
  auto best_of = [&]() {
    s = -INFINITY;
    tie = ~0ull;
    for (int l = t; l < lists; l += 256) {
      double hs;
      uint64_t ht;
      head(l, taken[l], hs, ht);
      if (hs > s || (hs == s && ht < tie)) {
        s = hs;
        tie = ht;
        mine = l;
      }
    }
  };
  best_of();
  for (int n = 0; n < a.count; ++n) {
    double ws = s;
    uint64_t wt = tie;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double os = __shfl_xor(ws, o);
      const uint64_t ot = __shfl_xor((unsigned long long)wt, o);
      if (os > ws || (os == ws && ot < wt)) {
        ws = os;
        wt = ot;
      }
    }
    if (lane == 0) {
      wbest[n & 1][wave] = ws;
      wtie[n & 1][wave] = wt;
    }
    __syncthreads();
    ws = wbest[n & 1][0];
    wt = wtie[n & 1][0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (wbest[n & 1][i] > ws || (wbest[n & 1][i] == ws && wtie[n & 1][i] < wt)) {
        ws = wbest[n & 1][i];
        wt = wtie[n & 1][i];
      }
    const bool none = wt == ~0ull;
    const long long o = (long long)b * a.count + n;
    const int row = row0 + (int)(wt >> 32), token = (int)(uint32_t)wt;
    if (t == 0) {
      a.tokens[o] = none ? -1 : token;
      a.parents[o] = none ? -1 : row;
      a.out_scores[o] = none ? -INFINITY : (float)ws;
      if (a.out_finished) a.out_finished[o] = !none && ((a.finished && a.finished[row]) || token == a.eos);
    }
    if (!none && tie == wt) {  // (a beam and token stand in one list)
      ++taken[mine];
      best_of();
    }
  }
}

// dst row i = src row index[i], `unit` bytes (16, 4 or 1) at a time.
extern "C" __global__ void __launch_bounds__(256) qmm_beam_reorder(const char* src, long long src_rows, long long ld_src,
                                                                   char* dst, long long ld_dst, long long row_bytes,
                                                                   const int32_t* index, int unit) {
  const long long i = blockIdx.x, from = index[i];
  if (from < 0 || from >= src_rows) return;
  const char* s = src + from * ld_src;
  char* d = dst + i * ld_dst;
  const long long n = row_bytes / unit, step = gridDim.y * 256LL;
  for (long long x = blockIdx.y * 256LL + threadIdx.x; x < n; x += step) {
    if (unit == 16)
      ((uint4*)d)[x] = ((const uint4*)s)[x];
    else if (unit == 4)
      ((uint32_t*)d)[x] = ((const uint32_t*)s)[x];
    else
      d[x] = s[x];
  }
}

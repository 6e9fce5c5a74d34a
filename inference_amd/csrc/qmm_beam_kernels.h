// A beam search's selection (qmm_beam_select) and the reordering of what its beams hold.
//
// A continuation's score is beam score + logit - lse, lse = log sum exp(logits of the
// beam). Within a beam the order is the logits', so the first launch takes the largest
// `count` logits of each slice of a beam's row, with the slice's maximum and sum, in one
// pass over the logits; the second joins the slices' sums and takes the best of all lists,
// which are sorted, by their heads.
//
// 16 searches of 8 beams over 128256 bf16 logits, 16 continuations: slices 22.0 us for 32.8 MB (6.1 us at a copy's rate),
// merge 7.7 (medians of a kernel trace). Of the slices' time 6.4 us are the exponentials, 12.5 f64 instructions each at the f32 rate,
// 1.7 the ranking, the rest the first loads and the bound; slices twice as long, whose threads hold 32 logits,
// took 32 us. 4 beams: 5.6 and 5.4 us, all of it latency.
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

// e^x for x <= 0, to 2^-34 of its value (at least e^-700): x = n ln 2 + y, |y| <= ln 2 / 2, n from
// the low bits of a sum with 1.5 2^52, e^y by the polynomial 1 + y q(y) of the seventh degree whose
// largest relative error there is least (4.7e-11; fitted), n added to the exponent's bits. e^0 is 1:
// a token of probability one has the log probability 0, and a beam that takes it ties with one that has ended.
__device__ __forceinline__ double exp_neg(double x) {
  x = fmax(x, -700.0);
  const double t = fma(x, 1.4426950408889634, 6755399441055744.0);
  const double y = fma(t - 6755399441055744.0, -0.6931471805599453, x);
  double r = 0.00019767672511961202;
  r = fma(r, y, 0.0013945897752758946);
  r = fma(r, y, 0.008333568897089748);
  r = fma(r, y, 0.04166627255180138);
  r = fma(r, y, 0.16666665163805036);
  r = fma(r, y, 0.5000000077146097);
  r = fma(r, y, 1.0000000002085943);
  r = fma(r, y, 1.0);
  return __hiloint2double(__double2hiint(r) + (__double2loint(t) << 20), __double2loint(r));
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

// Sum over the 64 lanes of a wave, the same in each: rows of 16 lanes by patterns, then the four
// rows' (a shuffle has ten times the latency).
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  return __hiloint2double(dpp_i<CTRL>(__double2hiint(v)), dpp_i<CTRL>(__double2loint(v)));
}
__device__ __forceinline__ double readlane_d(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp_d<0xb1>(v);
  v += dpp_d<0x4e>(v);
  v += dpp_d<0x141>(v);
  v += dpp_d<0x140>(v);
  return (readlane_d(v, 0) + readlane_d(v, 16)) + (readlane_d(v, 32) + readlane_d(v, 48));
}

// A value as a number whose order is its own, 0 for -inf (no continuation).
__device__ __forceinline__ uint32_t beam_order(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return x == -INFINITY ? 0 : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
// The least value whose number is at or above u (>= 1).
__device__ __forceinline__ float beam_least(uint32_t u) {
  return __builtin_bit_cast(float, u < 0x00800000u ? 0xff7fffffu : u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
// The largest number with zeros behind its first BITS bits that k lanes of the wave are not
// below (0 where k of them have no more): each bit is one comparison and a count of lanes.
template <int BITS>
__device__ __forceinline__ uint32_t wave_bound(uint32_t x, int k) {
  uint32_t p = 0;
#pragma unroll
  for (int b = 31; b >= 32 - BITS; --b) {
    const uint32_t q = p | 1u << b;
    if (__popcll(__ballot(x >= q)) >= k) p = q;
  }
  return p;
}
// A bound that `count` of the workgroup's 256 values pass, from its four waves: a quarter of
// them in each wave, or (ALL) all in one.
template <int BITS, bool ALL>
__device__ __forceinline__ uint32_t block_bound(uint32_t x, int count, uint32_t (*lds)[2]) {
  const int wave = threadIdx.x >> 6;
  const uint32_t part = wave_bound<BITS>(x, (count + 3) / 4), all = ALL && count <= 64 ? wave_bound<BITS>(x, count) : 0;
  if ((threadIdx.x & 63) == 0) {
    lds[wave][0] = part;
    lds[wave][1] = all;
  }
  __syncthreads();
  return max(min(min(lds[0][0], lds[1][0]), min(lds[2][0], lds[3][0])),
             max(max(lds[0][1], lds[1][1]), max(lds[2][1], lds[3][1])));
}
constexpr int kBeamPass = 2048;  // keys that a workgroup can rank: 16 * 128
constexpr int kBeamMany = 512;   // where a closer bound costs less than the ranking

// A slice's maximum, sum of exponentials and `count` largest logits. A thread holds 16 logits;
// a bound that the `count` largest of the threads' maxima pass is one that as many logits of the
// slice pass. A key's place is the number of larger ones among those that do. Where more than
// kBeamMany do (equal logits, a wave without any), the bound is the count-th largest of the threads' largest keys,
// which no two logits share: `count` threads have a key at or above it and no other thread has.
template <int TYPE>
__device__ __forceinline__ void beam_slice(const BeamArgs& a) {
  constexpr int WIDE = TYPE == kTypeF32 ? 4 : 8;  // consecutive logits of a thread (16 bytes)
  __shared__ uint64_t pass[kBeamPass];
  __shared__ uint32_t bounds[4][2];
  __shared__ uint64_t bound;
  __shared__ int passed;
  __shared__ float wmax[4];
  __shared__ double wsum[4];
  const int row = blockIdx.y, sl = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (!beam_live(a, row)) return;
  const int first = sl * kBeamSlice;
  // (a last slice, which is short, is spread over the waves)
  const bool whole = a.wide && first + kBeamSlice <= a.vocab;
  auto token = [&](int i) { return first + (whole ? 256 * WIDE * (i / WIDE) + WIDE * t + i % WIDE : 256 * i + t); };
  float x[16];
  if (whole) {
#pragma unroll
    for (int u = 0; u < 16 / WIDE; ++u) {
      const long long at = row * a.ld + first + 256 * WIDE * u + WIDE * t;
      if constexpr (TYPE == kTypeF32) {
        const float4 v = *(const float4*)((const float*)a.logits + at);
        x[4 * u] = v.x, x[4 * u + 1] = v.y, x[4 * u + 2] = v.z, x[4 * u + 3] = v.w;
      } else {
        const uint4 v = *(const uint4*)((const uint16_t*)a.logits + at);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[8 * u + e] = from_half((uint16_t)(w[e / 2] >> 16 * (e & 1)), TYPE);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = token(i) < a.vocab ? load_typed(a.logits, row * a.ld + token(i), TYPE) : -INFINITY;
  }
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) odd |= !(fabsf(x[i]) < INFINITY);
  if (__any(odd)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = beam_logit(x[i]);
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] += 0.0f;  // (-0 is 0)
    m = fmaxf(m, x[i]);
  }
  const uint32_t mine = beam_order(m);
  m = wave_max(m);
  if (lane == 0) wmax[wave] = m;
  if (t == 0) passed = 0;
  const uint32_t least = max(block_bound<16, false>(mine, a.count, bounds), 1u);
  m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  // the places of a wave's keys, taken at once
  const float low = beam_least(least);
  int n_wave = 0, at = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) n_wave += __popcll(__ballot(x[i] >= low));
  if (lane == 0) at = atomicAdd(&passed, n_wave);
  at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t in = __ballot(x[i] >= low);
    if (in) {
      const int to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
      if (x[i] >= low && to < kBeamPass) pass[to] = beam_key(x[i], token(i));
      at += __popcll(in);
    }
  }
  double z = 0.0;
  if (m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < 16; ++i) z += exp_neg((double)x[i] - (double)m);
  }
  z = wave_sum64(z);
  if (lane == 0) wsum[wave] = z;
  __syncthreads();
  if (__builtin_expect(passed > kBeamMany, 0)) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint64_t k = beam_key(x[i], token(i));
      best = k > best ? k : best;
    }
    __syncthreads();
    pass[t] = best;
    __syncthreads();
    // (threads without a key have the key 0: the lower thread first)
    int place = 0;
    for (int i = 0; i < 256; ++i) place += pass[i] > best || (pass[i] == best && i < t) ? 1 : 0;
    if (place == a.count - 1) bound = best;
    if (t == 0) passed = 0;
    __syncthreads();
    const uint64_t exact = bound ? bound : 1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint64_t k = beam_key(x[i], token(i));
      if (k >= exact) pass[atomicAdd(&passed, 1)] = k;
    }
    __syncthreads();
  }
  const long long slot = (long long)row * a.slices + sl;
  uint64_t* list = a.lists + slot * a.count;
  const int n = passed;
  for (int i0 = 0; i0 < n; i0 += 64) {  // four threads a key
    const int i = i0 + t / 4;
    const uint64_t k = i < n ? pass[i] : 0;
    int place = 0;
#pragma unroll 4
    for (int j = t % 4; j < n; j += 4) place += pass[j] > k;
    place += dpp_i<0xb1>(place);
    place += dpp_i<0x4e>(place);
    if (i < n && t % 4 == 0 && place < a.count) list[place] = k;
  }
  for (int i = n + t; i < a.count; i += 256) list[i] = 0;
  if (t == 0) {
    a.maxima[slot] = m;
    a.sums[slot] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
  }
}

// A continuation: its score, and beam and key, which order equal ones (a beam past all: none).
struct BeamBest {
  double s;
  uint64_t key;
  int beam;
  __device__ __forceinline__ bool before(const BeamBest& o) const {
    return s > o.s || (s == o.s && (beam < o.beam || (beam == o.beam && key > o.key)));
  }
};
constexpr int kBeamNone = 0x7fffffff;
constexpr int kBeamRank = 1024;  // continuations that the merge ranks
}  // namespace qmm

// Grid slices x rows.
extern "C" __global__ void __launch_bounds__(256, 8) qmm_beam_slices_f32(qmm::BeamArgs a) { qmm::beam_slice<qmm::kTypeF32>(a); }
extern "C" __global__ void __launch_bounds__(256, 8) qmm_beam_slices_f16(qmm::BeamArgs a) { qmm::beam_slice<qmm::kTypeF16>(a); }
extern "C" __global__ void __launch_bounds__(256, 8) qmm_beam_slices_bf16(qmm::BeamArgs a) { qmm::beam_slice<qmm::kTypeBF16>(a); }

// One workgroup a search: the beams' lse, then the best of its lists (beams x slices of them,
// list l = beam * slices + slice; a finished beam's first list is its end). A bound that the
// `count` best of the threads' best heads pass is one that as many continuations pass; a
// thread takes what passes from the heads of its lists on, and places are counted as in a
// slice (with a branch on equal scores the launch took 12.6 us, without 7.5: bf16 logits are
// often equal). Where more than kBeamRank pass, the best head is taken `count` times, a dependent
// round each: so it is with fewer lists than `count`, whose heads give no bound (one beam of 32 slices: 64
// continuations 119 us, 128 233).
extern "C" __global__ void __launch_bounds__(256) qmm_beam_merge(qmm::BeamArgs a) {
  using namespace qmm;
  __shared__ double lse[64], total[64];
  __shared__ float score[64];  // -inf: no continuation
  __shared__ int ended[64];
  __shared__ uint32_t bounds[4][2];
  __shared__ int passed;
  __shared__ double pass_s[kBeamRank];
  __shared__ uint64_t pass_key[kBeamRank];
  __shared__ int pass_beam[kBeamRank];
  __shared__ BeamBest wbest[2][4];
  __shared__ uint8_t taken[kBeamMaxLists];  // entries that each list has given
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, row0 = b * a.beams;
  const int lists = a.beams * a.slices;
  // all first loads at once; of beams without a slice's results they are not used
  const uint64_t* all = a.lists + (long long)row0 * a.slices * a.count;
  uint64_t early[4];  // the first entries of this thread's first list
#pragma unroll
  for (int i = 0; i < 4; ++i) early[i] = all[(long long)min(t, lists - 1) * a.count + min(i, a.count - 1)];
  if (t < a.beams) {
    const float s = a.scores[row0 + t];
    score[t] = s == s ? s + 0.0f : -INFINITY;  // (-0 is 0: the bound goes by bits)
    ended[t] = a.finished ? a.finished[row0 + t] : 0;
  }
  if (t == 0) passed = 0;
  for (int w0 = wave; w0 < a.beams; w0 += 16) {  // four beams a wave, their loads together
    float m0[4];
    double z0[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long at = (long long)(row0 + min(w0 + 4 * i, a.beams - 1)) * a.slices + min(lane, a.slices - 1);
      m0[i] = a.maxima[at];
      z0[i] = a.sums[at];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int w = w0 + 4 * i;
      if (w >= a.beams) break;
      const long long at = (long long)(row0 + w) * a.slices;
      if (lane >= a.slices) m0[i] = -INFINITY;
      float m = m0[i];
      for (int j = lane + 64; j < a.slices; j += 64) m = fmaxf(m, a.maxima[at + j]);
      m = wave_max(m);
      double z = m0[i] > -INFINITY ? z0[i] * exp_neg((double)m0[i] - (double)m) : 0.0;
      for (int j = lane + 64; j < a.slices; j += 64)
        if (a.maxima[at + j] > -INFINITY) z += a.sums[at + j] * exp_neg((double)a.maxima[at + j] - (double)m);
      z = wave_sum64(z);
      if (lane == 0) {
        lse[w] = (double)m;
        total[w] = z;
      }
    }
  }
  __syncthreads();
  if (t < a.beams) lse[t] += log(total[t]);
  __syncthreads();
  const BeamBest none = {-INFINITY, 0, kBeamNone};
  // entry `skip` of list l
  auto entry = [&](int l, int skip) {
    const int w = l / a.slices;
    if (!(score[w] > -INFINITY)) return none;
    if (ended[w]) return l % a.slices == 0 && skip == 0 ? BeamBest{score[w], beam_key(0.0f, a.eos), w} : none;
    if (skip >= a.count) return none;
    const uint64_t k = l == t && skip < 4 ? (skip < 2 ? (skip ? early[1] : early[0]) : (skip == 2 ? early[2] : early[3]))
                                          : all[(long long)l * a.count + skip];
    if (k == 0) return none;
    return BeamBest{(double)score[w] + ((double)beam_value(k) - lse[w]), k, w};
  };
  auto put = [&](int n, const BeamBest& x) {
    const bool no = x.beam == kBeamNone;
    const long long o = (long long)b * a.count + n;
    const int token = beam_token(x.key);
    a.tokens[o] = no ? -1 : token;
    a.parents[o] = no ? -1 : row0 + x.beam;
    a.out_scores[o] = no ? -INFINITY : (float)x.s;
    if (a.out_finished) a.out_finished[o] = !no && (ended[x.beam] || token == a.eos);
  };
  // (a rounding to f32 keeps the order, so what passes a bound as f32 holds the best; scores below f32's range are the
  // least of it, not none)
  auto rounded = [&](const BeamBest& x) { return x.beam == kBeamNone ? -INFINITY : fmaxf((float)x.s, -3.402823466e38f); };
  float top = -INFINITY;
  for (int l = t; l < lists; l += 256) top = fmaxf(top, rounded(entry(l, 0)));
  const uint32_t least = max(block_bound<20, true>(beam_order(top), a.count, bounds), 1u);
  if (beam_order(top) >= least)
    for (int l = t; l < lists; l += 256)
      for (int i = 0; i < a.count; ++i) {
        const BeamBest x = entry(l, i);
        if (beam_order(rounded(x)) < least) break;
        const int at = atomicAdd(&passed, 1);
        if (at < kBeamRank) pass_s[at] = x.s, pass_key[at] = x.key, pass_beam[at] = x.beam;
      }
  __syncthreads();
  const int n = passed;
  if (__builtin_expect(n <= kBeamRank, 1)) {
    for (int i0 = 0; i0 < n; i0 += 64) {  // four threads a continuation
      const int i = i0 + t / 4, me = min(i, n - 1);
      const BeamBest x = {pass_s[me], pass_key[me], pass_beam[me]};
      int place = 0;
#pragma unroll 4
      for (int j = t % 4; j < n; j += 4) {
        const BeamBest y = {pass_s[j], pass_key[j], pass_beam[j]};
        const int equal = (y.beam < x.beam) | ((y.beam == x.beam) & (y.key > x.key));
        place += (y.s > x.s) | ((y.s == x.s) & equal);
      }
      place += dpp_i<0xb1>(place);
      place += dpp_i<0x4e>(place);
      if (t % 4 == 0 && i < n && place < a.count) put(place, x);
    }
    for (int i = n + t; i < a.count; i += 256) put(i, none);
    return;
  }
  for (int l = t; l < lists; l += 256) taken[l] = 0;  // (a thread's own lists)
  BeamBest best = none;
  int mine = 0;  // the best head of this thread's lists, and its list
  auto best_of = [&]() {
    best = none;
    for (int l = t; l < lists; l += 256) {
      const BeamBest x = entry(l, taken[l]);
      if (x.before(best)) {
        best = x;
        mine = l;
      }
    }
  };
  best_of();
  for (int i = 0; i < a.count; ++i) {
    BeamBest w = best;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const BeamBest x = {__shfl_xor(w.s, o), (uint64_t)__shfl_xor((unsigned long long)w.key, o), __shfl_xor(w.beam, o)};
      if (x.before(w)) w = x;
    }
    if (lane == 0) wbest[i & 1][wave] = w;
    __syncthreads();
    w = wbest[i & 1][0];
#pragma unroll
    for (int j = 1; j < 4; ++j)
      if (wbest[i & 1][j].before(w)) w = wbest[i & 1][j];
    if (t == 0) put(i, w);
    if (w.beam != kBeamNone && best.beam == w.beam && best.key == w.key) {  // (a beam and token stand in one list)
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

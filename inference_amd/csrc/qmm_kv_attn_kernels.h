// Attention of a step's packed rows over the pages of their sequences (qmm_kv_attention).
//
// Row j of slot s sees the positions t < lens[s] and those lens[s] + i that its mask has:
//   out = sum_t w_t v_t / sum_t w_t,  w_t = e^(scale q . k_t - m),  m the largest score,
// in one pass over the positions with a running m, sum and output.
//
// Per kv head, the G = heads / kv_heads query heads of consecutive rows are columns (column =
// row * G + head) of tiles of N = 32 or 16; positions are taken 32 at a time. With NG = 64 / N
// groups of N lanes (g = lane / N, col = lane % N):
//   S^T = K Q^T      A = N keys, B = the N columns. A column's scores of 32 keys are N / 2
//                    registers of each group: register r is key 4 NG (r / 4) + 4 g + r % 4.
//   O^T += V^T P^T   A = V^T, B = P^T where S^T left it: the k index of a product may be
//                    permuted freely, so V's rows are taken in P's order. Row m of V^T's
//                    tile j is element DTN m + j (DTN = head_dim / N): a lane's values of a
//                    key are DTN contiguous ones (32 j + m where LDS transposes: kv_values_lds).
// K goes straight to LDS (buffer_load ... lds, 16 bytes a lane), its 16-byte chunks XORed by
// the key so that the keys' reads of a chunk meet distinct banks.
//
// One tile of columns (a token of each sequence, small trees): the waves of a workgroup take
// the key tiles of a chunk in turn, each with its own softmax state, and their states are
// joined through LDS. V goes to registers; K of the next tile is in flight from the end of
// the S product on, V of the next from the end of this tile's: a wave has up to two tiles in
// flight and waits for the oldest. More columns: the four waves have a tile of columns each
// and share the keys, K and V through LDS, two tiles deep. A sequence's chunks are joined by a
// second launch.
//
// What bounds them (medians of a kernel trace). 32 heads over 8, head_dim 128: one token of each of 24
// sequences of up to 8000 positions, bf16: K and V's 411 MB, 79.7 us and 5.0 for the join (the bytes alone
// 77 at a copy's rate). One token over 1500 f32 positions: 8.6 and 4.2 us, latency (launch, page ids, K, V,
// join). 8 trees of up to 26 nodes over up to 4000 bf16 positions with f32 rows: 40.4 and 7.4 us, where the
// bytes take 14 and the products, three times over for the parts, 12 at a large product's rate: smaller
// trees fill their tiles in part, waves without a row only load, and a chunk's beginning counts. 4 trees of
// 64 nodes over 30000 f16 positions: 292 and 17 us (248 for both in a row of passes without the trace), the
// products 180 at that rate: of the cycles in which a CU has work the matrix cores are busy in 47% and the
// vector ALUs in 53%, in turn rather than at once (two waves a SIMD are all that the registers and the LDS
// of 64-key tiles leave). A prompt of 2000 rows: 101 us in 16 bits, 489 in f32, the products 30 (45 with the
// weights' parts) and 213; the f32 matrix cores are busy in 66% of those cycles.
//
// Pages. A tile's two halves of 16 positions each lie in one page (pages are 16 or more), so
// a half is one buffer whose end is the last position there is: rows past it read as 0 and
// nothing past it is touched. A wave's lanes hold the page ids of 64 halves at a time.
//
// Types. An f32 cache runs on the f32 matrix cores. A 16-bit cache runs on the 16-bit ones,
// 16 times their rate, with the f32 operand split into parts that each have the cache's
// type. q: all of its bits, but for 2^-23 of an f32 value in the two parts of f16 (QP parts: 3
// of bf16 or 2 of f16 for f32, 2 of bf16 for f16, else 1). The weights, in PP parts: 3 of bf16
// for f32 rows lose 2^-24 of a weight; 2 of f16 lose up to 2^-21, toward zero; 2 of bf16 for
// 16-bit rows lose 2^-16, where the output's own rounding is 2^-8 (bf16) or 2^-11: about one bf16
// output in 500 is rounded the other way for it (as is one in 2000 by the order of f32 sums), and
// the third part would cost half as many products again. For f16, whose range is small, a
// column's q is scaled by a power of two to [2^13, 2^14) and the weights by 2^12, which divides out.
//
// What a column does not see has the score -inf and the weight 0, but 0 times an infinity or
// a NaN of such a value row is NaN, as is a split infinity: a workgroup whose state is not
// finite computes its chunk again, column by column and position by position, with what the
// column sees alone.
#pragma once

#include <type_traits>

#include "qmm_kv_common.h"

namespace qmm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
// Scores are held as the products q . k and c = |scale| log2 e (a column's; a negative scale
// turns q's sign), weights as 2^(c x - c m): one fma, the rounding of c m common to every weight
// of a state, whose reference c m (rounded) is what states are joined by. From |c m| = 2^24 on
// that rounding alone would over- or underflow 2^x, so there the difference is taken first.
constexpr float kBigRef = 16777216.0f;
// of a state with the reference m; 0 for -inf
__device__ __forceinline__ float state_weight(float m, float most) {
  return __builtin_amdgcn_exp2f(m - (most == -INFINITY ? 0.0f : most));
}
__device__ __forceinline__ float finite(float x) { return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f); }

// Over the lanes l, l + N, ... of a wave (each receives it).
template <int N>
__device__ __forceinline__ float groups_max(float x) {
  if constexpr (N == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int N>
__device__ __forceinline__ float groups_sum(float x) {
  if constexpr (N == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct KvAttn {
  KvCache c;
  KvRows r;
  const void* q;
  const uint64_t* masks;
  void* out;
  float *part, *state;  // [rows][heads][splits] records: head_dim floats; reference and sum
  long long ldq, ldm, ldo;
  int layer, x_type, heads, wide, out_wide, splits, chunk;
  int tiles, group_rows;  // groups of a slot's rows that a workgroup takes, rows of one
  int join_lanes;
  float scale;
};

// Whether row j (packed row `row`) of a step sees the step's row i.
__device__ __forceinline__ bool kv_sees(const KvAttn& a, int row, int j, int i) {
  if (!a.masks) return i <= j;
  return i >> 6 < a.ldm && (a.masks[(long long)row * a.ldm + (i >> 6)] >> (i & 63) & 1);
}
// The 32 bits of a row's mask from bit `i` (>= 0) on.
__device__ __forceinline__ uint32_t kv_mask_bits(const KvAttn& a, int row, int i) {
  const uint32_t* w = (const uint32_t*)(a.masks + (long long)row * a.ldm);
  const long long n = 2 * a.ldm, x = i >> 5;
  const uint32_t lo = x < n ? w[x] : 0, hi = x + 1 < n ? w[x + 1] : 0;
  return (uint32_t)(((uint64_t)hi << 32 | lo) >> (i & 31));
}

// Positions that any row of the group at row i0 (nrow rows) of a slot sees, and the length of
// the chunks they are split into: `chunk`, or a split's share where that is more.
struct KvTile {
  int base, n, nrow, len;
};
__device__ __forceinline__ KvTile kv_tile(const KvAttn& a, const KvSpan& sp, int s, int i0) {
  KvTile t;
  t.base = a.c.length(s);
  t.nrow = min(a.group_rows, sp.n - i0);
  t.n = min(t.base + (a.masks ? sp.n : i0 + t.nrow), a.c.capacity());
  t.len = max(a.chunk, ((t.n + a.splits - 1) / a.splits + 127) / 128 * 128);
  return t;
}

// One column's share of positions [k0, k1), a position at a time: what the tiles have to give.
// The wave's lanes hold head_dim / 64 values each.
template <int R>
__device__ __forceinline__ void kv_column(const KvAttn& a, int s, int row, int j, int h, int base, int k0, int k1,
                                          float (&o)[R], float& m, float& l) {
  const int lane = threadIdx.x & 63, g = h / (a.heads / a.c.kv_heads), dim = 64 * R;
  float q[R];
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < R; ++e) {
    q[e] = load_typed(a.q, row * a.ldq + (long long)h * dim + R * lane + e, a.x_type);
    o[e] = 0.0f;
  }
#pragma unroll 1
  for (int t = k0; t < k1; ++t) {
    if (t >= base && !kv_sees(a, row, j, t - base)) continue;
    const int p = a.c.page(s, t >> a.c.page_log);
    float d = 0.0f, v[R];
    if (p < 0) {
      d = NAN;
#pragma unroll
      for (int e = 0; e < R; ++e) v[e] = NAN;
    } else {
      const long long at = a.c.row(a.layer, p, g, t & ((1 << a.c.page_log) - 1)) + R * lane;
#pragma unroll
      for (int e = 0; e < R; ++e) d += q[e] * load_typed(a.c.k, at + e, a.c.dtype);
#pragma unroll
      for (int e = 0; e < R; ++e) v[e] = load_typed(a.c.v, at + e, a.c.dtype);
      d = wave_sum(d) * a.scale;
    }
    const float mx = fmaxf(m, d);
    const float x = mx == -INFINITY ? 0.0f : expf(m - mx), w = d == -INFINITY ? 0.0f : expf(d - mx);
    m = mx;
    l = l * x + w;
#pragma unroll
    for (int e = 0; e < R; ++e) o[e] = o[e] * x + w * v[e];
  }
}

// f32 pairs as two 16-bit values, rounded to nearest (bf16) or toward zero (f16: one
// instruction; the next part takes up what it left), and what a pair leaves.
template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (TYPE == kTypeF16) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
  }
}
template <int TYPE>
__device__ __forceinline__ float low_of(uint32_t w) {
  return TYPE == kTypeF16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)w) : __builtin_bit_cast(float, w << 16);
}
template <int TYPE>
__device__ __forceinline__ float high_of(uint32_t w) {
  return TYPE == kTypeF16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)) : __builtin_bit_cast(float, w & 0xffff0000u);
}
// What a cache type, a head size and a tile of N columns fix.
template <int TYPE_, int DIM, int N_>
struct KvShape {
  static constexpr int TYPE = TYPE_, dim = DIM, N = N_;
  static constexpr bool F32 = TYPE == kTypeF32;
  static constexpr int EB = F32 ? 4 : 2, RB = dim * EB;  // bytes of a value and of a row
  static constexpr int CH = RB / 16, RPL = 64 / CH;      // 16-byte chunks of a row, rows of a load to LDS
  static constexpr int SH = RB == 128 ? 1 : 0;           // (two rows of 128 bytes fill the banks once)
  static constexpr int RLOG = RB == 128 ? 7 : RB == 256 ? 8 : RB == 512 ? 9 : 10;
  static constexpr int KB = 32 * RB;                     // bytes of 32 rows
  static constexpr int NG = 64 / N, STEPS = CH / NG;     // lane groups; chunks of a row that a lane has
  static constexpr int SUB = 32 / N, NR = N / 2;         // S products of 32 keys; their score registers
  static constexpr int DTN = dim / N, AR = N * N / 64;   // V^T tiles; registers of one
  static constexpr int GRP = NR / 8;                     // groups of eight score registers
  typedef float Acc __attribute__((ext_vector_type(AR)));
  struct VRow {
    uint32_t w[DTN * EB / 4];
  };
  // row of a result register
  static __device__ __forceinline__ int out_row(int r, int g) { return 4 * NG * (r >> 2) + 4 * g + (r & 3); }
  // key of score register r
  static __device__ __forceinline__ int key(int r, int g) { return 4 * NG * (r >> 2) + 4 * g + (r & 3); }
};

template <class S>
__device__ __forceinline__ typename S::Acc mfma_f32(float a, float b, typename S::Acc c) {
  if constexpr (S::N == 32)
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <class S>
__device__ __forceinline__ typename S::Acc mfma_16(u32x4 a, u32x4 b, typename S::Acc c) {
  if constexpr (S::TYPE == kTypeF16 && S::N == 32)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else if constexpr (S::TYPE == kTypeF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else if constexpr (S::N == 32)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The q of a lane's column (packed row, head): chunks NG c + g, in parts of the cache's type.
// Returns the column's c.
template <class S, int QP>
__device__ __forceinline__ float kv_load_q(const KvAttn& a, int row, int head, int g, u32x4 (&w)[QP][S::STEPS]) {
  constexpr int E = 16 / S::EB;  // values of a chunk
  float x[S::STEPS][E];
  const long long at = row * a.ldq + (long long)head * S::dim;
  // (a branch a type and boundary, all loads in each: in flight together)
  auto load = [&](auto bytes, auto wide) {
    constexpr int B = decltype(bytes)::value;
#pragma unroll
    for (int c = 0; c < S::STEPS; ++c)
#pragma unroll
      for (int y = 0; y < E / 4; ++y) {
        float f[4];
        load4_typed(f, a.q, at + E * (S::NG * c + g) + 4 * y, B == 4 ? kTypeF32 : a.x_type, decltype(wide)::value);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[c][4 * y + e] = f[e];
      }
  };
  const std::integral_constant<int, 4> four;
  const std::integral_constant<int, 2> two;
  if (a.x_type == kTypeF32)
    a.wide ? load(four, std::true_type()) : load(four, std::false_type());
  else
    a.wide ? load(two, std::true_type()) : load(two, std::false_type());
  if (a.scale <= 0.0f) {  // (c = 0 would make NaN of the scores that are -inf: equal weights are products of zeros)
    const float turn = a.scale < 0.0f ? -1.0f : 0.0f;
#pragma unroll
    for (int c = 0; c < S::STEPS; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) x[c][e] *= turn;
  }
  float down = 1.0f;
  if constexpr (S::TYPE == kTypeF16) {
    float most = 0.0f;
#pragma unroll
    for (int c = 0; c < S::STEPS; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) most = fmaxf(most, fabsf(x[c][e]));
    most = groups_max<S::N>(most);
    int up = 0;
    if (most > 0.0f && most < INFINITY) up = min(max(14 - __builtin_amdgcn_frexp_expf(most), -100), 100);
    down = __builtin_ldexpf(1.0f, -up);
#pragma unroll
    for (int c = 0; c < S::STEPS; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) x[c][e] = __builtin_ldexpf(x[c][e], up);
  }
#pragma unroll
  for (int c = 0; c < S::STEPS; ++c) {
    if constexpr (S::F32) {
      w[0][c] = u32x4{__float_as_uint(x[c][0]), __float_as_uint(x[c][1]), __float_as_uint(x[c][2]), __float_as_uint(x[c][3])};
    } else {
#pragma unroll
      for (int p = 0; p < QP; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b = (uint32_t)to_half(x[c][2 * e], S::TYPE) | (uint32_t)to_half(x[c][2 * e + 1], S::TYPE) << 16;
          w[p][c][e] = b;
          x[c][2 * e] -= low_of<S::TYPE>(b);
          x[c][2 * e + 1] -= high_of<S::TYPE>(b);
        }
    }
  }
  return a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e * down;
}

// q where a workgroup keeps it: in registers, or in LDS (chunk c of part p of every lane).
template <class S, int QP>
struct KvQRegs {
  u32x4 w[QP][S::STEPS];
  __device__ __forceinline__ u32x4 get(int p, int c) const { return w[p][c]; }
};
template <class S, int QP>
struct KvQLds {
  const char* at;  // this lane's
  __device__ __forceinline__ u32x4 get(int p, int c) const { return *(const u32x4*)(at + (p * S::STEPS + c) * 1024); }
};

// The scores of 32 keys in LDS at kb, before the scale.
template <class S, int QP, class Q>
__device__ __forceinline__ void kv_scores(float (&sc)[S::NR], const char* kb, const Q& q, int col, int g) {
#pragma unroll
  for (int sub = 0; sub < S::SUB; ++sub) {
    // (chunk NG c + g is an XOR away from chunk g; the asm keeps the addresses from being hoisted into a register each)
    const int row = S::N * sub + col;
    unsigned at = (unsigned)row * S::RB + 16u * ((unsigned)g ^ ((unsigned)(row >> S::SH) & (S::CH - 1)));
    asm volatile("" : "+v"(at));
    auto chunk = [&](int c) { return *(const u32x4*)(kb + (at ^ (16u * S::NG * c))); };
    typename S::Acc s;
    if constexpr (S::F32) {
      // eight chains of roundings, each an eighth of the sum: two at a time
      constexpr int Q4 = S::STEPS / 4;
      u32x4 ka = chunk(0), qa = q.get(0, 0);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        typename S::Acc c2[2] = {(typename S::Acc)(0.0f), (typename S::Acc)(0.0f)};
#pragma unroll
        for (int c = y * Q4; c < (y + 1) * Q4; ++c) {  // the next chunks' reads fly under this one's products
          const int nx = c + 1 < S::STEPS ? c + 1 : c;
          const u32x4 kn = chunk(nx), qn = q.get(0, nx);
#pragma unroll
          for (int e = 0; e < 4; ++e) c2[e & 1] = mfma_f32<S>(__uint_as_float(ka[e]), __uint_as_float(qa[e]), c2[e & 1]);
          __builtin_amdgcn_sched_barrier(0);
          ka = kn;
          qa = qn;
        }
        s = y == 0 ? c2[0] + c2[1] : s + (c2[0] + c2[1]);
        asm volatile("" : "+v"(s));  // (added here: all four pairs of chains at once do not fit the registers)
      }
    } else {
      // one chain; of q's parts the smallest first
      s = (typename S::Acc)(0.0f);
#pragma unroll
      for (int c = 0; c < S::STEPS; ++c) {
        const u32x4 ka = chunk(c);
#pragma unroll
        for (int p = QP - 1; p >= 0; --p) s = mfma_16<S>(ka, q.get(p, c), s);
      }
    }
#pragma unroll
    for (int r = 0; r < S::AR; ++r) sc[S::AR * sub + r] = s[r];
  }
}

// A column's running softmax: largest product, the reference c m (0 while it is -inf), this
// lane's part of the sum.
struct KvState {
  float m = -INFINITY, ml = 0.0f, l = 0.0f;
  __device__ __forceinline__ float ref() const { return m == -INFINITY ? m : ml; }
};

// The bits of the 32 keys from t0 on that row j sees, none from position k1 on.
__device__ __forceinline__ uint32_t kv_visible(const KvAttn& a, int row, int j, int base, int t0, int k1) {
  uint32_t see;
  if (a.masks) {
    const int rel = t0 - base;
    see = rel >= 0 ? kv_mask_bits(a, row, rel) : rel <= -32 ? ~0u : kv_mask_bits(a, row, 0) << -rel | ((1u << -rel) - 1);
  } else {
    const int c = base + j + 1 - t0;
    see = c >= 32 ? ~0u : c <= 0 ? 0 : (1u << c) - 1;
  }
  return k1 - t0 < 32 ? see & ((1u << max(k1 - t0, 0)) - 1) : see;
}

// NS products to weights; returns the factor of what there was.
template <class S, int NS>
__device__ __forceinline__ float kv_softmax(float (&sc)[NS], KvState& st, float c) {
  constexpr float kUp = S::TYPE == kTypeF16 ? 12.0f : 0.0f;
  float x[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
  for (int r = 4; r < NS; ++r) x[r & 3] = fmaxf(x[r & 3], sc[r]);
  const float mx = fmaxf(st.m, groups_max<S::N>(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))));
  const float ml = mx == -INFINITY ? 0.0f : mx * c;
  float w;
  if (__builtin_expect(__any(!(fabsf(ml) < kBigRef)), 0)) {  // (see kBigRef)
    const float off = mx == -INFINITY ? 0.0f : mx;
    w = __builtin_amdgcn_exp2f((st.m - off) * c);
#pragma unroll
    for (int r = 0; r < NS; ++r) sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r] - off, c, kUp));
  } else {
    w = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.ml - ml);
#pragma unroll
    for (int r = 0; r < NS; ++r) sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], c, kUp - ml));
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = sc[r];
#pragma unroll
  for (int r = 4; r < NS; ++r) x[r & 3] += sc[r];
  st.l = st.l * w + ((x[0] + x[1]) + (x[2] + x[3]));
  st.m = mx;
  st.ml = finite(ml);
  return w;
}

// Eight weights as the parts of a product's operand.
template <class S, int PP>
__device__ __forceinline__ void kv_parts(u32x4 (&p)[PP], const float* sc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = sc[2 * e], y = sc[2 * e + 1];
#pragma unroll
    for (int q = 0; q < PP; ++q) {
      p[q][e] = pack2<S::TYPE>(x, y);
      x -= low_of<S::TYPE>(p[q][e]);
      y -= high_of<S::TYPE>(p[q][e]);
    }
  }
}
// acc += V^T P^T of eight score registers and their keys' value rows; f32: acc times w first
// (16-bit caches: kv_rescale).
template <class S, int PP>
__device__ __forceinline__ void kv_values(typename S::Acc (&acc)[S::DTN], const float* sc, const typename S::VRow (&v)[8],
                                          float w) {
  if constexpr (S::F32) {
    // these keys' products are summed on their own and added to the running sum once
    typename S::Acc o[2];
#pragma unroll
    for (int d = 0; d <= S::DTN; ++d) {
      if (d < S::DTN) {
        o[d & 1] = (typename S::Acc)(0.0f);
#pragma unroll
        for (int r = 0; r < 8; ++r) o[d & 1] = mfma_f32<S>(__uint_as_float(v[r].w[d]), sc[r], o[d & 1]);
      }
      if (d > 0) {  // added while the next products run
#pragma unroll
        for (int r = 0; r < S::AR; ++r) acc[d - 1][r] = __builtin_fmaf(acc[d - 1][r], w, o[(d - 1) & 1][r]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    u32x4 p[PP];
    kv_parts<S, PP>(p, sc);
#pragma unroll
    for (int d = 0; d < S::DTN; ++d) {
      u32x4 vt;  // eight keys' value d of this lane
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vt[e] = __builtin_amdgcn_perm(v[2 * e + 1].w[d / 2], v[2 * e].w[d / 2], d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int q = PP - 1; q >= 0; --q) acc[d] = mfma_16<S>(vt, p[q], acc[d]);
    }
  }
}
// The same with 16-bit V rows in LDS, transposed as they are read: 16 lanes read 16 values of four
// rows, four values each, and lane i of them gets value i of the four. Row m of V^T's tile j is
// element 32 j + m here. `at`: this lane's place in the tile of 16 keys, of tile 0. (Rows read as
// they lie and interleaved by permutations: 4 trees of 64 nodes over 30000 positions 276 us, this 266.)
__device__ __forceinline__ u32x2 read_transposed(const char* lds) {
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)lds));
}
template <class S, int PP>
__device__ __forceinline__ void kv_values_lds(typename S::Acc (&acc)[S::DTN], const float* sc, const char* vb, unsigned at) {
  u32x4 p[PP];
  kv_parts<S, PP>(p, sc);
#pragma unroll
  for (int d = 0; d < S::DTN; ++d) {
    const char* v = vb + (at ^ (64u * d));
    const u32x2 x = read_transposed(v), y = read_transposed(v + 8 * S::RB);
    const u32x4 vt = {x[0], x[1], y[0], y[1]};
#pragma unroll
    for (int q = PP - 1; q >= 0; --q) acc[d] = mfma_16<S>(vt, p[q], acc[d]);
  }
}
template <class S>
__device__ __forceinline__ void kv_rescale(typename S::Acc (&acc)[S::DTN], float w) {
  if constexpr (!S::F32) {
    if (__all(w == 1.0f)) return;
#pragma unroll
    for (int d = 0; d < S::DTN; ++d)
#pragma unroll
      for (int r = 0; r < S::AR; ++r) acc[d][r] *= w;
  }
}
// Whether a wave's sums are all finite.
template <class S>
__device__ __forceinline__ bool kv_finite(const typename S::Acc (&acc)[S::DTN], float l) {
  float z = l * 0.0f;
#pragma unroll
  for (int d = 0; d < S::DTN; ++d)
#pragma unroll
    for (int r = 0; r < S::AR; ++r) z = __builtin_fmaf(acc[d][r], 0.0f, z);
  return !__any(z != 0.0f);  // (0 * inf and 0 * NaN are NaN)
}

// The unit of a workgroup: slot, chunk, kv head; its positions and its group of rows. A unit's
// groups follow each other on one XCD, which then has the unit's keys in its L2: workgroups
// are dealt to the eight of them in turn.
struct KvUnit {
  KvSpan sp;
  KvTile tl;
  int s, g, chunk, i0, k0, k1;
  bool any;
  // bytes from a pool's start to the kv head's rows in page 0 of the layer, and from page to page
  long long first;
  unsigned step;
};
__device__ __forceinline__ KvUnit kv_unit(const KvAttn& a) {
  KvUnit u;
  u.any = false;
  const unsigned id = blockIdx.x, kv = a.c.kv_heads;
  const int group = (int)((id >> 3) % (unsigned)a.tiles);
  const unsigned unit = (id >> 3) / (unsigned)a.tiles * 8 + (id & 7);
  if (unit >= (unsigned)a.c.slots * (unsigned)a.splits * kv) return u;
  u.g = (int)(unit % kv), u.chunk = (int)(unit / kv % (unsigned)a.splits), u.s = (int)(unit / kv / (unsigned)a.splits);
  u.sp = kv_span(a.r, u.s);
  u.i0 = group * a.group_rows;
  if (u.i0 >= u.sp.n) return u;
  u.tl = kv_tile(a, u.sp, u.s, u.i0);
  const long long start = (long long)u.chunk * u.tl.len;
  if (start >= u.tl.n) return u;
  u.k0 = (int)start, u.k1 = min(u.k0 + u.tl.len, u.tl.n);
  u.first = a.c.row(a.layer, 0, u.g, 0) << a.c.esize_log();
  u.step = (unsigned)(a.c.kv_heads * a.c.head_dim << a.c.page_log << a.c.esize_log());  // (2^28 at most)
  u.any = true;
  return u;
}

// Key tiles of a wave, of H halves of 16 positions each: tile i at k0 + first + step i. Lane l
// holds the page id of the half l % H of tile l / H of a block of 64 / H.
template <int H>
struct KvPages {
  int ids;
  int first, step;
  static constexpr int BLOCK = 64 / H;
  __device__ __forceinline__ void load(const KvAttn& a, const KvUnit& u, int i) {
    const int lane = threadIdx.x & 63;
    const long long pos = u.k0 + first + (long long)step * (i + lane / H) + 16 * (lane % H);
    ids = pos < u.k1 ? a.c.page(u.s, (int)pos >> a.c.page_log) : -1;
  }
  // half x of tile i: where it begins, how many rows it has (0 without a page), bytes from a pool's start
  __device__ __forceinline__ long long at(const KvAttn& a, const KvUnit& u, int i, int x, int row_log, int& rows) const {
    const int pos = __builtin_amdgcn_readfirstlane(u.k0 + first + step * i + 16 * x);
    const int p = __builtin_amdgcn_readlane(ids, __builtin_amdgcn_readfirstlane(H * (i % BLOCK) + x));
    rows = p < 0 ? 0 : min(max(u.k1 - pos, 0), 16);
    return u.first + (long long)((unsigned long long)(unsigned)max(p, 0) * u.step) + ((long long)(pos & ((1 << a.c.page_log) - 1)) << row_log);
  }
  // whether tile i has a position without a page
  __device__ __forceinline__ bool missing(const KvUnit& u, int i) const {
    const int lane = threadIdx.x & 63;
    return __any(lane / H == i % BLOCK && ids < 0 && u.k0 + first + (long long)step * i + 16 * (lane % H) < u.k1);
  }
};
// A half as a buffer that ends at the last position.
template <class S>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv_buffer(void* pool, long long at, int rows) {
  return __builtin_amdgcn_make_buffer_rsrc((char*)pool + at, 0, __builtin_amdgcn_readfirstlane(rows * S::RB), 0x00020000);
}
// Loads to LDS are 64 chunks, RPL rows; chunk c of row r goes to slot c ^ (r >> SH) % CH (K), c (V
// in 32 bits), or c ^ 2 ((r >> SH) % min(8, CH / 2)) (V in 16: the four rows of a transposed read, 32 bytes each, in
// banks of their own). A lane's byte offset in its load of K, of the rows from `row` on (a multiple of 8), of
// which the load's own rows take an XOR and an addition.
template <class S>
__device__ __forceinline__ unsigned kv_k_lane(int row) {
  const int lane = threadIdx.x & 63, r = row + lane / S::CH;
  return (unsigned)(r & 15) * S::RB + 16u * ((unsigned)(lane % S::CH) ^ ((unsigned)(r >> S::SH) & (S::CH - 1)));
}
template <class S>
__device__ __forceinline__ unsigned kv_k_load(unsigned lane, int x, int half = 0) {  // x: load within 16 rows of `half`
  return (lane ^ (16u * ((unsigned)((16 * half + S::RPL * x) >> S::SH) & (S::CH - 1)))) + 1024u * x;
}
template <class S>
__device__ __forceinline__ unsigned kv_v_swap(int row) {
  return S::F32 ? 0 : 2u * ((unsigned)(row >> S::SH) & (S::CH >= 16 ? 7 : S::CH / 2 - 1));
}
template <class S>
__device__ __forceinline__ unsigned kv_v_lane(int row) {
  const int lane = threadIdx.x & 63, r = row + lane / S::CH;
  return (unsigned)(r & 15) * S::RB + 16u * ((unsigned)(lane % S::CH) ^ kv_v_swap<S>(r));
}
template <class S>
__device__ __forceinline__ unsigned kv_v_load(unsigned lane, int x) {
  return (lane ^ (16u * kv_v_swap<S>(S::RPL * x))) + 1024u * x;
}
__device__ __forceinline__ void kv_to_lds(__amdgpu_buffer_rsrc_t rs, unsigned at, char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)to, 16, at, 0, 0, 0);
}

// A column's result, or its record where there are several chunks.
template <class S>
__device__ __forceinline__ long long kv_record(const KvAttn& a, const KvUnit& u, int row, int head) {
  return ((long long)row * a.heads + head) * a.splits + u.chunk;
}

// The columns c of `count` (packed row row0 + c / G) again, position by position (see above).
template <class S>
__device__ __forceinline__ void kv_again(const KvAttn& a, const KvUnit& u, int j0, int count, int first, int step) {
  constexpr int R = S::dim / 64;
  const int lane = threadIdx.x & 63, G = a.heads / a.c.kv_heads;
  const bool whole = u.tl.len >= u.tl.n;
#pragma unroll 1
  for (int c = first; c < count; c += step) {
    float o[R], m, l;
    const int j = j0 + c / G, r = u.sp.first + j, h = u.g * G + c % G;
    kv_column<R>(a, u.s, r, j, h, u.tl.base, u.k0, u.k1, o, m, l);
    if (whole) {
#pragma unroll
      for (int e = 0; e < R; ++e)
        store_typed(a.out, r * a.ldo + (long long)h * S::dim + R * lane + e, a.x_type, l == 0.0f ? 0.0f : o[e] / l);
    } else {
      const long long rec = kv_record<S>(a, u, r, h);
      const float up = S::TYPE == kTypeF16 ? 4096.0f : 1.0f;  // (as the tiles' weights)
#pragma unroll
      for (int e = 0; e < R; ++e) a.part[rec * S::dim + R * lane + e] = o[e] * up;
      if (lane == 0) {
        // (scores that are all NaN have the maximum -inf, and a sum that must not be left out)
        a.state[2 * rec] = m == -INFINITY ? (l != 0.0f ? 0.0f : m) : finite(m * kLog2e);
        a.state[2 * rec + 1] = l * up;
      }
    }
  }
}

// One tile of columns: the waves take the key tiles in turn.
template <int TYPE, int DIM, int N, int QP, int PP>
__device__ __forceinline__ void kv_attn_narrow(const KvAttn& a) {
  typedef KvShape<TYPE, DIM, N> S;
  constexpr int NW = S::F32 && DIM == 256 ? 2 : 4;  // waves (K tiles of f32 rows of 256: 32 KB each)
  constexpr int HJ = N == 16 || S::DTN < 4 ? S::DTN : 4;  // V^T tiles joined at a time
  constexpr int JOIN = NW * N * N * HJ * 4;
  constexpr bool QLDS = N == 32 && (S::F32 || QP > 1);
  constexpr int QB = QLDS ? QP * S::STEPS * 1024 : 0;
  constexpr int ST = NW * N * 2 * 4 + 64;
  constexpr int LDS = NW * S::KB + QB > JOIN + ST ? NW * S::KB + QB : JOIN + ST;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int g = lane / N, col = lane % N, G = a.heads / a.c.kv_heads;
  const KvUnit u = kv_unit(a);
  if (!u.any) return;
  const int pi = min(col / G, u.tl.nrow - 1);  // columns past the rows repeat the last row; they are not stored
  const int j = u.i0 + pi, row = u.sp.first + j, head = u.g * G + col % G;

  KvPages<2> pg;
  pg.first = 32 * wave, pg.step = 32 * NW;
  pg.load(a, u, 0);
  char* kb = lds + wave * S::KB;
  bool missing;
  __amdgpu_buffer_rsrc_t v0, v1;  // V's halves of the tile that is in flight or in registers
  unsigned klane = kv_k_lane<S>(0), vlane = (unsigned)(4 * g) * S::RB + (unsigned)(S::DTN * S::EB) * col;
  auto load_k = [&](int i) {
    asm volatile("" : "+v"(klane));
    missing = pg.missing(u, i);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int rows;
      const long long at = pg.at(a, u, i, h, S::RLOG, rows);
      const auto rs = kv_buffer<S>(a.c.k, at, rows);
#pragma unroll
      for (int x = 0; x < 16 / S::RPL; ++x) kv_to_lds(rs, kv_k_load<S>(klane, x, h), kb + 1024 * (16 / S::RPL * h + x));
      (h ? v1 : v0) = kv_buffer<S>(a.c.v, at, rows);
    }
  };
  typename S::VRow v[S::GRP][8];
  // f32 rows of 128 and more on tiles of 32 columns: V's second group of rows is loaded behind the S product, which
  // needs the room
  constexpr int EARLY = S::F32 && N == 32 && DIM >= 128 ? 1 : S::GRP;
  auto load_v = [&](auto from, auto to) {
    asm volatile("" : "+v"(vlane));
#pragma unroll
    for (int q = decltype(from)::value; q < decltype(to)::value; ++q)
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        constexpr int B = S::DTN * S::EB;  // bytes of a lane
        const unsigned at = vlane + (unsigned)(S::key(8 * q + r, 0) & 15) * S::RB;
        const auto rs = (8 * q + r) / (S::NR / 2) == 0 ? v0 : v1;
        if constexpr (B == 4) {
          v[q][r].w[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0);
        } else if constexpr (B == 8) {
          const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0));
          v[q][r].w[0] = x[0], v[q][r].w[1] = x[1];
        } else {
#pragma unroll
          for (int y = 0; y < B / 16; ++y) {
            const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + 16 * y, 0, 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][r].w[4 * y + e] = x[e];
          }
        }
      }
  };
  const std::integral_constant<int, 0> v_first;
  const std::integral_constant<int, EARLY> v_early;
  const std::integral_constant<int, S::GRP> v_last;
  constexpr int VLOADS = EARLY * 8 * (S::DTN * S::EB > 16 ? S::DTN * S::EB / 16 : 1);  // early loads of V
  static_assert(VLOADS < 64, "vmcnt");
  load_k(0);
  __builtin_amdgcn_sched_barrier(0);
  u32x4 qw[QP][S::STEPS];
  const float c = kv_load_q<S, QP>(a, row, head, g, qw);
  __builtin_amdgcn_sched_barrier(0);
  load_v(v_first, v_early);
  __builtin_amdgcn_sched_barrier(0);
  std::conditional_t<QLDS, KvQLds<S, QP>, KvQRegs<S, QP>> q;
  if constexpr (QLDS) {
    char* qb = lds + NW * S::KB + 16 * lane;
#pragma unroll
    for (int c = 0; c < S::STEPS; ++c)
      if (c % NW == wave) {
#pragma unroll
        for (int p = 0; p < QP; ++p) *(u32x4*)(qb + (p * S::STEPS + c) * 1024) = qw[p][c];
      }
    q.at = qb;
    __syncthreads();
  } else {
#pragma unroll
    for (int p = 0; p < QP; ++p)
#pragma unroll
      for (int c = 0; c < S::STEPS; ++c) q.w[p][c] = qw[p][c];
  }

  typename S::Acc acc[S::DTN];
#pragma unroll
  for (int d = 0; d < S::DTN; ++d) acc[d] = (typename S::Acc)(0.0f);
  KvState st;
#pragma unroll 1
  for (int i = 0; u.k0 + pg.first + pg.step * i < u.k1; ++i) {
    const int t0 = u.k0 + pg.first + pg.step * i;
    const bool poison = missing;
    // K is in LDS once no loads but V's are out (vmcnt's bits 0-3 and 14-15)
    __builtin_amdgcn_s_waitcnt(0x0f70 | (VLOADS & 15) | (VLOADS >> 4) << 14);
    __builtin_amdgcn_sched_barrier(0);
    float sc[S::NR];
    kv_scores<S, QP>(sc, kb, q, col, g);
    __builtin_amdgcn_sched_barrier(0);
    // every lane's reads of the K tile are consumed: the next may overwrite it. Unconditional (past the end the
    // buffers are empty): under a condition the waits for V would have to assume it was not issued.
    load_v(v_early, v_last);
    if ((i + 1) % pg.BLOCK == 0) pg.load(a, u, i + 1);
    load_k(i + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (__builtin_expect(poison, 0)) {
#pragma unroll
      for (int r = 0; r < S::NR; ++r) sc[r] = NAN;
    }
    if (t0 + 32 > u.tl.base || t0 + 32 > u.k1) {
      const uint32_t see = kv_visible(a, row, j, u.tl.base, t0, u.k1);
#pragma unroll
      for (int r = 0; r < S::NR; ++r)
        if (!(see >> S::key(r, g) & 1)) sc[r] = -INFINITY;
    }
    const float w = kv_softmax<S>(sc, st, c);
    kv_rescale<S>(acc, w);
#pragma unroll
    for (int x = 0; x < S::GRP; ++x) kv_values<S, PP>(acc, sc + 8 * x, v[x], x == 0 ? w : 1.0f);
    __builtin_amdgcn_sched_barrier(0);
    load_v(v_first, v_early);
    __builtin_amdgcn_sched_barrier(0);
  }

  // ---- the waves' states
  const bool bad = !kv_finite<S>(acc, st.l);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): no K load may land on what follows
  __syncthreads();
  float(*sv)[2][N] = (float(*)[2][N])(lds + JOIN);
  int* sbad = (int*)(lds + JOIN + NW * N * 2 * 4);
  const float l = groups_sum<N>(st.l);
  if (g == 0) {
    sv[wave][0][col] = st.ref();
    sv[wave][1][col] = l;
  }
  if (lane == 0) sbad[wave] = bad;
  const bool whole = u.tl.len >= u.tl.n;  // one chunk: the result itself
  const int count = G * u.tl.nrow;
  int any = 0;
#pragma unroll
  for (int jp = 0; jp < S::DTN / HJ; ++jp) {
    if (jp) __syncthreads();  // (the last part is read)
    float* ob = (float*)lds + wave * N * N * HJ;
    if (col < count) {
#pragma unroll
      for (int r = 0; r < S::AR; ++r)
#pragma unroll
        for (int d = 0; d < HJ; ++d) ob[(col * N + (S::out_row(r, g) ^ col)) * HJ + d] = acc[jp * HJ + d][r];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= sbad[w];
    if (__builtin_expect(any, 0)) break;
#pragma unroll 1
    for (int x = t; x < count * N; x += 64 * NW) {
      const int c = x / N, e = x % N;
      float M = -INFINITY, lsum = 0.0f, o[HJ];
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, sv[w][0][c]);
#pragma unroll
      for (int d = 0; d < HJ; ++d) o[d] = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = state_weight(sv[w][0][c], M);
        lsum += sv[w][1][c] * f;
#pragma unroll
        for (int d = 0; d < HJ; ++d) o[d] += ((const float*)lds)[((w * N + c) * N + (e ^ c)) * HJ + d] * f;
      }
      const int at = S::DTN * e + jp * HJ, r = u.sp.first + u.i0 + c / G, h = u.g * G + c % G;
      if (whole) {
        const long long to = r * a.ldo + (long long)h * S::dim + at;
#pragma unroll
        for (int d = 0; d < HJ; ++d) o[d] = lsum == 0.0f ? 0.0f : o[d] / lsum;
        store_values<HJ>(a.out, to, a.x_type, a.out_wide, o);
      } else {
        const long long rec = kv_record<S>(a, u, r, h);
#pragma unroll
        for (int d = 0; d < HJ; ++d) a.part[rec * S::dim + at + d] = o[d];
        if (e == 0 && jp == 0) {
          a.state[2 * rec] = M;
          a.state[2 * rec + 1] = lsum;
        }
      }
    }
  }
  if (__builtin_expect(any, 0)) kv_again<S>(a, u, u.i0, count, wave, NW);
}

// Four tiles of 32 columns over the same keys, a wave each; K and V of two tiles of KT keys in
// LDS, of which a wave loads the quarter rows.
template <int TYPE, int DIM, int QP, int PP>
__device__ __forceinline__ void kv_attn_wide(const KvAttn& a) {
  typedef KvShape<TYPE, DIM, 32> S;
  // 64 keys a tile: one maximum, one rescaling and one barrier for twice the products (they do not fit f32 or q in parts)
  constexpr int NW = 4, KT = S::F32 || QP > 1 ? 32 : 64, H = KT / 16, RW = KT / NW, NI = RW / S::RPL;  // rows and loads of a wave
  constexpr int TB = KT * S::RB, NS = KT / 2;
  __shared__ __attribute__((aligned(16))) char lds[2 * 2 * TB];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int g = lane / 32, col = lane % 32, G = a.heads / a.c.kv_heads, P = 32 / G;
  const KvUnit u = kv_unit(a);
  if (!u.any) return;
  const int j0 = u.i0 + P * wave, nrow = min(P, u.sp.n - j0);  // of this wave (none: it helps with the loads)
  const int j = min(j0 + col / G, u.sp.n - 1), row = u.sp.first + j, head = u.g * G + col % G;

  KvPages<H> pg;
  pg.first = 0, pg.step = KT;
  pg.load(a, u, 0);
  bool missing = false, next_missing = false;
  unsigned klane = kv_k_lane<S>(RW * wave), vlane = kv_v_lane<S>(RW * wave);
  auto load = [&](int i) {
    if (i && i % pg.BLOCK == 0) pg.load(a, u, i);
    asm volatile("" : "+v"(klane), "+v"(vlane));
    missing = next_missing;
    next_missing = pg.missing(u, i);
    int rows;
    const long long at = pg.at(a, u, i, RW * wave / 16, S::RLOG, rows);
    const auto ks = kv_buffer<S>(a.c.k, at, rows), vs = kv_buffer<S>(a.c.v, at, rows);
    char* to = lds + (i & 1) * 2 * TB + 1024 * NI * wave;
#pragma unroll
    for (int x = 0; x < NI; ++x) kv_to_lds(ks, kv_k_load<S>(klane, x), to + 1024 * x);
#pragma unroll
    for (int x = 0; x < NI; ++x) kv_to_lds(vs, kv_v_load<S>(vlane, x), to + TB + 1024 * x);
  };
  load(0);
  __builtin_amdgcn_sched_barrier(0);
  KvQRegs<S, QP> q;
  const float c = kv_load_q<S, QP>(a, row, head, g, q.w);
  typename S::Acc acc[S::DTN];
#pragma unroll
  for (int d = 0; d < S::DTN; ++d) acc[d] = (typename S::Acc)(0.0f);
  KvState st;
  const int tiles = (u.k1 - u.k0 + KT - 1) / KT;
  const int l16 = lane % 16;
  const unsigned vread = (unsigned)(4 * g + l16 / 4) * S::RB + 8u * (l16 % 2) +
                         16u * ((unsigned)(2 * (lane / 16 % 2) + l16 % 4 / 2) ^ kv_v_swap<S>(4 * g + l16 / 4));
#pragma unroll 1
  for (int i = 0; i < tiles; ++i) {
    const int t0 = u.k0 + KT * i;
    // tile i is in LDS, by this wave and (behind the barrier) by the others; all have read tile i - 1, whose place
    // the next one takes
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    load(i + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (nrow <= 0) continue;
    const char* kb = lds + (i & 1) * 2 * TB;
    float sc[NS];
    // (matrix work first: the CU's other workgroup then has its softmax meanwhile; 4 trees of 26 nodes over 3000 f32
    // positions 81 us, 89 without)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < KT / 32; ++x) {
      float y[S::NR];
      kv_scores<S, QP>(y, kb + x * S::KB, q, col, g);
#pragma unroll
      for (int r = 0; r < S::NR; ++r) sc[S::NR * x + r] = y[r];
    }
    __builtin_amdgcn_s_setprio(0);
    if (__builtin_expect(missing, 0)) {
#pragma unroll
      for (int r = 0; r < NS; ++r) sc[r] = NAN;
    }
    if (t0 + KT > u.tl.base || t0 + KT > u.k1) {
#pragma unroll
      for (int x = 0; x < KT / 32; ++x) {
        const uint32_t see = kv_visible(a, row, j, u.tl.base, t0 + 32 * x, u.k1);
#pragma unroll
        for (int r = 0; r < S::NR; ++r)
          if (!(see >> S::key(r, g) & 1)) sc[S::NR * x + r] = -INFINITY;
      }
    }
    const float w = kv_softmax<S>(sc, st, c);
    kv_rescale<S>(acc, w);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < NS / 8; ++x) {
      if constexpr (S::F32) {
        const char* vb = kb + TB + S::DTN * S::EB * col;
        typename S::VRow v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = *(const typename S::VRow*)(vb + S::key(8 * x + r, g) * S::RB);
        kv_values<S, PP>(acc, sc + 8 * x, v, x == 0 ? w : 1.0f);
      } else {
        kv_values_lds<S, PP>(acc, sc + 8 * x, kb + TB + 16 * x * S::RB, vread);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // (no load may land in LDS that another workgroup has got)
  if (nrow <= 0) return;
  if (__builtin_expect(!kv_finite<S>(acc, st.l), 0)) {
    kv_again<S>(a, u, j0, G * nrow, 0, 1);
    return;
  }
  const float l = groups_sum<32>(st.l);
  if (col >= G * nrow) return;
  if (u.tl.len >= u.tl.n) {
    const long long to = row * a.ldo + (long long)head * DIM;
#pragma unroll
    for (int r = 0; r < S::AR; r += S::F32 ? 1 : 4)
#pragma unroll
      for (int d = 0; d < S::DTN; d += S::F32 ? S::DTN : 1) {
        float o[S::F32 ? S::DTN : 4];
#pragma unroll
        for (int e = 0; e < (S::F32 ? S::DTN : 4); ++e) o[e] = l == 0.0f ? 0.0f : (S::F32 ? acc[e][r] : acc[d][r + e]) / l;
        store_values(a.out, to + (S::F32 ? S::DTN * S::out_row(r, g) : 32 * d + S::out_row(r, g)), a.x_type, a.out_wide, o);
      }
  } else {
    const long long rec = kv_record<S>(a, u, row, head);
#pragma unroll
    for (int d = 0; d < S::DTN; ++d)
#pragma unroll
      for (int r = 0; r < S::AR; ++r)
        a.part[rec * DIM + (S::F32 ? S::DTN * S::out_row(r, g) + d : 32 * d + S::out_row(r, g))] = acc[d][r];
    if (g == 0) {
      a.state[2 * rec] = st.ref();
      a.state[2 * rec + 1] = l;
    }
  }
}
}  // namespace qmm

// Grid: 8 * ceil(slots * splits * kv_heads / 8) * tiles. Named by the cache's type, head_dim, the
// form (n16, n32: one tile of so many columns; wide: four of 32) and the parts of q and of the weights.
#define QMM_KV_ATTN(NAME, TYPE, DIM, QP, PP, NT, W16, W32, WW)                                                         \
  extern "C" __global__ void __launch_bounds__(NT, W16) qmm_kv_attn_##NAME##_n16_q##QP##_p##PP(qmm::KvAttn a) {        \
    qmm::kv_attn_narrow<TYPE, DIM, 16, QP, PP>(a);                                                                     \
  }                                                                                                                    \
  extern "C" __global__ void __launch_bounds__(NT, W32) qmm_kv_attn_##NAME##_n32_q##QP##_p##PP(qmm::KvAttn a) {        \
    qmm::kv_attn_narrow<TYPE, DIM, 32, QP, PP>(a);                                                                     \
  }                                                                                                                    \
  extern "C" __global__ void __launch_bounds__(256, WW) qmm_kv_attn_##NAME##_wide_q##QP##_p##PP(qmm::KvAttn a) {       \
    qmm::kv_attn_wide<TYPE, DIM, QP, PP>(a);                                                                           \
  }
// (the last three: waves a SIMD that leave the registers each form needs)
QMM_KV_ATTN(f32_d64, qmm::kTypeF32, 64, 1, 1, 256, 3, 2, 2)
QMM_KV_ATTN(f32_d128, qmm::kTypeF32, 128, 1, 1, 256, 2, 2, 2)
QMM_KV_ATTN(f32_d256, qmm::kTypeF32, 256, 1, 1, 128, 1, 1, 1)
#define QMM_KV_ATTN16(DIM, W1, W2, W3, W32, WW)                                      \
  QMM_KV_ATTN(f16_d##DIM, qmm::kTypeF16, DIM, 1, 2, 256, W1, W32, WW)                \
  QMM_KV_ATTN(f16_d##DIM, qmm::kTypeF16, DIM, 2, 2, 256, W2, W32, WW)                \
  QMM_KV_ATTN(bf16_d##DIM, qmm::kTypeBF16, DIM, 1, 2, 256, W1, W32, WW)              \
  QMM_KV_ATTN(bf16_d##DIM, qmm::kTypeBF16, DIM, 2, 2, 256, W2, W32, WW)              \
  QMM_KV_ATTN(bf16_d##DIM, qmm::kTypeBF16, DIM, 3, 3, 256, W3, W32, WW)
QMM_KV_ATTN16(64, 4, 4, 4, 2, 2)
QMM_KV_ATTN16(128, 3, 3, 2, 2, 2)
QMM_KV_ATTN16(256, 2, 2, 1, 1, 1)

// The chunks of a row joined: grid rows x heads / heads of a workgroup; four values a thread,
// join_lanes threads over a head's chunks. A row of one chunk has its result already.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_attn_join(qmm::KvAttn a) {
  using namespace qmm;
  __shared__ int lds4[4];
  __shared__ float lm[256], ll[256];
  __shared__ float4 lo[256];
  const int row = blockIdx.x, dim = a.c.head_dim, t = threadIdx.x;
  const int per = dim / 4, Y = a.join_lanes, hw = 256 / (per * Y);  // heads of a workgroup
  const int x = t % per, y = t / per % Y, h = blockIdx.y * hw + t / per / Y;
  const int s = kv_slot_of(a.r, a.c.slots, row, lds4);
  if (s < 0) return;
  const KvSpan sp = kv_span(a.r, s);
  const KvTile tl = kv_tile(a, sp, s, (row - sp.first) / a.group_rows * a.group_rows);
  if (tl.len >= tl.n) return;
  const int chunks = (tl.n + tl.len - 1) / tl.len;
  const bool on = h < a.heads;
  const long long rec = ((long long)row * a.heads + (on ? h : 0)) * a.splits;
  const float2* st = (const float2*)a.state + rec;
  const float4* part = (const float4*)(a.part + rec * dim) + x;
  // (a running maximum, four chunks' loads at a time)
  float M = -INFINITY, l = 0.0f;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c0 = y; c0 < chunks; c0 += 4 * Y) {
    float2 z[4];
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = min(c0 + i * Y, chunks - 1);
      z[i] = st[c];
      v[i] = part[(long long)c * per];
    }
    float m = M;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c0 + i * Y >= chunks) z[i] = {-INFINITY, 0.0f}, v[i] = {0.0f, 0.0f, 0.0f, 0.0f};
      m = fmaxf(m, z[i].x);
    }
    const float f = state_weight(M, m);
    l *= f;
    o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = state_weight(z[i].x, m);
      l += z[i].y * w;
      o.x += v[i].x * w, o.y += v[i].y * w, o.z += v[i].z * w, o.w += v[i].w * w;
    }
    M = m;
  }
  if (Y > 1) {
    lm[t] = M, ll[t] = l, lo[t] = o;
    __syncthreads();
    if (y != 0) return;
    float m = M;
    for (int i = 1; i < Y; ++i) m = fmaxf(m, lm[t + i * per]);
    l = 0.0f;
    o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < Y; ++i) {
      const float w = state_weight(lm[t + i * per], m);
      const float4 v = lo[t + i * per];
      l += ll[t + i * per] * w;
      o.x += v.x * w, o.y += v.y * w, o.z += v.z * w, o.w += v.w * w;
    }
  }
  if (!on) return;
  const long long to = row * a.ldo + (long long)h * dim + 4 * x;
  float r[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = l == 0.0f ? 0.0f : r[e] / l;
  store_values<4>(a.out, to, a.x_type, a.out_wide, r);
}

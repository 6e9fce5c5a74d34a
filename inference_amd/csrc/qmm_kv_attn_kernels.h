// Attention of a step's packed rows over the pages of their sequences (qmm_kv_attention).
//
// Row j of slot s sees the positions t < lens[s] and those lens[s] + i that its mask has:
//   out = sum_t w_t v_t / sum_t w_t,  w_t = e^(scale q . k_t - m),  m the largest score,
// in one pass over the positions with a running m, sum and output.
//
// Per kv head, the G = heads / kv_heads query heads of P = 32 / G consecutive rows form one
// tile of 32 columns (column = row * G + head). A workgroup takes a tile and a chunk of the
// positions; wave w has its key tiles w, w + NW, ... of 32 positions and a softmax state of
// its own; the waves' states are joined through LDS, the chunks' by a second launch.
//
// One key tile of a wave:
//   S^T = K Q^T      A = the 32 keys, B = the 32 columns. The result's column is lane & 31,
//                    so a column's 32 scores are 16 registers of two lanes: register r of
//                    lane half h is key 8 (r / 4) + 4 h + r % 4.
//   O^T += V^T P^T   A = V^T, B = P^T where S^T left it: the k index of a product may be
//                    permuted freely, so V's rows are loaded in P's order. Row m of V^T's
//                    tile j is element DT m + j (DT = head_dim / 32): a lane's loads are
//                    DT contiguous values of a key.
// K goes straight to LDS (buffer_load ... lds, 16 bytes a lane), its 16-byte chunks XORed by
// the key so that the 32 keys' reads of a chunk meet distinct banks; V goes to registers.
// K of the next tile is in flight from the end of the S product on, V of the next from the
// end of this tile's: a wave has up to two tiles in flight and waits for the oldest.
//
// Pages. A tile's two halves of 16 positions each lie in one page (pages are 16 or more), so
// a half is one buffer whose end is the last position there is: rows past it read as 0 and
// nothing past it is touched. A lane holds the page ids of 32 tiles at a time.
//
// Types. An f32 cache runs on the f32 matrix cores. A 16-bit cache runs on the 16-bit ones,
// 16 times their rate, with the f32 operand split into parts that each have the cache's
// type: q (QP parts: as many as hold its bits) and the weights (PP parts: 3 of bf16, 2 of
// f16 for an f32 output, which lose 2^-24 and 2^-22 of a weight; 2 of bf16 for a 16-bit
// output, 2^-16 of a weight against its rounding's 2^-9). For f16, whose range is small,
// a column's q is scaled by a power of two to [2^13, 2^14) and the weights by 2^12, which
// divides out.
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
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
// e^(s - m) is 2^(s log2 e - m log2 e): one fma, the rounding of m log2 e common to every
// weight of a column. From |m log2 e| = 2^24 on that rounding alone would over- or underflow
// 2^x, so there the difference is taken first. Either form is (s - off) log2 e - nl.
constexpr float kBigRef = 16777216.0f;
struct AttnRef {
  float off, nl;
};
__device__ __forceinline__ AttnRef attn_ref(float m) {
  const float nl = m == -INFINITY ? 0.0f : m * kLog2e;
  const bool big = !(fabsf(nl) < kBigRef);
  return {big ? m : 0.0f, big ? 0.0f : nl};
}
// 2^up e^(s - m)
__device__ __forceinline__ float score_weight(float s, const AttnRef& ref, float up) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(s - ref.off, kLog2e, up - ref.nl));
}
// of a state with the maximum m (its own reference m log2 e, rounded); 0 for -inf
__device__ __forceinline__ float state_weight(float m, const AttnRef& ref) {
#pragma clang fp contract(off)
  return __builtin_amdgcn_exp2f((m - ref.off) * kLog2e - ref.nl);
}

struct KvAttn {
  KvCache c;
  KvRows r;
  const void* q;
  const uint64_t* masks;
  void* out;
  float *part, *state;  // [rows][heads][splits] records: head_dim floats; maximum and sum
  long long ldq, ldm, ldo;
  int layer, x_type, heads, wide, splits, chunk, tiles;
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

// Positions that any row of the tile at row i0 (nrow rows) of a slot sees, and the length of
// the chunks they are split into: `chunk`, or a split's share where that is more.
struct KvTile {
  int base, n, nrow, len;
};
__device__ __forceinline__ KvTile kv_tile(const KvAttn& a, const KvSpan& sp, int s, int i0, int rows) {
  KvTile t;
  t.base = a.c.length(s);
  t.nrow = min(rows, sp.n - i0);
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
template <int TYPE>
__device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (TYPE == kTypeF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// TYPE: of the cache. DT = head_dim / 32. f32: QP = PP = 1.
template <int TYPE, int DT, int QP, int PP>
__device__ __forceinline__ void kv_attn_tile(const KvAttn& a) {
  constexpr bool F32 = TYPE == kTypeF32;
  constexpr int EB = F32 ? 4 : 2, dim = 32 * DT, RB = dim * EB;  // bytes of a value and of a row
  constexpr int NW = F32 && DT == 8 ? 2 : 4;                     // waves (K tiles of f32 rows of 256: 32 KB each)
  constexpr int CH = RB / 16, RPL = 64 / CH, STEPS = CH / 2;     // chunks of a row, rows a load, chunk pairs
  constexpr int SH = RB == 128 ? 1 : 0;                          // (two rows of 128 bytes fill the banks once)
  constexpr int KB = 32 * RB;                                    // bytes of a K tile
  constexpr int HJ = DT < 4 ? DT : 4;                            // V^T tiles joined at a time
  constexpr int JOIN = NW * 32 * 32 * HJ * 4;
  constexpr bool QLDS = F32 || QP > 1;
  constexpr int QB = QLDS ? QP * 32 * RB : 0;
  constexpr int ST = NW * 32 * 2 * 4 + 64;
  constexpr int LDS = NW * KB + QB > JOIN + ST ? NW * KB + QB : JOIN + ST;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int half = lane >> 5, col = lane & 31;

  // A unit (slot, chunk, kv head) and its tiles of columns follow each other on one XCD, which
  // then has the unit's keys in its L2: workgroups are dealt to the eight of them in turn.
  const int kv = a.c.kv_heads, G = a.heads / kv, P = 32 / G;
  const long long id = blockIdx.x;
  const int ct = (int)((id >> 3) % a.tiles);
  const long long unit = (id >> 3) / a.tiles * 8 + (id & 7);
  if (unit >= (long long)a.c.slots * a.splits * kv) return;
  const int g = (int)(unit % kv), chunk = (int)(unit / kv % a.splits), s = (int)(unit / kv / a.splits);
  const KvSpan sp = kv_span(a.r, s);
  const int i0 = ct * P;
  if (i0 >= sp.n) return;
  const KvTile tl = kv_tile(a, sp, s, i0, P);
  const long long start = (long long)chunk * tl.len;
  if (start >= tl.n) return;
  const int k0 = (int)start, k1 = min(k0 + tl.len, tl.n), base = tl.base;
  const int pi = min(col / G, tl.nrow - 1);  // columns past the rows repeat the last row; they are not stored
  const int row = sp.first + i0 + pi, j = i0 + pi;
  const int head = g * G + col % G;

  // ---- pages of this wave's tiles i = 0, 1, ... (positions k0 + 32 (wave + NW i)): lane l has the half l & 1 of tile
  // l / 2 of a block of 32
  const int lg = a.c.page_log;
  auto load_ids = [&](int i) {
    const long long pos = k0 + 32LL * (wave + (long long)NW * (i + (lane >> 1))) + 16 * (lane & 1);
    return pos < k1 ? a.c.page(s, (int)pos >> lg) : -1;
  };
  int ids = load_ids(0);
  struct Half {
    __amdgpu_buffer_rsrc_t k, v;
  };
  // Half x of tile i as buffers that end at the last position (of no bytes without a page).
  bool missing = false;
  auto half_of = [&](int i, int x) {
    const int pos = __builtin_amdgcn_readfirstlane(k0 + 32 * (wave + NW * i) + 16 * x);
    const int p = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + x);
    const int rows = min(max(k1 - pos, 0), 16);
    missing |= p < 0 && rows > 0;
    const long long at = a.c.row(a.layer, max(p, 0), g, pos & ((1 << lg) - 1)) * EB;
    const int bytes = __builtin_amdgcn_readfirstlane(p < 0 ? 0 : rows * RB);
    Half hf;
    hf.k = __builtin_amdgcn_make_buffer_rsrc((char*)a.c.k + at, 0, bytes, 0x00020000);
    hf.v = __builtin_amdgcn_make_buffer_rsrc((char*)a.c.v + at, 0, bytes, 0x00020000);
    return hf;
  };
  char* kb = lds + wave * KB;
  // K rows, 64 chunks a load: chunk c of row r in slot c ^ (r >> SH) % CH
  const int lr = lane / CH;
  auto load_k = [&](const Half& h0, const Half& h1) {
#pragma unroll
    for (int i = 0; i < 32 / RPL; ++i) {
      const int r = RPL * i + lr;
      const unsigned at = (unsigned)(r & 15) * RB + 16u * ((unsigned)(lane % CH) ^ ((unsigned)(r >> SH) & (CH - 1)));
      __builtin_amdgcn_raw_ptr_buffer_load_lds(RPL * i < 16 ? h0.k : h1.k,
                                               (__attribute__((address_space(3))) void*)(kb + 1024 * i), 16, at, 0, 0, 0);
    }
  };
  struct VRow {
    uint32_t w[DT * EB / 4];
  };
  VRow v[16];
  // f32 rows of 128 and more: the first eight registers of V early, the others behind the S product, which needs
  // the room (with all 16 early 31 registers went to scratch)
  constexpr int VEARLY = F32 && DT >= 4 ? 8 : 16;
  const std::integral_constant<int, 0> v_first;
  const std::integral_constant<int, VEARLY> v_early;
  const std::integral_constant<int, 16> v_last;
  auto load_v = [&](const Half& h0, const Half& h1, auto from, auto to) {
#pragma unroll
    for (int r = decltype(from)::value; r < decltype(to)::value; ++r) {
      const unsigned at = (unsigned)(8 * ((r >> 2) & 1) + 4 * half + (r & 3)) * RB + (unsigned)(DT * EB) * col;
      const auto rs = r < 8 ? h0.v : h1.v;
      if constexpr (DT * EB == 4) {
        v[r].w[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0);
      } else if constexpr (DT * EB == 8) {
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0));
        v[r].w[0] = x[0], v[r].w[1] = x[1];
      } else {
#pragma unroll
        for (int y = 0; y < DT * EB / 16; ++y) {
          const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + 16 * y, 0, 0));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[r].w[4 * y + e] = x[e];
        }
      }
    }
  };
  Half h0 = half_of(0, 0), h1 = half_of(0, 1);
  load_k(h0, h1);
  __builtin_amdgcn_sched_barrier(0);

  // ---- q: a lane has chunks 2 c + half of its column
  float down = 1.0f;  // the score's power of two that q's scaling put in
  u32x4 qreg[QLDS ? 1 : STEPS];
  char* qb = lds + NW * KB;
  {
    constexpr int E = 16 / EB;  // values of a chunk
    float x[STEPS][E];
    const long long at = row * a.ldq + (long long)head * dim;
    // (a branch a type and boundary, all loads in each: in flight together)
    auto load_q = [&](auto bytes, auto wide) {
      constexpr int B = decltype(bytes)::value;
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int y = 0; y < E / 4; ++y) {
          float f[4];
          load4_typed(f, a.q, at + E * (2 * c + half) + 4 * y, B == 4 ? kTypeF32 : a.x_type, decltype(wide)::value);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c][4 * y + e] = f[e];
        }
    };
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 2> two;
    if (a.x_type == kTypeF32)
      a.wide ? load_q(four, std::true_type()) : load_q(four, std::false_type());
    else
      a.wide ? load_q(two, std::true_type()) : load_q(two, std::false_type());
    float most = 0.0f;
#pragma unroll
    for (int c = 0; c < STEPS; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) most = fmaxf(most, fabsf(x[c][e]));
    if constexpr (TYPE == kTypeF16) {
      most = fmaxf(most, __shfl_xor(most, 32));
      int up = 0;
      if (most > 0.0f && most < INFINITY) up = min(max(14 - __builtin_amdgcn_frexp_expf(most), -100), 100);
      down = __builtin_ldexpf(1.0f, -up);
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int e = 0; e < E; ++e) x[c][e] = __builtin_ldexpf(x[c][e], up);
    }
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
      u32x4 w[QP];
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[0][e] = __builtin_bit_cast(uint32_t, x[c][e]);
      } else {
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t b = (uint32_t)to_half(x[c][2 * e], TYPE) | (uint32_t)to_half(x[c][2 * e + 1], TYPE) << 16;
            w[p][e] = b;
            x[c][2 * e] -= low_of<TYPE>(b);
            x[c][2 * e + 1] -= high_of<TYPE>(b);
          }
      }
      if constexpr (QLDS) {
        if (c % NW == wave) {
#pragma unroll
          for (int p = 0; p < QP; ++p) *(u32x4*)(qb + ((p * STEPS + c) * 64 + lane) * 16) = w[p];
        }
      } else {
        qreg[c] = w[0];
      }
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  load_v(h0, h1, v_first, v_early);
  __builtin_amdgcn_sched_barrier(0);
  const float scale = a.scale * down;
  constexpr float kUp = TYPE == kTypeF16 ? 12.0f : 0.0f;

  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = (f32x16)(0.0f);
  float m = -INFINITY, ml = 0.0f, l = 0.0f;  // maximum, maximum * log2 e (0 while it is -inf), this half's sum
  const unsigned kread = (unsigned)col * RB, kx = (unsigned)(col >> SH) & (CH - 1);
  if constexpr (QLDS) __syncthreads();

#pragma unroll 1
  for (int i = 0; k0 + 32 * (wave + NW * i) < k1; ++i) {
    const int t0 = k0 + 32 * (wave + NW * i);
    const bool poison = missing;
    missing = false;
    // K is in LDS once no loads but V's are out: 8 of f32 rows of 128, else 16
    __builtin_amdgcn_s_waitcnt(F32 && DT == 4 ? 0x0f78 : 0x4f70);
    __builtin_amdgcn_sched_barrier(0);
    auto kchunk = [&](int c) { return *(const u32x4*)(kb + kread + 16u * ((unsigned)(2 * c + half) ^ kx)); };
    f32x16 sc;
    if constexpr (F32) {
      // eight chains of roundings, each an eighth of the sum
      u32x4 ka = kchunk(0), qa = *(const u32x4*)(qb + lane * 16);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        f32x16 c4[4] = {(f32x16)(0.0f), (f32x16)(0.0f), (f32x16)(0.0f), (f32x16)(0.0f)};
#pragma unroll
        for (int c = x * STEPS / 2; c < (x + 1) * STEPS / 2; ++c) {  // the next chunks' reads fly under this one's products
          const int nx = c + 1 < STEPS ? c + 1 : c;
          const u32x4 kn = kchunk(nx), qn = *(const u32x4*)(qb + (nx * 64 + lane) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            c4[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(ka[e]), __uint_as_float(qa[e]), c4[e], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          ka = kn;
          qa = qn;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float y = (c4[0][r] + c4[1][r]) + (c4[2][r] + c4[3][r]);
          sc[r] = x == 0 ? y : sc[r] + y;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // two chains; of q's parts the smallest first
      f32x16 c2[2] = {(f32x16)(0.0f), (f32x16)(0.0f)};
#pragma unroll
      for (int c = 0; c < STEPS; ++c) {
        const u32x4 ka = kchunk(c);
        if constexpr (QLDS) {
#pragma unroll
          for (int p = QP - 1; p >= 0; --p)
            c2[c & 1] = mfma16<TYPE>(ka, *(const u32x4*)(qb + ((p * STEPS + c) * 64 + lane) * 16), c2[c & 1]);
        } else {
          c2[c & 1] = mfma16<TYPE>(ka, qreg[c], c2[c & 1]);
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = c2[0][r] + c2[1][r];
    }
    __builtin_amdgcn_sched_barrier(0);
    // every lane's reads of the K tile are consumed: the next may overwrite it. Unconditional (past the end the
    // buffers are empty): under a condition the waits for V would have to assume it was not issued.
    load_v(h0, h1, v_early, v_last);
    if (((i + 1) & 31) == 0) ids = load_ids(i + 1);
    h0 = half_of(i + 1, 0);
    h1 = half_of(i + 1, 1);
    load_k(h0, h1);
    __builtin_amdgcn_sched_barrier(0);

#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] *= scale;
    if (poison) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = NAN;
    }
    if (t0 + 32 > base || t0 + 32 > k1) {
      uint32_t see;
      if (a.masks) {
        const int rel = t0 - base;
        see = rel >= 0 ? kv_mask_bits(a, row, rel) : rel <= -32 ? ~0u : kv_mask_bits(a, row, 0) << -rel | ((1u << -rel) - 1);
      } else {
        const int c = base + j + 1 - t0;
        see = c >= 32 ? ~0u : c <= 0 ? 0 : (1u << c) - 1;
      }
      if (k1 - t0 < 32) see &= (1u << (k1 - t0)) - 1;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!(see >> (8 * (r >> 2) + 4 * half + (r & 3)) & 1)) sc[r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[r]);
    mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
    const float nml = mx == -INFINITY ? 0.0f : mx * kLog2e;
    float w;  // of what there was
    if (__builtin_expect(__any(!(fabsf(nml) < kBigRef)), 0)) {  // (see kBigRef)
      const AttnRef ref = attn_ref(mx);
      w = state_weight(m, ref);
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = score_weight(sc[r], ref, kUp);
    } else {
      w = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml - nml);
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], kLog2e, kUp - nml));
    }
    l *= w;
    m = mx;
    ml = nml;
#pragma unroll
    for (int r = 0; r < 16; ++r) l += sc[r];
    if constexpr (F32) {
      // 16 keys' products are summed on their own and added to the running sum once
      f32x16 o[2];
#pragma unroll
      for (int d = 0; d <= 2 * DT; ++d) {
        if (d < 2 * DT) {
          o[d & 1] = (f32x16)(0.0f);
#pragma unroll
          for (int r = 0; r < 8; ++r)
            o[d & 1] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v[(d < DT ? 0 : 8) + r].w[d % DT]),
                                                            sc[(d < DT ? 0 : 8) + r], o[d & 1], 0, 0, 0);
        }
        if (d > 0) {  // added while the next 16 keys' products run
          const int x = (d - 1) % DT;
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[x][r] = __builtin_fmaf(acc[x][r], d <= DT ? w : 1.0f, o[(d - 1) & 1][r]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      if (!__all(w == 1.0f)) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= w;
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        u32x4 p[PP];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = sc[8 * st + 2 * e], y = sc[8 * st + 2 * e + 1];
#pragma unroll
          for (int q = 0; q < PP; ++q) {
            p[q][e] = pack2<TYPE>(x, y);
            x -= low_of<TYPE>(p[q][e]);
            y -= high_of<TYPE>(p[q][e]);
          }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 vt;  // eight keys' value d of this lane
#pragma unroll
          for (int e = 0; e < 4; ++e)
            vt[e] = __builtin_amdgcn_perm(v[8 * st + 2 * e + 1].w[d / 2], v[8 * st + 2 * e].w[d / 2], d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int q = PP - 1; q >= 0; --q) acc[d] = mfma16<TYPE>(vt, p[q], acc[d]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v(h0, h1, v_first, v_early);
    __builtin_amdgcn_sched_barrier(0);
  }

  // ---- the waves' states
  bool bad;
  {
    float z = l * 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) z = __builtin_fmaf(acc[d][r], 0.0f, z);
    bad = __any(z != 0.0f);  // (NaN, of an infinity or a NaN)
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): no K load may land on what follows
  __syncthreads();
  float(*st)[2][32] = (float(*)[2][32])(lds + JOIN);
  int* sbad = (int*)(lds + JOIN + NW * 32 * 2 * 4);
  l += __shfl_xor(l, 32);
  if (half == 0) {
    st[wave][0][col] = m;
    st[wave][1][col] = l;
  }
  if (lane == 0) sbad[wave] = bad;
  const bool whole = tl.len >= tl.n;  // one chunk: the result itself
  auto record = [&](int c) { return (((long long)(sp.first + i0 + c / G)) * a.heads + g * G + c % G) * a.splits + chunk; };
#pragma unroll
  for (int jp = 0; jp < DT / HJ; ++jp) {
    if (jp) __syncthreads();  // (the last part is read)
    float* ob = (float*)lds + wave * 32 * 32 * HJ;
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int d = 0; d < HJ; ++d)
        ob[(col * 32 + ((8 * (r >> 2) + 4 * half + (r & 3)) ^ col)) * HJ + d] = acc[jp * HJ + d][r];
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= sbad[w];
    if (__builtin_expect(any, 0)) break;
#pragma unroll
    for (int y = 0; y < 32 * 32 / (64 * NW); ++y) {
      const int x = 64 * NW * y + t, c = x >> 5, e = x & 31;
      if (c >= G * tl.nrow) break;
      float M = -INFINITY, lsum = 0.0f, o[HJ];
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, st[w][0][c]);
      const AttnRef ref = attn_ref(M);
#pragma unroll
      for (int d = 0; d < HJ; ++d) o[d] = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = state_weight(st[w][0][c], ref);
        lsum += st[w][1][c] * f;
#pragma unroll
        for (int d = 0; d < HJ; ++d)
          o[d] += ((const float*)lds)[((w * 32 + c) * 32 + (e ^ c)) * HJ + d] * f;
      }
      const int at = DT * e + jp * HJ;
      if (whole) {
        const long long to = (sp.first + i0 + c / G) * a.ldo + (long long)(g * G + c % G) * dim + at;
#pragma unroll
        for (int d = 0; d < HJ; ++d) store_typed(a.out, to + d, a.x_type, lsum == 0.0f ? 0.0f : o[d] / lsum);
      } else {
        const long long rec = record(c);
#pragma unroll
        for (int d = 0; d < HJ; ++d) a.part[rec * dim + at + d] = o[d];
        if (e == 0 && jp == 0) {
          a.state[2 * rec] = M;
          a.state[2 * rec + 1] = lsum;
        }
      }
    }
  }
  {
    int any = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= sbad[w];
    if (__builtin_expect(!any, 1)) return;
  }
  constexpr int R = dim / 64;
#pragma unroll 1
  for (int c = wave; c < G * tl.nrow; c += NW) {
    float o[R], cm, cl;
    const int r = sp.first + i0 + c / G, h = g * G + c % G;
    kv_column<R>(a, s, r, i0 + c / G, h, base, k0, k1, o, cm, cl);
    if (whole) {
#pragma unroll
      for (int e = 0; e < R; ++e)
        store_typed(a.out, r * a.ldo + (long long)h * dim + R * lane + e, a.x_type, cl == 0.0f ? 0.0f : o[e] / cl);
    } else {
      const long long rec = record(c);
      const float up = TYPE == kTypeF16 ? 4096.0f : 1.0f;  // (as the tiles' weights)
#pragma unroll
      for (int e = 0; e < R; ++e) a.part[rec * dim + R * lane + e] = o[e] * up;
      if (lane == 0) {
        // (scores that are all NaN have the maximum -inf, and a sum that must not be left out)
        a.state[2 * rec] = cm == -INFINITY && cl != 0.0f ? 0.0f : cm;
        a.state[2 * rec + 1] = cl * up;
      }
    }
  }
}
}  // namespace qmm

// Grid: 8 * ceil(slots * splits * kv_heads / 8) * tiles. Named by the cache's type, head_dim
// and the parts of q and of the weights.
#define QMM_KV_ATTN(NAME, TYPE, DT, QP, PP, NT, WPS)                                                     \
  extern "C" __global__ void __launch_bounds__(NT, WPS) qmm_kv_attn_##NAME(qmm::KvAttn a) {              \
    qmm::kv_attn_tile<TYPE, DT, QP, PP>(a);                                                              \
  }
QMM_KV_ATTN(f32_d64_q1_p1, qmm::kTypeF32, 2, 1, 1, 256, 2)
QMM_KV_ATTN(f32_d128_q1_p1, qmm::kTypeF32, 4, 1, 1, 256, 2)
QMM_KV_ATTN(f32_d256_q1_p1, qmm::kTypeF32, 8, 1, 1, 128, 1)
#define QMM_KV_ATTN16(DT, D, WPS)                                                    \
  QMM_KV_ATTN(f16_d##D##_q1_p2, qmm::kTypeF16, DT, 1, 2, 256, WPS)                   \
  QMM_KV_ATTN(f16_d##D##_q2_p2, qmm::kTypeF16, DT, 2, 2, 256, WPS)                   \
  QMM_KV_ATTN(bf16_d##D##_q1_p2, qmm::kTypeBF16, DT, 1, 2, 256, WPS)                 \
  QMM_KV_ATTN(bf16_d##D##_q2_p2, qmm::kTypeBF16, DT, 2, 2, 256, WPS)                 \
  QMM_KV_ATTN(bf16_d##D##_q3_p3, qmm::kTypeBF16, DT, 3, 3, 256, WPS)
QMM_KV_ATTN16(2, 64, 2)
QMM_KV_ATTN16(4, 128, 2)
QMM_KV_ATTN16(8, 256, 1)

// The chunks of a row joined: grid rows, heads. A row of one chunk has its result already.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_attn_join(qmm::KvAttn a) {
  using namespace qmm;
  __shared__ int lds4[4];
  const int row = blockIdx.x, dim = a.c.head_dim, P = 32 / (a.heads / a.c.kv_heads);
  const int s = kv_slot_of(a.r, a.c.slots, row, lds4);
  if (s < 0) return;
  const KvSpan sp = kv_span(a.r, s);
  const KvTile tl = kv_tile(a, sp, s, (row - sp.first) / P * P, P);
  if (tl.len >= tl.n) return;
  const int chunks = (tl.n + tl.len - 1) / tl.len;
  const int x = blockIdx.y * 256 + threadIdx.x;
  if (x >= a.heads * dim) return;
  const int h = x / dim, d = x % dim;
  const long long rec = ((long long)row * a.heads + h) * a.splits;
  float M = -INFINITY;
  for (int c = 0; c < chunks; ++c) M = fmaxf(M, a.state[2 * (rec + c)]);
  const AttnRef ref = attn_ref(M);
  float l = 0.0f, o = 0.0f;
  for (int c = 0; c < chunks; ++c) {
    const float f = state_weight(a.state[2 * (rec + c)], ref);
    l += a.state[2 * (rec + c) + 1] * f;
    o += a.part[(rec + c) * dim + d] * f;
  }
  store_typed(a.out, row * a.ldo + (long long)h * dim + d, a.x_type, l == 0.0f ? 0.0f : o / l);
}

// y = x . W^T of MXFP4 weights and digit planes (qmm_mx_common.h), for dense rows and
// for routed rows of stacked expert weights.
#pragma once

#include "qmm_mx_common.h"

namespace qmm {

// One weight matrix of a launch, its output and what happens to it there.
struct MxOut {
  const uint8_t* w;
  void* y;
  const void* bias;  // [n] or null
  int y_type, bias_type;
  int accumulate;    // y +=
  int wide;          // rows of y start on a boundary of four values
};

// Which rows a workgroup multiplies: rows [first, first + count) of the planes and of
// the output by rows [w0, w0 + n) of the stacked weights.
struct MxRows {
  long long w0;
  int first, count;
};

// Tile `y` of an expert-ordered list, BM rows a tile: the expert and the tile's rows.
// Expert e holds rows offsets[e] .. offsets[e] + counts[e]; tiles are numbered through
// the experts. False past the last tile. Every lane of a wave takes 64 experts' counts
// at a time. Counts and offsets are the caller's: they are cut to [0, pairs].
__device__ __forceinline__ bool mx_expert_tile(const int* __restrict__ counts, const int* __restrict__ offsets,
                                               int experts, int pairs, int n, int bm, int y, MxRows& r) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane;
    int off = 0, cnt = 0;
    if (e < experts) {
      off = min(max(offsets[e], 0), pairs);
      cnt = min(max(counts[e], 0), pairs - off);
    }
    const int tiles = (cnt + bm - 1) / bm;
    int sum = tiles;  // inclusive prefix over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned long long hit = __ballot(base + sum > y);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int t = y - (base + __shfl(sum, l) - __shfl(tiles, l));
      const int o = __shfl(off, l), c = __shfl(cnt, l);
      r.w0 = (long long)(e0 + l) * n;
      r.first = o + t * bm;
      r.count = min(c - t * bm, bm);
      return true;
    }
    base += __shfl(sum, 63);
  }
  return false;
}

// A lane's place in the units: row `row` of the weight or of the planes (clamped by the
// caller), lane half h. Rows need not start on a tile: experts' rows follow each other.
__device__ __forceinline__ long long mx_w_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxUnit) + 512 * h + 16 * (row & 31);
}
__device__ __forceinline__ long long mx_ws_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxUnit) + kMxScaleOff + 128 * h + 4 * (row & 31);
}
__device__ __forceinline__ long long mx_x_at(long long row, int kc) { return (row >> 5) * ((long long)kc * kMxXUnit); }
__device__ __forceinline__ long long mx_xs_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxXUnit) + kMxXScaleOff + 128 * h + 4 * (row & 31);
}

// A lane's block of a step as its two digits, from the step's memory or LDS. `l`: the
// lane's place, 16 (32 h + r).
struct MxX {
  mx_u32x6 hi, lo;
};
__device__ __forceinline__ mx_u32x6 mx_digit(const uint8_t* p, const uint8_t* tail) {
  const mx_u32x4 a = *reinterpret_cast<const mx_u32x4*>(p);
  const mx_u32x2 b = *reinterpret_cast<const mx_u32x2*>(tail);
  return mx_u32x6{a[0], a[1], a[2], a[3], b[0], b[1]};
}
__device__ __forceinline__ MxX mx_get_x(const uint8_t* step, unsigned l) {
  MxX x;
  x.hi = mx_digit(step + l, step + kMxXTail + l / 2);
  x.lo = mx_digit(step + kMxXLo + l, step + kMxXTail + 512 + l / 2);
  return x;
}

template <int T>
struct MxType {
  static constexpr int value = T;
};

// Four columns of a row of the output from col on (those below n).
__device__ __forceinline__ mx_f32x4 mx_bias4(const MxOut& o, int col, int n) {
  mx_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (o.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < n) v[j] = mx_load(o.bias, o.bias_type, col + j);
  }
  return v;
}
template <int T>
__device__ __forceinline__ void mx_put4(const MxOut& o, long long row, int ldy, int col, int n, mx_f32x4 v) {
  const long long at = row * ldy + col;
  if (o.wide && col + 3 < n) {
    if constexpr (T == kF32) {
      mx_f32x4* p = reinterpret_cast<mx_f32x4*>(static_cast<float*>(o.y) + at);
      if (o.accumulate) v += *p;
      *p = v;
    } else {
      *reinterpret_cast<mx_u32x2*>(static_cast<uint16_t*>(o.y) + at) =
          mx_u32x2{mx_to16(v[0], T) | (uint32_t)mx_to16(v[1], T) << 16, mx_to16(v[2], T) | (uint32_t)mx_to16(v[3], T) << 16};
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < n) {
      if constexpr (T == kF32) {
        float* p = static_cast<float*>(o.y) + at + j;
        *p = o.accumulate ? *p + v[j] : v[j];
      } else {
        static_cast<uint16_t*>(o.y)[at + j] = mx_to16(v[j], T);
      }
    }
}

// Up to 32 rows: a workgroup of W waves takes one 32-column tile of the output and
// splits K over its waves by chunks; the waves' sums meet in LDS, in wave order.
template <int W>
__device__ __forceinline__ void mx_gemv(const MxOut& o, const MxRows& rows, int n, int kc, int tile,
                                        const uint8_t* __restrict__ xq, int ldy) {
  __shared__ float red[W][32][33];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, c = lane & 31;
  const long long wrow = rows.w0 + min(kMxTile * tile + c, n - 1);
  const long long xrow = rows.first + min(c, rows.count - 1);
  const uint8_t* wp = o.w + mx_w_at(wrow, h, kc);
  const uint8_t* wsp = o.w + mx_ws_at(wrow, h, kc);
  const uint8_t* xp = xq + mx_x_at(xrow, kc);
  const unsigned xl = 512 * h + 16 * (unsigned)(xrow & 31);
  const uint8_t* xsp = xq + mx_xs_at(xrow, h, kc);
  mx_f32x16 acc = (mx_f32x16)(0.0f);
  for (int k = wave; k < kc; k += W) {
    const uint8_t* wk = wp + (long long)k * kMxUnit;
    const uint8_t* xk = xp + (long long)k * kMxXUnit;
    const int sw = *reinterpret_cast<const int*>(wsp + (long long)k * kMxUnit);
    const int sx = *reinterpret_cast<const int*>(xsp + (long long)k * kMxXUnit), sl = sx - 0x04040404;
    MxX x;
#define QMM_MX_STEP(S)                                                                                          \
  x = mx_get_x(xk + S * kMxXStep, xl);                                                                          \
  acc = mx_mfma<S>(*reinterpret_cast<const mx_u32x4*>(wk + S * kMxStepBytes), x.hi, x.lo, acc, sw, sx, sl);
    QMM_MX_STEP(0)
    QMM_MX_STEP(1)
    QMM_MX_STEP(2)
    QMM_MX_STEP(3)
#undef QMM_MX_STEP
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) red[wave][c][8 * (r >> 2) + 4 * h + (r & 3)] = acc[r];
  __syncthreads();
  for (int j = t; j < 8 * rows.count; j += 64 * W) {
    const int m = j >> 3, q = 4 * (j & 7), col = kMxTile * tile + q;
    mx_f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = red[0][m][q + i];
#pragma unroll
      for (int w = 1; w < W; ++w) v[i] += red[w][m][q + i];
    }
    v += mx_bias4(o, col, n);
    if (o.y_type == kF32) mx_put4<kF32>(o, rows.first + m, ldy, col, n, v);
    else if (o.y_type == kF16) mx_put4<kF16>(o, rows.first + m, ldy, col, n, v);
    else mx_put4<kBF16>(o, rows.first + m, ldy, col, n, v);
  }
}

// A tile of 32 FM WM rows x 32 FN WN columns by WM x WN waves, a wave 32 FM x 32 FN of it.
// RW steps of weights in registers (this one and those on their way).
template <int FM, int FN, int WM, int WN, int RW>
__device__ __forceinline__ void mx_gemm(const MxOut& o, const MxRows& rows, int n, int kc, int n0,
                                        const uint8_t* __restrict__ xq, int ldy) {
  constexpr int NW = WM * WN, XF = FM * WM, FW = XF / NW;
  static_assert(XF % NW == 0, "whole fragments a wave");
  constexpr int kStage = XF * kMxXStep;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, c = lane & 31, wm = wave % WM, wn = wave / WM;
  // 64-bit bases at the tile's first row, 32-bit offsets from them
  const long long xt = rows.first >> 5;
  const uint8_t* xb = xq + xt * ((long long)kc * kMxXUnit);
  // the fragments that this wave brings to LDS: a lane's place in the 16-byte and in
  // the 8-byte parts
  unsigned xo[FW][2], xso[FM], wo[FN], wso[FN];
#pragma unroll
  for (int j = 0; j < FW; ++j) {
    const long long r = rows.first + min(32 * (FW * wave + j) + c, rows.count - 1) - 32 * xt;
    xo[j][0] = (unsigned)mx_x_at(r, kc) + 512 * h + 16 * (unsigned)(r & 31);
    xo[j][1] = (unsigned)mx_x_at(r, kc) + kMxXTail + 256 * h + 8 * (unsigned)(r & 31);
  }
#pragma unroll
  for (int b = 0; b < FM; ++b)
    xso[b] = (unsigned)mx_xs_at(rows.first + min(32 * (FM * wm + b) + c, rows.count - 1) - 32 * xt, h, kc);
  const long long wt = (rows.w0 + n0) >> 5;
  const uint8_t* wb = o.w + wt * ((long long)kc * kMxUnit);
#pragma unroll
  for (int a = 0; a < FN; ++a) {
    const long long r = rows.w0 + min(n0 + 32 * (FN * wn + a) + c, n - 1) - 32 * wt;
    wo[a] = (unsigned)mx_w_at(r, h, kc);
    wso[a] = (unsigned)mx_ws_at(r, h, kc);
  }
  mx_f32x16 acc[FN][FM];
#pragma unroll
  for (int a = 0; a < FN; ++a)
#pragma unroll
    for (int b = 0; b < FM; ++b) acc[a][b] = (mx_f32x16)(0.0f);

  MxX st[FW];            // x on its way to LDS
  mx_u32x4 w[RW][FN];    // weights of this step and the next ones
  MxX x[2][FM];          // x of this step and the next
  int sw[2][FN], sx[2][FM];
  auto load_x = [&](int k, int s) {
    const unsigned at = (unsigned)k * kMxXUnit + s * kMxXStep;
#pragma unroll
    for (int j = 0; j < FW; ++j) {
      const uint8_t* p = xb + (xo[j][0] + at);
      const uint8_t* q = xb + (xo[j][1] + at);
      st[j].hi = mx_digit(p, q);
      st[j].lo = mx_digit(p + kMxXLo, q + 512);
    }
  };
  auto put_x = [&](int buf) {
#pragma unroll
    for (int j = 0; j < FW; ++j) {
      uint8_t* d = &lds[buf][kMxXStep * (FW * wave + j)];
      const mx_u32x6 u = st[j].hi, v = st[j].lo;
      *reinterpret_cast<mx_u32x4*>(d + 16 * lane) = mx_u32x4{u[0], u[1], u[2], u[3]};
      *reinterpret_cast<mx_u32x4*>(d + kMxXLo + 16 * lane) = mx_u32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<mx_u32x2*>(d + kMxXTail + 8 * lane) = mx_u32x2{u[4], u[5]};
      *reinterpret_cast<mx_u32x2*>(d + kMxXTail + 512 + 8 * lane) = mx_u32x2{v[4], v[5]};
    }
  };
  auto get_x = [&](int buf, MxX (&d)[FM]) {
#pragma unroll
    for (int b = 0; b < FM; ++b) d[b] = mx_get_x(&lds[buf][kMxXStep * (FM * wm + b)], 16 * lane);
  };
  auto load_w = [&](int k, int s, mx_u32x4 (&d)[FN]) {
    const unsigned at = (unsigned)k * kMxUnit + s * kMxStepBytes;
#pragma unroll
    for (int a = 0; a < FN; ++a) d[a] = *reinterpret_cast<const mx_u32x4*>(wb + (wo[a] + at));
  };
  auto load_s = [&](int k, int i) {
#pragma unroll
    for (int a = 0; a < FN; ++a) sw[i][a] = *reinterpret_cast<const int*>(wb + (wso[a] + (unsigned)k * kMxUnit));
#pragma unroll
    for (int b = 0; b < FM; ++b) sx[i][b] = *reinterpret_cast<const int*>(xb + (xso[b] + (unsigned)k * kMxXUnit));
  };
  auto sync = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's writes are in LDS
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  load_s(0, 0);
  load_x(0, 0);
#pragma unroll
  for (int s = 0; s < RW - 1; ++s) load_w(0, s, w[s]);
  put_x(0);
  load_x(0, 1);
  sync();
  get_x(0, x[0]);
#define QMM_MX_HALF(S, I, B0, B1)                                                                              \
  _Pragma("unroll") for (int b = B0; b < B1; ++b) {                                                            \
    _Pragma("unroll") for (int a = 0; a < FN; ++a) acc[a][b] =                                                 \
        mx_mfma1<S>(w[S % RW][a], x[S & 1][b].hi, acc[a][b], sw[I][a], sx[I][b]);                              \
    _Pragma("unroll") for (int a = 0; a < FN; ++a) acc[a][b] =                                                 \
        mx_mfma1<S>(w[S % RW][a], x[S & 1][b].lo, acc[a][b], sw[I][a], sx[I][b] - 0x04040404);                 \
  }
#define QMM_MX_STEP(S, I)                                                                                      \
  {                                                                                                            \
    put_x((S + 1) & 1);                                                                                        \
    load_x(S + 2 < 4 ? k : kn, (S + 2) & 3);                                                                   \
    load_w(S + RW - 1 < 4 ? k : kn, (S + RW - 1) & 3, w[(S + RW - 1) % RW]);                                   \
    if (S == 1) load_s(kn, 1 - I);                                                                             \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
    QMM_MX_HALF(S, I, 0, FM / 2)                                                                               \
    sync();                                                                                                    \
    get_x((S + 1) & 1, x[(S + 1) & 1]);                                                                        \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
    QMM_MX_HALF(S, I, FM / 2, FM)                                                                              \
  }
  // (past the last chunk the loads read it again, and what they bring is not used)
#pragma unroll 1
  for (int k = 0; k < kc; ++k) {
    const int kn = min(k + 1, kc - 1);
    QMM_MX_STEP(0, 0)
    QMM_MX_STEP(1, 0)
    QMM_MX_STEP(2, 0)
    QMM_MX_STEP(3, 0)
#pragma unroll
    for (int a = 0; a < FN; ++a) sw[0][a] = sw[1][a];
#pragma unroll
    for (int b = 0; b < FM; ++b) sx[0][b] = sx[1][b];
  }
#undef QMM_MX_STEP
#undef QMM_MX_HALF
  auto put = [&](auto type) {
#pragma unroll
    for (int a = 0; a < FN; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = n0 + 32 * (FN * wn + a) + 8 * q + 4 * h;
        const mx_f32x4 bias = mx_bias4(o, col, n);
#pragma unroll
        for (int b = 0; b < FM; ++b) {
          const int m = 32 * (FM * wm + b) + c;
          mx_f32x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = acc[a][b][4 * q + j] + bias[j];
          if (m < rows.count) mx_put4<decltype(type)::value>(o, rows.first + m, ldy, col, n, v);
        }
      }
  };
  if (o.y_type == kF32) put(MxType<kF32>{});
  else if (o.y_type == kF16) put(MxType<kF16>{});
  else put(MxType<kBF16>{});
}
}  // namespace qmm

// Dense rows: grid (32-column tiles, 32-row tiles).
extern "C" __global__ void __launch_bounds__(512) qmm_mx_gemv(qmm::MxOut o, int m, int n, int kc,
                                                              const uint8_t* __restrict__ xq, int ldy) {
  const int first = 32 * blockIdx.y;
  const qmm::MxRows r = {0, first, min(m - first, 32)};
  qmm::mx_gemv<8>(o, r, n, kc, blockIdx.x, xq, ldy);
}

// Routed rows: grid (32-column tiles, row tiles, weights).
extern "C" __global__ void __launch_bounds__(512) qmm_mx_expert_gemv(qmm::MxOut o0, qmm::MxOut o1, int experts,
                                                                     int pairs, int n, int kc,
                                                                     const int* __restrict__ counts,
                                                                     const int* __restrict__ offsets,
                                                                     const uint8_t* __restrict__ xq, int ldy) {
  qmm::MxRows r;
  if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 32, blockIdx.y, r)) return;
  qmm::mx_gemv<8>(blockIdx.z ? o1 : o0, r, n, kc, blockIdx.x, xq, ldy);
}

#define QMM_MX_GEMM(NAME, FM, FN, WM, WN, RW, EU)                                                              \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN, EU) qmm_mx_gemm_##NAME(                           \
      qmm::MxOut o, int m, int n, int kc, const uint8_t* __restrict__ xq, int ldy) {                           \
    const int first = 32 * FM * WM * blockIdx.y;                                                               \
    const qmm::MxRows r = {0, first, min(m - first, 32 * FM * WM)};                                            \
    qmm::mx_gemm<FM, FN, WM, WN, RW>(o, r, n, kc, 32 * FN * WN * blockIdx.x, xq, ldy);                             \
  }                                                                                                            \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN, EU) qmm_mx_expert_gemm_##NAME(                    \
      qmm::MxOut o0, qmm::MxOut o1, int experts, int pairs, int n, int kc, const int* __restrict__ counts,     \
      const int* __restrict__ offsets, const uint8_t* __restrict__ xq, int ldy) {                              \
    qmm::MxRows r;                                                                                             \
    if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 32 * FM * WM, blockIdx.y, r)) return;         \
    qmm::mx_gemm<FM, FN, WM, WN, RW>(blockIdx.z ? o1 : o0, r, n, kc, 32 * FN * WN * blockIdx.x, xq, ldy);          \
  }
QMM_MX_GEMM(256x256, 4, 4, 2, 2, 2, 1)
QMM_MX_GEMM(128x256, 2, 4, 2, 2, 2, 2)

// out[t] = sum over token t's pairs, in increasing expert order, of weight * yp[pair],
// then + shared[t] (times sg[t] when the shared expert is gated), rounded once to the
// output's type. Four columns a thread (n is a multiple of 32).
extern "C" __global__ void __launch_bounds__(256) qmm_mx_combine(const float* __restrict__ yp,
                                                                 const float* __restrict__ pair_weight,
                                                                 const int* __restrict__ token_pairs, int tokens,
                                                                 int topk, int n, const float* __restrict__ shared,
                                                                 const float* __restrict__ sg, void* __restrict__ out,
                                                                 int out_type, long long ldo, int wide) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int nq = n / 4;
  if (i >= (long long)tokens * nq) return;
  const int t = (int)(i / nq), c = 4 * (int)(i % nq);
  qmm::mx_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < topk; ++s) {
    const long long p = token_pairs[(long long)t * topk + s];
    acc += pair_weight[p] * *reinterpret_cast<const qmm::mx_f32x4*>(yp + p * n + c);
  }
  if (shared != nullptr) {
    const float g = sg != nullptr ? sg[t] : 1.0f;
    acc += g * *reinterpret_cast<const qmm::mx_f32x4*>(shared + (long long)t * n + c);
  }
  const long long at = t * ldo + c;
  if (!wide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) qmm::mx_store(out, out_type, at + j, acc[j]);
  } else if (out_type == qmm::kF32) {
    *reinterpret_cast<qmm::mx_f32x4*>(static_cast<float*>(out) + at) = acc;
  } else {
    *reinterpret_cast<qmm::mx_u32x2*>(static_cast<uint16_t*>(out) + at) =
        qmm::mx_u32x2{qmm::mx_to16(acc[0], out_type) | (uint32_t)qmm::mx_to16(acc[1], out_type) << 16,
                      qmm::mx_to16(acc[2], out_type) | (uint32_t)qmm::mx_to16(acc[3], out_type) << 16};
  }
}

// sg[t] = sigmoid(x[t] . g), a wave a token (qmm_moe_shared_gate for typed rows).
extern "C" __global__ void __launch_bounds__(256) qmm_mx_shared_gate(const void* __restrict__ x, int x_type,
                                                                     long long ldx, const float* __restrict__ g, int n,
                                                                     int tokens, float* __restrict__ sg) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= tokens) return;
  float acc = 0.0f;
  for (int c = lane; c < n; c += 64) acc += qmm::mx_load(x, x_type, t * ldx + c) * g[c];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) acc += __shfl_xor(acc, d);
  if (lane == 0) sg[t] = 1.0f / (1.0f + expf(-acc));
}

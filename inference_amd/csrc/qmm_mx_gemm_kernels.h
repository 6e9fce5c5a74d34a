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
  int accumulate;    // y += (f32)
};

// Which rows a workgroup multiplies: rows [first, first + count) of the output, whose
// activations are rows src[first + i] (or first + i) of the planes, by rows
// [w0, w0 + n) of the stacked weights.
struct MxRows {
  long long w0;
  int first, count;
  const int* src;
};

// Tile `y` of an expert-ordered list, BM rows a tile: the expert and the tile's rows.
// Expert e holds rows offsets[e] .. offsets[e] + counts[e]; tiles are numbered through
// the experts. False past the last tile. Every lane of a wave takes 64 experts' counts
// at a time. Counts and offsets are the caller's: they are cut to [0, pairs].
__device__ __forceinline__ bool mx_expert_tile(const int* __restrict__ counts, const int* __restrict__ offsets,
                                               int experts, int pairs, int n, int bm, int y,
                                               const int* __restrict__ src, MxRows& r) {
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
      r.src = src;
      return true;
    }
    base += __shfl(sum, 63);
  }
  return false;
}

// A lane's place in the weight's units: row `row` (clamped by the caller), lane half h.
__device__ __forceinline__ long long mx_w_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxUnit) + 512 * h + 16 * (row & 31);
}
__device__ __forceinline__ long long mx_ws_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxUnit) + kMxScaleOff + 128 * h + 4 * (row & 31);
}

__device__ __forceinline__ void mx_get_digits(const uint8_t* __restrict__ p, mx_u32x6& hi, mx_u32x6& lo) {
  const mx_u32x4* q = reinterpret_cast<const mx_u32x4*>(p);
  const mx_u32x4 a = q[0], b = q[1], c = q[2];
  hi = mx_u32x6{a[0], a[1], a[2], a[3], b[0], b[1]};
  lo = mx_u32x6{b[2], b[3], c[0], c[1], c[2], c[3]};
}

__device__ __forceinline__ void mx_finish(const MxOut& o, long long row, int ldy, int col, float v) {
  const long long at = row * ldy + col;
  if (o.bias != nullptr) v += mx_load(o.bias, o.bias_type, col);
  if (o.accumulate) v += mx_load(o.y, o.y_type, at);
  mx_store(o.y, o.y_type, at, v);
}

// Up to 32 rows: a workgroup of W waves takes one 32-column tile of the output and
// splits K over its waves by chunks; the waves' sums meet in LDS, in wave order.
template <int W>
__device__ __forceinline__ void mx_gemv(const MxOut& o, const MxRows& rows, int n, int kc, int tile,
                                        const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, int ldy) {
  __shared__ float red[W][32][33];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, c = lane & 31;
  const int col = min(kMxTile * tile + c, n - 1);
  const long long wrow = rows.w0 + col;
  const int i = rows.first + min(c, rows.count - 1);
  const long long xrow = rows.src ? rows.src[i] : i;
  const uint8_t* wp = o.w + mx_w_at(wrow, h, kc);
  const uint8_t* wsp = o.w + mx_ws_at(wrow, h, kc);
  const uint8_t* xp = xq + xrow * kc * kMxDigitChunk + kMxDigitBlock * h;
  const int* sp = reinterpret_cast<const int*>(xs + xrow * kc * 8) + h;
  mx_f32x16 acc = (mx_f32x16)(0.0f);
  for (int k = wave; k < kc; k += W) {
    const uint8_t* wk = wp + (long long)k * kMxUnit;
    const uint8_t* xk = xp + (long long)k * kMxDigitChunk;
    const int sw = *reinterpret_cast<const int*>(wsp + (long long)k * kMxUnit);
    const int sx = sp[2 * k], sl = sx - 0x04040404;
    mx_u32x6 hi, lo;
#define QMM_MX_STEP(S)                                                    \
  mx_get_digits(xk + S * 2 * kMxDigitBlock, hi, lo);                      \
  acc = mx_mfma<S>(*reinterpret_cast<const mx_u32x4*>(wk + S * kMxStepBytes), hi, lo, acc, sw, sx, sl);
    QMM_MX_STEP(0)
    QMM_MX_STEP(1)
    QMM_MX_STEP(2)
    QMM_MX_STEP(3)
#undef QMM_MX_STEP
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) red[wave][c][8 * (r >> 2) + 4 * h + (r & 3)] = acc[r];
  __syncthreads();
  for (int j = t; j < 32 * rows.count; j += 64 * W) {
    const int m = j >> 5, q = j & 31;
    if (kMxTile * tile + q >= n) continue;
    float v = red[0][m][q];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w][m][q];
    mx_finish(o, rows.first + m, ldy, kMxTile * tile + q, v);
  }
}

// 64 rows x 64 columns a wave, straight from memory.
__device__ __forceinline__ void mx_tile(const MxOut& o, const MxRows& rows, int n, int kc, int col0,
                                        const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, int ldy) {
  const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
  const uint8_t *wp[2], *wsp[2], *xp[2];
  const int* sp[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const long long wrow = rows.w0 + min(col0 + 32 * j + c, n - 1);
    const int i = rows.first + min(32 * j + c, rows.count - 1);
    const long long xrow = rows.src ? rows.src[i] : i;
    wp[j] = o.w + mx_w_at(wrow, h, kc);
    wsp[j] = o.w + mx_ws_at(wrow, h, kc);
    xp[j] = xq + xrow * kc * kMxDigitChunk + kMxDigitBlock * h;
    sp[j] = reinterpret_cast<const int*>(xs + xrow * kc * 8) + h;
  }
  mx_f32x16 acc[2][2] = {{(mx_f32x16)(0.0f), (mx_f32x16)(0.0f)}, {(mx_f32x16)(0.0f), (mx_f32x16)(0.0f)}};
  for (int k = 0; k < kc; ++k) {
    int sw[2], sx[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sw[j] = *reinterpret_cast<const int*>(wsp[j] + (long long)k * kMxUnit);
      sx[j] = sp[j][2 * k];
    }
#define QMM_MX_STEP(S)                                                                                               \
  {                                                                                                                  \
    mx_u32x4 w[2];                                                                                                   \
    mx_u32x6 hi[2], lo[2];                                                                                           \
    _Pragma("unroll") for (int j = 0; j < 2; ++j) {                                                                  \
      w[j] = *reinterpret_cast<const mx_u32x4*>(wp[j] + (long long)k * kMxUnit + S * kMxStepBytes);                  \
      mx_get_digits(xp[j] + (long long)k * kMxDigitChunk + S * 2 * kMxDigitBlock, hi[j], lo[j]);                     \
    }                                                                                                                \
    _Pragma("unroll") for (int a = 0; a < 2; ++a) _Pragma("unroll") for (int b = 0; b < 2; ++b) acc[a][b] =           \
        mx_mfma<S>(w[a], hi[b], lo[b], acc[a][b], sw[a], sx[b], sx[b] - 0x04040404);                                 \
  }
    QMM_MX_STEP(0)
    QMM_MX_STEP(1)
    QMM_MX_STEP(2)
    QMM_MX_STEP(3)
#undef QMM_MX_STEP
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int m = 32 * b + c;
    if (m >= rows.count) continue;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int q = col0 + 32 * a + 8 * (r >> 2) + 4 * h + (r & 3);
        if (q < n) mx_finish(o, rows.first + m, ldy, q, acc[a][b][r]);
      }
  }
}
}  // namespace qmm

// Dense rows: grid (32-column tiles, 32-row tiles).
extern "C" __global__ void __launch_bounds__(512) qmm_mx_gemv(qmm::MxOut o, int m, int n, int kc,
                                                              const uint8_t* __restrict__ xq,
                                                              const uint8_t* __restrict__ xs, int ldy) {
  const int first = 32 * blockIdx.y;
  const qmm::MxRows r = {0, first, min(m - first, 32), nullptr};
  qmm::mx_gemv<8>(o, r, n, kc, blockIdx.x, xq, xs, ldy);
}

// Routed rows: grid (32-column tiles, row tiles, weights).
extern "C" __global__ void __launch_bounds__(512) qmm_mx_expert_gemv(qmm::MxOut o0, qmm::MxOut o1, int experts,
                                                                     int pairs, int n, int kc,
                                                                     const int* __restrict__ counts,
                                                                     const int* __restrict__ offsets,
                                                                     const int* __restrict__ src,
                                                                     const uint8_t* __restrict__ xq,
                                                                     const uint8_t* __restrict__ xs, int ldy) {
  qmm::MxRows r;
  if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 32, blockIdx.y, src, r)) return;
  qmm::mx_gemv<8>(blockIdx.z ? o1 : o0, r, n, kc, blockIdx.x, xq, xs, ldy);
}

// Dense rows: grid (256-column tiles, 64-row tiles), a wave 64 of the columns.
extern "C" __global__ void __launch_bounds__(256) qmm_mx_gemm(qmm::MxOut o, int m, int n, int kc,
                                                              const uint8_t* __restrict__ xq,
                                                              const uint8_t* __restrict__ xs, int ldy) {
  const int first = 64 * blockIdx.y;
  const qmm::MxRows r = {0, first, min(m - first, 64), nullptr};
  const int col0 = 256 * blockIdx.x + 64 * (threadIdx.x >> 6);
  if (col0 < n) qmm::mx_tile(o, r, n, kc, col0, xq, xs, ldy);
}

extern "C" __global__ void __launch_bounds__(256) qmm_mx_expert_gemm(qmm::MxOut o0, qmm::MxOut o1, int experts,
                                                                     int pairs, int n, int kc,
                                                                     const int* __restrict__ counts,
                                                                     const int* __restrict__ offsets,
                                                                     const int* __restrict__ src,
                                                                     const uint8_t* __restrict__ xq,
                                                                     const uint8_t* __restrict__ xs, int ldy) {
  qmm::MxRows r;
  if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 64, blockIdx.y, src, r)) return;
  const int col0 = 256 * blockIdx.x + 64 * (threadIdx.x >> 6);
  if (col0 < n) qmm::mx_tile(blockIdx.z ? o1 : o0, r, n, kc, col0, xq, xs, ldy);
}

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

// y = x . W^T of MXFP4 weights and digit planes (qmm_mx_common.h), for dense rows and
// for routed rows of stacked expert weights.
#pragma once

#include "qmm_mx_common.h"
#include "qmm_mx_quant_kernels.h"

namespace qmm {

// One weight matrix of a launch, its output and what happens to it there.
struct MxOut {
  const uint8_t* w;
  void* y;
  const void* bias;  // [n] or null
  int y_type, bias_type;
  int accumulate;    // y +=
  int wide;          // rows of y start on 16-byte boundaries
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
      r.w0 = (long long)__builtin_amdgcn_readfirstlane(e0 + l) * n;
      r.first = __builtin_amdgcn_readfirstlane(o + t * bm);
      r.count = __builtin_amdgcn_readfirstlane(min(c - t * bm, bm));
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
__device__ __forceinline__ long long mx_x_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxXUnit) + 512 * h + 16 * (row & 31);
}
__device__ __forceinline__ long long mx_xs_at(long long row, int h, int kc) {
  return (row >> 5) * ((long long)kc * kMxXUnit) + kMxXScaleOff + 128 * h + 4 * (row & 31);
}

__device__ __forceinline__ mx_u32x12 mx_get_x(const uint8_t* p) {
  return mx_x(*reinterpret_cast<const mx_u32x4*>(p), *reinterpret_cast<const mx_u32x4*>(p + kMxXPart),
              *reinterpret_cast<const mx_u32x4*>(p + 2 * kMxXPart));
}

template <int T>
struct MxType {
  static constexpr int value = T;
};

// V columns of a row of the output from col on (those below n), 4 f32 or 8 16-bit ones.
template <int T, int V>
__device__ __forceinline__ void mx_put(const MxOut& o, long long row, int ldy, int col, int n, const float (&v)[V]) {
  const long long at = row * ldy + col;
  if constexpr (T == kF32) {
    float* p = static_cast<float*>(o.y) + at;
    if (o.wide && col + V <= n) {
      mx_f32x4 u = {v[0], v[1], v[2], v[3]};
      if (o.accumulate) u += *reinterpret_cast<const mx_f32x4*>(p);
      *reinterpret_cast<mx_f32x4*>(p) = u;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (col + j < n) p[j] = o.accumulate ? p[j] + v[j] : v[j];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(o.y) + at;
    if (o.wide && col + V <= n) {
      mx_u32x4 u;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = mx_to16(v[2 * j], T) | (uint32_t)mx_to16(v[2 * j + 1], T) << 16;
      *reinterpret_cast<mx_u32x4*>(p) = u;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (col + j < n) p[j] = mx_to16(v[j], T);
    }
  }
}

// Unquantized rows: row i of the product is row src[i] of x (or i), of type T.
struct MxRaw {
  const void* x;
  long long ldx;
  const int* src;
  int type, wide;
};

// The waves' sums of NT 16-column tiles, joined in wave order and written.
template <int W, int NT, bool GLU>
__device__ __forceinline__ void mx_gemv_join(const MxOut& o, const MxRows& rows, int n, int n0,
                                             float (&red)[W][16][16 * NT + 4], int ldy) {
  const int t = threadIdx.x;
  auto total = [&](int m, int q) {
    float v = red[0][m][q];
#pragma unroll
    for (int i = 1; i < W; ++i) v += red[i][m][q];
    return v;
  };
  if constexpr (GLU) {
    // h over the first wave's sums, then a lane a row
    const int cols = min(32, n - n0);
    float act[(32 * 16 + 64 * W - 1) / (64 * W)];
#pragma unroll
    for (int i = 0; i * 64 * W < 512; ++i) {
      const int j = t + i * 64 * W, m = j >> 5, q = j & 31;
      if (m < rows.count) {
        const float a = total(m, q), b = total(m, 32 + q);
        act[i] = a / (1.0f + expf(-a)) * b;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i * 64 * W < 512; ++i) {
      const int j = t + i * 64 * W;
      if (j >> 5 < rows.count) red[0][j >> 5][j & 31] = act[i];
    }
    __syncthreads();
    if (t >= rows.count) return;
    float v[32];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = red[0][t][j];
      amax = max(amax, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
    }
    mx_u32x6 hi, lo;
    const int e = mx_x_byte(amax);
    mx_digits(v, e, hi, lo);
    const long long r = rows.first + t;
    const int kf = (n + kMxChunk - 1) / kMxChunk, blk = n0 % kMxChunk / 32;
    uint8_t* unit = static_cast<uint8_t*>(o.y) + ((r >> 5) * kf + n0 / kMxChunk) * kMxXUnit;
    mx_put_block(unit, blk >> 1, 32 * (blk & 1) + (int)(r & 31), e, hi, lo);
    if (n0 + cols >= n)  // the rest of the chunk: the product reads whole ones
      for (int z = blk + 1; z < 8; ++z)
        mx_put_block(unit, z >> 1, 32 * (z & 1) + (int)(r & 31), 4, (mx_u32x6)(0u), (mx_u32x6)(0u));
    return;
  }
  auto put = [&](auto type) {
    constexpr int T = decltype(type)::value, V = T == kF32 ? 4 : 8, LR = 16 * NT / V;
    for (int j = t; j < LR * rows.count; j += 64 * W) {
      const int m = j / LR, q = V * (j % LR), col = n0 + q;
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = total(m, q + i);
        if (o.bias != nullptr && col + i < n) v[i] += mx_load(o.bias, o.bias_type, col + i);
      }
      mx_put<T, V>(o, rows.first + m, ldy, col, n, v);
    }
  };
  if (o.y_type == kF32) put(MxType<kF32>{});
  else if (o.y_type == kF16) put(MxType<kF16>{});
  else put(MxType<kBF16>{});
}

// Tiles of up to 16 rows: a workgroup of W waves takes every gridDim.x-th group of NT 16-column
// tiles of the output and splits K over its waves by chunks (wave i: chunks i, i + W,
// ..., U of them in flight); the waves' sums meet in LDS, in wave order. GLU: half of the
// tiles are rows of o.w, half the same rows of `up`, and silu(first) * second of their 32
// columns becomes one block of the digit planes o.y.
// RAW: up to two rows, f32 (1) or 16 bits (2), quantized here (each wave its own chunks, a
// block a lane) into LDS; else digit planes.
//
// What bounds it: the weights' stream. A wave loads a chunk of a tile (2 KB) in two
// instructions, 16 waves a CU (128 registers a lane) ask for 32 KB at least at a time, and
// the next group's weights are on their way while this one's sums are joined. Keeping a
// wave's digits in registers from group to group took 156 registers and a second
// workgroup's place: 37 us against 24 for the gate and up of 24 tokens with 6 of 64 experts
// each, 2048 x 1408. One matrix instruction
// takes 16 columns x 128 of K by up to 16 rows, so rows cost nothing until their digits'
// reads show. Rows of x are read by every workgroup: quantized ahead into planes (1.5
// bytes a value) above two rows, in place below, where a launch of its own costs more
// than it takes (2.4 us and the gap).
template <int W, int NT, int U, bool GLU, int RAW>
__device__ __forceinline__ void mx_gemv(const MxOut& o, const uint8_t* __restrict__ up, const MxRows& rows, int n, int k,
                                        const uint8_t* __restrict__ xq, const MxRaw& raw, int ldy) {
  constexpr int NC = GLU ? NT / 2 : NT;  // 16-column tiles of the output
  static_assert(!GLU || NT == 4, "a block of 32 columns");
  constexpr int kRowF = 16 * NT + 4;     // floats of a row of sums, padded
  __shared__ __attribute__((aligned(16))) float red[W][16][kRowF];
  // RAW: [chunk][row][block] of 48 bytes of digits and a scale; a wave's chunks are its own
  extern __shared__ __attribute__((aligned(16))) uint8_t blocks[];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4, h = g & 1;
  const int kc = (k + kMxChunk - 1) / kMxChunk;
  const int groups = (n + 16 * NC - 1) / (16 * NC);
  const int xc = min(c, rows.count - 1);
  const uint8_t *xp = nullptr, *xs = nullptr;
  if constexpr (!RAW) {
    xp = xq + mx_x_at(rows.first + xc, h, kc) + (g >> 1) * kMxXStep;
    xs = xq + mx_xs_at(rows.first + xc, h, kc);
  }
  mx_u32x4 w[U][NT][2];
  int sw[U][NT];
  // x of chunk kk into slot u: planes are asked for together with the weights (loads return
  // in order), except with four tiles, whose weights leave no registers for them
  constexpr bool kAhead = !RAW && NT == 1;
  mx_u32x12 x[kAhead ? U : 1][2];
  int sx[kAhead ? U : 1][2];
  auto load_x = [&](int u, int kk) {
    if constexpr (RAW) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint8_t* d = blocks + 64 * (16 * kk + 8 * xc + 4 * q + g);
        x[u][q] = mx_x(*reinterpret_cast<const mx_u32x4*>(d), *reinterpret_cast<const mx_u32x4*>(d + 16),
                       *reinterpret_cast<const mx_u32x4*>(d + 32));
        sx[u][q] = *reinterpret_cast<const int*>(d + 48);
      }
    } else {
      const uint8_t* p = xp + (long long)kk * kMxXUnit;
      x[u][0] = mx_get_x(p);
      x[u][1] = mx_get_x(p + 2 * kMxXStep);
      sx[u][0] = *reinterpret_cast<const int*>(xs + (long long)kk * kMxXUnit) >> (8 * (g >> 1));
      sx[u][1] = sx[u][0] >> 16;
    }
  };
  auto load_one = [&](int grp, int kk, int u) {
    if (kAhead && kk >= kc) return;
    if constexpr (kAhead) load_x(u, kk);
    else kk = min(kk, kc - 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const long long r = rows.w0 + min(16 * (NC * grp + j % NC) + c, n - 1);
      const uint8_t* b = j < NC ? o.w : up;
      const uint8_t* wp = b + mx_w_at(r, h, kc) + (g >> 1) * kMxStepBytes + (long long)kk * kMxUnit;
      w[u][j][0] = *reinterpret_cast<const mx_u32x4*>(wp);
      w[u][j][1] = *reinterpret_cast<const mx_u32x4*>(wp + 2 * kMxStepBytes);
      sw[u][j] = *reinterpret_cast<const int*>(b + mx_ws_at(r, h, kc) + (long long)kk * kMxUnit);
    }
  };
  auto load_w = [&](int grp, int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) load_one(grp, k0 + W * u, u);
  };
  int grp = blockIdx.x;
  if constexpr (RAW) {
    // Lane 16 u + 8 row + block of four chunks. The first chunks' values are asked for
    // before the weights: loads return in order, and the weights come from afar.
    const int row = (lane >> 3) & 1, blk = lane & 7;
    const int r = rows.first + min(row, rows.count - 1);
    const long long src = (raw.src ? raw.src[r] : r) * raw.ldx;
    mx_u32x4 v[RAW == 1 ? 8 : 4];
    auto load = [&](int k0) {
      const int col = min(kMxChunk * (k0 + W * (lane >> 4)) + 32 * blk, k - 32);
      if (raw.wide) {
        const uint8_t* p = static_cast<const uint8_t*>(raw.x) + (src + col) * (RAW == 1 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < (RAW == 1 ? 8 : 4); ++i) v[i] = reinterpret_cast<const mx_u32x4*>(p)[i];
      } else if constexpr (RAW == 1) {
        const uint32_t* p = static_cast<const uint32_t*>(raw.x) + src + col;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i / 4][i % 4] = p[i];
      } else {
        const uint16_t* p = static_cast<const uint16_t*>(raw.x) + src + col;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i / 4][i % 4] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
      }
    };
    load(wave);
    load_w(grp, wave);
    for (int k0 = wave; k0 < kc; k0 += 4 * W) {
      if (k0 != wave) load(k0);
      const int kk = k0 + W * (lane >> 4);
      if (row < rows.count && kk < kc) {
        float f[32];
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if constexpr (RAW == 1) {
            const uint32_t u = v[i / 4][i % 4];
            f[i] = __builtin_bit_cast(float, u);
          } else {
            const uint16_t u = (uint16_t)(v[i / 8][i % 8 / 2] >> (16 * (i & 1)));
            f[i] = raw.type == kF16 ? (float)__builtin_bit_cast(_Float16, u) : bf16_to_f32(u);
          }
          amax = max(amax, __builtin_bit_cast(uint32_t, f[i]) & 0x7fffffffu);
        }
        const bool in = kMxChunk * kk + 32 * blk < k;  // (the last chunk's blocks past k are zero)
        if (!in) {
          amax = 0;
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = 0.0f;
        }
        mx_u32x6 hi, lo;
        const int e = mx_x_byte(amax);
        mx_digits(f, e, hi, lo);
        uint8_t* d = blocks + 64 * (16 * kk + 8 * row + blk);
        *reinterpret_cast<mx_u32x4*>(d) = mx_u32x4{hi[0], hi[1], hi[2], hi[3]};
        *reinterpret_cast<mx_u32x4*>(d + 16) = mx_u32x4{hi[4], hi[5], lo[0], lo[1]};
        *reinterpret_cast<mx_u32x4*>(d + 32) = mx_u32x4{lo[2], lo[3], lo[4], lo[5]};
        *reinterpret_cast<int*>(d + 48) = e;
      }
    }
    __builtin_amdgcn_wave_barrier();
  } else {
    load_w(grp, wave);
  }
#pragma unroll 1
  for (; grp < groups; grp += gridDim.x) {
    mx_f32x4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = (mx_f32x4)(0.0f);
#pragma unroll 1
    for (int k0 = wave; k0 < kc; k0 += W * U) {
      // the next chunks of this group or the next group's first
      const bool more = k0 + W * U < kc;
      const bool any = more || grp + (int)gridDim.x < groups;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kk = k0 + W * u;
        if (kk < kc) {
          constexpr int X = kAhead ? 1 : 0;
          if constexpr (!kAhead) load_x(0, kk);
          const int s0 = sx[X * u][0] & 255, s1 = sx[X * u][1] & 255;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const int b = sw[u][j] >> (8 * (g >> 1));  // block 2 s + h of steps s = g / 2 and 2 + g / 2
            acc[j] = mx_mfma16<0>(w[u][j][0], mx_hi(x[X * u][0]), acc[j], b, s0);
            acc[j] = mx_mfma16<0>(w[u][j][0], mx_lo(x[X * u][0]), acc[j], b, s0 - 4);
            acc[j] = mx_mfma16<0>(w[u][j][1], mx_hi(x[X * u][1]), acc[j], b >> 16, s1);
            acc[j] = mx_mfma16<0>(w[u][j][1], mx_lo(x[X * u][1]), acc[j], b >> 16, s1 - 4);
          }
        }
        if (any) load_one(more ? grp : grp + (int)gridDim.x, (more ? k0 + W * U : wave) + W * u, u);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<mx_f32x4*>(&red[wave][c][16 * j + 4 * g]) = acc[j];
    __syncthreads();
    mx_gemv_join<W, NT, GLU>(o, rows, n, 16 * NC * grp, red, ldy);
    __syncthreads();
  }
}

// A tile of 32 FM WM rows x 32 FN WN columns by WM x WN waves, a wave FM x FN fragments;
// WK such groups of waves share the columns of x (K) by chunks and join their sums.
// GLU: half of a wave's column fragments are rows of o.w, half the same rows of `up`, and
// silu(first) * second becomes digit planes (o.y), the down product's input.
//
// What bounds it: the matrix cores' power. 4096 rows x 16384 x 8192 takes 564 us, 1.95
// PFLOP/s of products and twice that of instructions; without any loads or LDS the same
// instructions take 414 us on random values (and 272 us on zeros: the clock falls with
// the values' toggling). Per step (64 columns) a wave issues 2 FM FN instructions of 32
// cycles. x goes through LDS (two buffers, one barrier a step): the waves of a column
// of the tile share it. The weights go straight to registers: a step's operand is 1 KB
// contiguous, and the LDS has no time for them (reads of x alone take 384 of the 1024
// cycles of a step on a CU). The first half of a step's fragments of x is read in the
// second half of the step before, the second half in the first: neither waits. Two
// workgroups a CU, so that one's barrier and epilogue fall into the other's products:
// 327 us at K = 4096 against 360 with one 256 x 256 workgroup of four waves (128 x 128
// a wave, sums in the second register file). x straight to LDS without registers
// measured the same (339 us, and two steps ahead in four buffers 339 us).
template <int FM, int FN, int WM, int WN, int WK, bool GLU>
__device__ __forceinline__ void mx_gemm(const MxOut& o, const uint8_t* __restrict__ up, const MxRows& rows, int n, int kc,
                                        int n0, const uint8_t* __restrict__ xq, int ldy) {
  constexpr int NW = WM * WN, XF = FM * WM, FW = XF / NW;
  constexpr int FC = GLU ? FN / 2 : FN;  // column fragments of a wave's output
  static_assert(XF % NW == 0 && FM % 2 == 0 && (!GLU || (FN == 4 && WK == 1)), "whole fragments a wave");
  constexpr int kStage = XF * kMxXStep;
  // the epilogue's 32 rows of a wave's columns, a row padded by 16 bytes
  constexpr int kRow = 32 * FC + 4, kLoop = 2 * WK * kStage, kEpi = WK * NW * 32 * kRow * 4;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kLoop > kEpi ? kLoop : kEpi];
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = all / NW, wave = all % NW;
  auto lds = reinterpret_cast<uint8_t(*)[kStage]>(smem + 2 * kStage * wk);
  const int h = lane >> 5, c = lane & 31, wm = wave % WM, wn = wave / WM;
  // 64-bit bases at the tile's first row, 32-bit offsets from them
  const long long xt = rows.first >> 5;
  const uint8_t* xb = xq + xt * ((long long)kc * kMxXUnit);
  unsigned xo[FW], xso[FM], wo[FC], wso[FC];
#pragma unroll
  for (int j = 0; j < FW; ++j)  // the fragments that this wave brings to LDS
    xo[j] = (unsigned)mx_x_at(rows.first + min(32 * (FW * wave + j) + c, rows.count - 1) - 32 * xt, h, kc);
#pragma unroll
  for (int b = 0; b < FM; ++b)
    xso[b] = (unsigned)mx_xs_at(rows.first + min(32 * (WM * b + wm) + c, rows.count - 1) - 32 * xt, h, kc);
  const long long wt = (rows.w0 + n0) >> 5;
  const uint8_t* wb[2] = {o.w + wt * ((long long)kc * kMxUnit), GLU ? up + wt * ((long long)kc * kMxUnit) : nullptr};
#pragma unroll
  for (int a = 0; a < FC; ++a) {
    const long long r = rows.w0 + min(n0 + 32 * (FC * wn + a) + c, n - 1) - 32 * wt;
    wo[a] = (unsigned)mx_w_at(r, h, kc);
    wso[a] = (unsigned)mx_ws_at(r, h, kc);
  }
  mx_f32x16 acc[FN][FM];
#pragma unroll
  for (int a = 0; a < FN; ++a)
#pragma unroll
    for (int b = 0; b < FM; ++b) acc[a][b] = (mx_f32x16)(0.0f);

  mx_u32x4 st[3 * FW];   // x on its way to LDS
  mx_u32x4 w[2][FN];     // weights of this step and the next
  mx_u32x12 x[FM];       // x of this step
  int sw[2][FN], sx[2][FM];
  auto load_x = [&](int k, int s) {
    const unsigned at = (unsigned)k * kMxXUnit + s * kMxXStep;
#pragma unroll
    for (int i = 0; i < 3 * FW; ++i)
      st[i] = *reinterpret_cast<const mx_u32x4*>(xb + (xo[i / 3] + at) + kMxXPart * (i % 3));
  };
  auto put_x = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 3 * FW; ++i)
      *reinterpret_cast<mx_u32x4*>(&lds[buf][kMxXPart * (3 * FW * wave + i) + 16 * lane]) = st[i];
  };
  auto get_x = [&](int buf, int b0, int b1) {
#pragma unroll
    for (int b = b0; b < b1; ++b) x[b] = mx_get_x(&lds[buf][kMxXStep * (WM * b + wm) + 16 * lane]);
  };
  auto load_w = [&](int k, int s, mx_u32x4 (&d)[FN]) {
    const unsigned at = (unsigned)k * kMxUnit + s * kMxStepBytes;
#pragma unroll
    for (int a = 0; a < FN; ++a) d[a] = *reinterpret_cast<const mx_u32x4*>(wb[a / FC] + (wo[a % FC] + at));
  };
  auto load_s = [&](int k, int i) {
#pragma unroll
    for (int a = 0; a < FN; ++a)
      sw[i][a] = *reinterpret_cast<const int*>(wb[a / FC] + (wso[a % FC] + (unsigned)k * kMxUnit));
#pragma unroll
    for (int b = 0; b < FM; ++b) sx[i][b] = *reinterpret_cast<const int*>(xb + (xso[b] + (unsigned)k * kMxXUnit));
  };
  auto sync = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's writes are in LDS
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // this group's chunks; every group makes as many rounds, so that the barriers match
  const int per = (kc + WK - 1) / WK, k0 = min(per * wk, kc - 1), live = min(per, kc - per * wk);
  // A wave's fragments of rows are wm, wm + WM, ...: a tile with few rows is spread over
  // its waves, and fragments without rows are left out.
  const int full = min((rows.count + 32 * (WM - wm) - 1) / (32 * WM), FM);
  load_s(k0, 0);
  load_x(k0, 0);
  load_w(k0, 0, w[0]);
  put_x(0);
  load_x(k0, 1);
  sync();
  get_x(0, 0, FM / 2);
#define QMM_MX_HALF(S, B0, B1)                                                                                 \
  _Pragma("unroll") for (int b = B0; b < B1; ++b) if (b < have) {                                              \
    _Pragma("unroll") for (int a = 0; a < FN; ++a) acc[a][b] =                                                 \
        mx_mfma<S>(w[S & 1][a], mx_hi(x[b]), acc[a][b], sw[0][a], sx[0][b]);                                   \
    _Pragma("unroll") for (int a = 0; a < FN; ++a) acc[a][b] =                                                 \
        mx_mfma<S>(w[S & 1][a], mx_lo(x[b]), acc[a][b], sw[0][a], sx[0][b] - kMxLoScale);                      \
  }
#define QMM_MX_STEP(S)                                                                                         \
  {                                                                                                            \
    put_x((S + 1) & 1);                                                                                        \
    load_x(S + 2 < 4 ? k : kn, (S + 2) & 3);                                                                   \
    load_w(S + 1 < 4 ? k : kn, (S + 1) & 3, w[(S + 1) & 1]);                                                   \
    if (S == 1) load_s(kn, 1);                                                                                 \
    get_x(S & 1, FM / 2, FM);                                                                                  \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
    QMM_MX_HALF(S, 0, FM / 2)                                                                                  \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
    sync();                                                                                                    \
    get_x((S + 1) & 1, 0, FM / 2);                                                                             \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
    QMM_MX_HALF(S, FM / 2, FM)                                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
  }
  // (past the last chunk the loads read it again, and what they bring is not used)
#pragma unroll 1
  for (int i = 0; i < per; ++i) {
    const int k = min(k0 + i, kc - 1), kn = min(k0 + i + 1, kc - 1);
    const int have = WK == 1 || i < live ? full : 0;
    QMM_MX_STEP(0)
    QMM_MX_STEP(1)
    QMM_MX_STEP(2)
    QMM_MX_STEP(3)
#pragma unroll
    for (int a = 0; a < FN; ++a) sw[0][a] = sw[1][a];
#pragma unroll
    for (int b = 0; b < FM; ++b) sx[0][b] = sx[1][b];
  }
#undef QMM_MX_STEP
#undef QMM_MX_HALF
  sync();
  float* e = reinterpret_cast<float*>(smem) + all * 32 * kRow;
  const int col0 = n0 + 32 * FC * wn;
  if constexpr (GLU) {
    // silu(g) * u of 64 columns: one step of a chunk of the planes, a block a lane
    if (col0 >= n) return;
    const int hb = h, kf = (n + kMxChunk - 1) / kMxChunk, s = col0 % kMxChunk / 64;
    const bool last = col0 + 64 >= n;
#pragma unroll
    for (int b = 0; b < FM; ++b) {
#pragma unroll
      for (int a = 0; a < FC; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mx_f32x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float g = acc[a][b][4 * i + j];
            v[j] = g / (1.0f + expf(-g)) * acc[a + FC][b][4 * i + j];
          }
          *reinterpret_cast<mx_f32x4*>(e + c * kRow + 32 * a + 8 * i + 4 * h) = v;
        }
      __builtin_amdgcn_wave_barrier();
      const int m = 32 * (WM * b + wm) + c;
      float v[32];
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const mx_f32x4 t = *reinterpret_cast<const mx_f32x4*>(e + c * kRow + 32 * hb + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[4 * j + i] = t[i];
          amax = max(amax, __builtin_bit_cast(uint32_t, v[4 * j + i]) & 0x7fffffffu);
        }
      }
      __builtin_amdgcn_wave_barrier();
      mx_u32x6 hi = (mx_u32x6)(0u), lo = (mx_u32x6)(0u);
      int byte = 4;
      if (col0 + 32 * hb < n) {
        byte = mx_x_byte(amax);
        mx_digits(v, byte, hi, lo);
      }
      if (m < rows.count) {
        const long long r = rows.first + m;
        uint8_t* u = static_cast<uint8_t*>(o.y) + ((r >> 5) * kf + col0 / kMxChunk) * kMxXUnit;
        const int l = 32 * hb + (int)(r & 31);
        mx_put_block(u, s, l, byte, hi, lo);
        if (last)  // the rest of the chunk: the product reads whole ones
          for (int z = s + 1; z < 4; ++z) mx_put_block(u, z, l, 4, (mx_u32x6)(0u), (mx_u32x6)(0u));
      }
    }
    return;
  }
  // The accumulators hold four columns of a row a lane; through LDS a wave writes 16
  // bytes a lane, whole runs of a row's 32 FN columns (writing them as they are, 8 bytes
  // a lane over 32 rows, took 36 us a 256 x 256 tile).
  auto put = [&](auto type) {
    constexpr int T = decltype(type)::value;
    constexpr int V = T == kF32 ? 4 : 8, LR = 32 * FN / V;  // columns and lanes of a 16-byte run and of a row
    constexpr int R = 32 / WK;  // rows that this group joins and writes
    const int q = V * (lane % LR);
    float bias[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      bias[j] = o.bias != nullptr && col0 + q + j < n ? mx_load(o.bias, o.bias_type, col0 + q + j) : 0.0f;
#pragma unroll
    for (int b = 0; b < FM; ++b) {
#pragma unroll
      for (int a = 0; a < FN; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<mx_f32x4*>(e + c * kRow + 32 * a + 8 * i + 4 * h) =
              mx_f32x4{acc[a][b][4 * i], acc[a][b][4 * i + 1], acc[a][b][4 * i + 2], acc[a][b][4 * i + 3]};
      if constexpr (WK == 1) __builtin_amdgcn_wave_barrier();
      else sync();
#pragma unroll 4
      for (int r = R * wk + lane / LR; r < R * wk + R; r += 64 / LR) {
        const int m = 32 * (WM * b + wm) + r;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          mx_f32x4 t = (mx_f32x4)(0.0f);
#pragma unroll
          for (int g = 0; g < WK; ++g)  // the groups' sums in order
            t += *reinterpret_cast<const mx_f32x4*>(e + (g - wk) * (NW * 32 * kRow) + r * kRow + q + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j + i] = t[i] + bias[j + i];
        }
        if (m < rows.count) mx_put<T, V>(o, rows.first + m, ldy, col0 + q, n, v);
      }
      if constexpr (WK == 1) __builtin_amdgcn_wave_barrier();
      else sync();
    }
  };
  if (o.y_type == kF32) put(MxType<kF32>{});
  else if (o.y_type == kF16) put(MxType<kF16>{});
  else put(MxType<kBF16>{});
}
}  // namespace qmm

// Grid: workgroups that share the columns, row tiles.
#define QMM_MX_GEMV(W, NT, U, NAME, RAW)                                                                       \
  extern "C" __global__ void __launch_bounds__(64 * W, 4) qmm_mx_gemv##NAME##_w##W##_n##NT##_u##U(             \
      qmm::MxOut o, int m, int n, int k, const uint8_t* __restrict__ xq, qmm::MxRaw raw, int ldy) {            \
    const qmm::MxRows r = {0, 16 * (int)blockIdx.y, min(16, m - 16 * (int)blockIdx.y)};                        \
    qmm::mx_gemv<W, NT, U, false, RAW>(o, nullptr, r, n, k, xq, raw, ldy);                                     \
  }
#define QMM_MX_EXPERT_GEMV(W, NT, U)                                                                           \
  extern "C" __global__ void __launch_bounds__(64 * W, 4) qmm_mx_expert_gemv_w##W##_n##NT##_u##U(              \
      qmm::MxOut o0, qmm::MxOut o1, int experts, int pairs, int n, int k, const int* __restrict__ counts,      \
      const int* __restrict__ offsets, const uint8_t* __restrict__ xq, int ldy) {                              \
    qmm::MxRows r;                                                                                             \
    if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 16, blockIdx.y, r)) return;                   \
    qmm::mx_gemv<W, NT, U, false, 0>(blockIdx.z ? o1 : o0, nullptr, r, n, k, xq, qmm::MxRaw{}, ldy);           \
  }
// Gate and up with the activation: dense rows (experts 0) or routed ones.
#define QMM_MX_GLU_GEMV(W, NAME, RAW)                                                                          \
  extern "C" __global__ void __launch_bounds__(64 * W, 4) qmm_mx_glu_gemv##NAME##_w##W(                        \
      qmm::MxOut o, const uint8_t* __restrict__ up, int experts, int pairs, int n, int k,                      \
      const int* __restrict__ counts, const int* __restrict__ offsets, const uint8_t* __restrict__ xq,         \
      qmm::MxRaw raw) {                                                                                        \
    qmm::MxRows r = {0, 16 * (int)blockIdx.y, min(16, pairs - 16 * (int)blockIdx.y)};                          \
    if (experts > 0 && !qmm::mx_expert_tile(counts, offsets, experts, pairs, n, RAW ? 2 : 16, blockIdx.y, r)) return;  \
    qmm::mx_gemv<W, 4, 1, true, RAW>(o, up, r, n, k, xq, raw, 0);                                              \
  }
#define QMM_MX_GEMVS(W)              \
  QMM_MX_GEMV(W, 1, 1, , 0)          \
  QMM_MX_GEMV(W, 4, 1, , 0)          \
  QMM_MX_GEMV(W, 1, 1, _raw32, 1)    \
  QMM_MX_GEMV(W, 1, 2, _raw32, 1)    \
  QMM_MX_GEMV(W, 1, 1, _raw16, 2)    \
  QMM_MX_GEMV(W, 1, 2, _raw16, 2)    \
  QMM_MX_EXPERT_GEMV(W, 1, 1)        \
  QMM_MX_EXPERT_GEMV(W, 4, 1)        \
  QMM_MX_GLU_GEMV(W, , 0)            \
  QMM_MX_GLU_GEMV(W, _raw32, 1)      \
  QMM_MX_GLU_GEMV(W, _raw16, 2)
QMM_MX_GEMVS(4)
QMM_MX_GEMVS(8)
QMM_MX_GEMVS(16)
// (planes of one column tile a group that has more chunks than waves get all 16)
QMM_MX_GEMV(16, 1, 2, , 0)
QMM_MX_EXPERT_GEMV(16, 1, 2)

#define QMM_MX_GEMM(NAME, FM, FN, WM, WN, WK, EU)                                                              \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN * WK, EU) qmm_mx_gemm_##NAME(                      \
      qmm::MxOut o, int m, int n, int kc, const uint8_t* __restrict__ xq, int ldy) {                           \
    const int first = 32 * FM * WM * blockIdx.y;                                                               \
    const qmm::MxRows r = {0, first, min(m - first, 32 * FM * WM)};                                            \
    qmm::mx_gemm<FM, FN, WM, WN, WK, false>(o, nullptr, r, n, kc, 32 * FN * WN * blockIdx.x, xq, ldy);         \
  }                                                                                                            \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN * WK, EU) qmm_mx_expert_gemm_##NAME(               \
      qmm::MxOut o0, qmm::MxOut o1, int experts, int pairs, int n, int kc, const int* __restrict__ counts,     \
      const int* __restrict__ offsets, const uint8_t* __restrict__ xq, int ldy) {                              \
    qmm::MxRows r;                                                                                             \
    if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 32 * FM * WM, blockIdx.y, r)) return;         \
    qmm::mx_gemm<FM, FN, WM, WN, WK, false>(blockIdx.z ? o1 : o0, nullptr, r, n, kc, 32 * FN * WN * blockIdx.x, xq,  \
                                            ldy);                                                              \
  }
QMM_MX_GEMM(128x256, 2, 4, 2, 2, 1, 2)
QMM_MX_GEMM(128x128, 2, 2, 2, 2, 1, 2)
QMM_MX_GEMM(64x128k4, 2, 2, 1, 2, 4, 2)

// Gate and up with the activation, into the planes of the down product's rows: dense
// rows, or routed ones.
extern "C" __global__ void __launch_bounds__(256, 2) qmm_mx_glu_128x128(qmm::MxOut o, const uint8_t* __restrict__ up,
                                                                       int m, int n, int kc,
                                                                       const uint8_t* __restrict__ xq) {
  const int first = 128 * blockIdx.y;
  const qmm::MxRows r = {0, first, min(m - first, 128)};
  qmm::mx_gemm<2, 4, 2, 2, 1, true>(o, up, r, n, kc, 128 * blockIdx.x, xq, 0);
}
extern "C" __global__ void __launch_bounds__(256, 2) qmm_mx_expert_glu_128x128(
    qmm::MxOut o, const uint8_t* __restrict__ up, int experts, int pairs, int n, int kc, const int* __restrict__ counts,
    const int* __restrict__ offsets, const uint8_t* __restrict__ xq) {
  qmm::MxRows r;
  if (!qmm::mx_expert_tile(counts, offsets, experts, pairs, n, 128, blockIdx.y, r)) return;
  qmm::mx_gemm<2, 4, 2, 2, 1, true>(o, up, r, n, kc, 128 * blockIdx.x, xq, 0);
}

// The down products of a token's experts and their weighted sum in one launch, for a
// token or two: out[t] = sum over t's pairs, in increasing expert order, of weight *
// down(h[pair]), then + shared[t] (times sg[t]), rounded once. Grid: 16-column groups,
// tokens. The pairs' chunks are one list that 16 waves split (wave i: chunks i, i + 16, ...,
// two in flight), a wave's sums of a pair are scaled when the list leaves it, and the waves'
// sums meet in LDS, in wave order.
//
// What bounds it: the weights' stream and its beginning. One token's two experts of 4096 x
// 14336 (62 MB): 13.7 us, against 12.9 and 3.9 of products by pair and their sum; the call
// 43.7 us against 45.7, with 6 of 64 experts of 2048 x 1408 23.3 against 26.2. Two tokens read
// an expert that both chose twice: 67.0 us against 64.8, and 32.6 against 37.2 (8 of 64).
extern "C" __global__ void __launch_bounds__(1024, 4)
    qmm_mx_down_sum(qmm::MxOut o, int experts, int topk, int n, int k, const int* __restrict__ counts,
                    const int* __restrict__ offsets, const int* __restrict__ token_pairs,
                    const float* __restrict__ pair_weight, const uint8_t* __restrict__ hq,
                    const float* __restrict__ shared, const float* __restrict__ sg, long long ldo) {
  using namespace qmm;
  constexpr int W = 16, U = 2, kPairs = 32;
  __shared__ int expert[kPairs];
  __shared__ __attribute__((aligned(16))) float red[W][16];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4, h = g & 1, token = blockIdx.y;
  const int* pairs = token_pairs + (long long)token * topk;
  for (int s = wave; s < topk; s += W) {  // the expert that holds row p of the list
    const int p = pairs[s];
    if (lane == 0) expert[s] = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
      const int e = e0 + lane;
      if (e < experts && p >= offsets[e] && p < offsets[e] + counts[e]) expert[s] = e;
    }
  }
  __syncthreads();
  const int kc = (k + kMxChunk - 1) / kMxChunk, col = min(16 * (int)blockIdx.x + c, n - 1);
  mx_u32x4 w[U][2];
  mx_u32x12 x[U][2];
  int sw[U], sx[U];
  auto load = [&](int u, int s, int kk) {
    const int p = __builtin_amdgcn_readfirstlane(pairs[s]);
    const long long r = (long long)__builtin_amdgcn_readfirstlane(expert[s]) * n + col;
    const uint8_t* xp = hq + mx_x_at(p, h, kc) + (g >> 1) * kMxXStep + (long long)kk * kMxXUnit;
    x[u][0] = mx_get_x(xp);
    x[u][1] = mx_get_x(xp + 2 * kMxXStep);
    sx[u] = *reinterpret_cast<const int*>(hq + mx_xs_at(p, h, kc) + (long long)kk * kMxXUnit);
    const uint8_t* wp = o.w + mx_w_at(r, h, kc) + (g >> 1) * kMxStepBytes + (long long)kk * kMxUnit;
    w[u][0] = *reinterpret_cast<const mx_u32x4*>(wp);
    w[u][1] = *reinterpret_cast<const mx_u32x4*>(wp + 2 * kMxStepBytes);
    sw[u] = *reinterpret_cast<const int*>(o.w + mx_ws_at(r, h, kc) + (long long)kk * kMxUnit);
  };
  int s = wave / kc, kk = wave % kc;  // the chunk in turn, and the one to load
  int sl = s, kl = kk;
  auto next = [&](int& s, int& kk) {
    kk += W;
    while (kk >= kc) {
      kk -= kc;
      ++s;
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (sl < topk) load(u, sl, kl);
    next(sl, kl);
  }
  mx_f32x4 sum = (mx_f32x4)(0.0f), acc = (mx_f32x4)(0.0f);
  auto weight = [&](int s) { return pair_weight[__builtin_amdgcn_readfirstlane(pairs[s])]; };
  int cur = s;
#pragma unroll 1
  while (s < topk) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s >= topk) break;
      if (s != cur) {
        sum += weight(cur) * acc;
        acc = (mx_f32x4)(0.0f);
        cur = s;
      }
      const int b = sw[u] >> (8 * (g >> 1)), e = sx[u] >> (8 * (g >> 1));
      const int s0 = e & 255, s1 = e >> 16 & 255;
      acc = mx_mfma16<0>(w[u][0], mx_hi(x[u][0]), acc, b, s0);
      acc = mx_mfma16<0>(w[u][0], mx_lo(x[u][0]), acc, b, s0 - 4);
      acc = mx_mfma16<0>(w[u][1], mx_hi(x[u][1]), acc, b >> 16, s1);
      acc = mx_mfma16<0>(w[u][1], mx_lo(x[u][1]), acc, b >> 16, s1 - 4);
      next(s, kk);
      if (sl < topk) load(u, sl, kl);
      next(sl, kl);
    }
  }
  if (cur < topk) sum += weight(cur) * acc;
  if (c == 0) *reinterpret_cast<mx_f32x4*>(&red[wave][4 * g]) = sum;
  __syncthreads();
  const int q = 16 * (int)blockIdx.x + t;
  if (t >= 16 || q >= n) return;
  float v = red[0][t];
#pragma unroll
  for (int i = 1; i < W; ++i) v += red[i][t];
  if (shared != nullptr) v += (sg != nullptr ? sg[token] : 1.0f) * shared[(long long)token * n + q];
  mx_store(o.y, o.y_type, token * ldo + q, v);
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

// Quantizers, converters and readers of the microscaled types (formats and layouts:
// qmm_mx_common.h). All are bound by memory: one pass, each value read once.
#pragma once

#include "qmm_mx_common.h"

namespace qmm {

// Weight units are made by one workgroup each (32 rows x 256 columns), thread
// 64 s + 32 h + r the block 2 s + h of row r: its 16 bytes of codes are written where
// the unit has them, so a wave writes 1 KB at once. The unit's values go through LDS,
// where a row is 260 floats so that 8 rows' 16-byte reads fall on distinct banks.
constexpr int kMxLdsRow = kMxChunk + 4;

__device__ __forceinline__ void mx_put_unit(uint8_t* __restrict__ unit, uint8_t (&sc)[256], int t, mx_u32x4 q, int e) {
  *reinterpret_cast<mx_u32x4*>(unit + 16 * t) = q;
  sc[4 * (t & 63) + (t >> 6)] = (uint8_t)e;
  __syncthreads();
  if (t < 64)
    *reinterpret_cast<uint32_t*>(unit + kMxScaleOff + 4 * t) = *reinterpret_cast<const uint32_t*>(sc + 4 * t);
}

// E2M1 codes of 32 values, value j in nibble j.
__device__ __forceinline__ mx_u32x4 mx_codes(const float (&x)[32], int e) {
  mx_u32x4 q;
  const int up = 127 - e;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    int v = 0;
#define QMM_MX_CVT(B)                                                                                       \
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, e == kMxNan ? 0.0f : __builtin_ldexpf(x[8 * w + 2 * B], up), \
                                               e == kMxNan ? 0.0f : __builtin_ldexpf(x[8 * w + 2 * B + 1], up), 1.0f, B)
    QMM_MX_CVT(0);
    QMM_MX_CVT(1);
    QMM_MX_CVT(2);
    QMM_MX_CVT(3);
#undef QMM_MX_CVT
    q[w] = (uint32_t)v;
  }
  return q;
}

// Four values of a typed matrix at element `at`; `wide`: they lie on a boundary of four.
template <int T>
__device__ __forceinline__ mx_f32x4 mx_load4(const void* __restrict__ p, long long at, bool wide) {
  mx_f32x4 v;
  if constexpr (T == kF32) {
    const float* q = static_cast<const float*>(p) + at;
    if (wide) return *reinterpret_cast<const mx_f32x4*>(q);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = q[j];
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    uint16_t s[4];
    if (wide) {
      const mx_u32x2 d = *reinterpret_cast<const mx_u32x2*>(q);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = (uint16_t)(d[j >> 1] >> (16 * (j & 1)));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = q[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = T == kF16 ? (float)__builtin_bit_cast(_Float16, s[j]) : bf16_to_f32(s[j]);
  }
  return v;
}

// This thread's block of a unit whose rows are in `buf`: its values and largest magnitude.
__device__ __forceinline__ uint32_t mx_unit_block(const float* buf, int t, float (&x)[32]) {
  const float* p = buf + (t & 31) * kMxLdsRow + 64 * (t >> 6) + (t & 32);
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const mx_f32x4 v = *reinterpret_cast<const mx_f32x4*>(p + 4 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[4 * j + i] = v[i];  // (a bit cast of the vector's own element would take its first one)
      amax = max(amax, __builtin_bit_cast(uint32_t, x[4 * j + i]) & 0x7fffffffu);
    }
  }
  return amax;
}

template <int T>
__device__ __forceinline__ void mx_quantize_w(const void* __restrict__ w, int n, int k, uint8_t* __restrict__ out,
                                              int kc) {
  __shared__ __attribute__((aligned(16))) float buf[kMxTile * kMxLdsRow];
  __shared__ __attribute__((aligned(16))) uint8_t sc[256];
  const int t = threadIdx.x;
  const long long u = blockIdx.x;
  const int r0 = (int)(u / kc) * kMxTile, c0 = (int)(u % kc) * kMxChunk;
  // four values a thread and row, whole rows of the unit by a wave (k % 32 == 0)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (t >> 6), c = 4 * (t & 63);
    mx_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r0 + r < n && c0 + c < k) v = mx_load4<T>(w, (long long)(r0 + r) * k + c0 + c, true);
    *reinterpret_cast<mx_f32x4*>(buf + r * kMxLdsRow + c) = v;
  }
  __syncthreads();
  float x[32];
  const int e = mx_w_byte(mx_unit_block(buf, t, x));
  mx_put_unit(out + u * kMxUnit, sc, t, mx_codes(x, e), e);
}

// The code's value of E2M1, doubled.
__device__ __forceinline__ int mx_twice(uint32_t code) {
  const int m = (int)((0xC8643210u >> (4 * (code & 7))) & 15u);
  return code & 8 ? -m : m;
}
// twice the value, under scale byte e (255: NaN); exact in f32 down to its smallest subnormal
__device__ __forceinline__ float mx_value(uint32_t code, int e) {
  return e == kMxNan ? __builtin_nanf("") : __builtin_ldexpf((float)mx_twice(code), e - 128);
}

}  // namespace qmm

#define QMM_MX_QUANTIZE_W(NAME, T)                                                                                \
  extern "C" __global__ void __launch_bounds__(256) qmm_mx_quantize_w_##NAME(                                     \
      const void* __restrict__ w, int n, int k, uint8_t* __restrict__ out, int kc) {                              \
    qmm::mx_quantize_w<T>(w, n, k, out, kc);                                                                      \
  }
QMM_MX_QUANTIZE_W(f32, qmm::kF32)
QMM_MX_QUANTIZE_W(f16, qmm::kF16)
QMM_MX_QUANTIZE_W(bf16, qmm::kBF16)

// GGML blocks -> units, and back. Load time only: byte reads of 17-byte blocks.
extern "C" __global__ void __launch_bounds__(256) qmm_mx_from_ggml(const uint8_t* __restrict__ src, int n, int k,
                                                                   uint8_t* __restrict__ out, int kc) {
  __shared__ __attribute__((aligned(16))) uint8_t sc[256];
  const int t = threadIdx.x;
  const long long u = blockIdx.x;
  const int row = (int)(u / kc) * qmm::kMxTile + (t & 31);
  const int blk = (int)(u % kc) * 8 + 2 * (t >> 6) + ((t >> 5) & 1);
  qmm::mx_u32x4 q = {0, 0, 0, 0};
  int e = 0;
  if (row < n && blk < k / 32) {
    const uint8_t* b = src + ((long long)row * (k / 32) + blk) * qmm::kMxFp4Bytes;
    e = b[0];
#pragma unroll
    for (int j = 0; j < 16; ++j) {  // byte j: value j low, value j + 16 high
      const uint32_t v = b[1 + j];
      q[j >> 3] |= (v & 15u) << (4 * (j & 7));
      q[2 + (j >> 3)] |= (v >> 4) << (4 * (j & 7));
    }
  }
  qmm::mx_put_unit(out + u * qmm::kMxUnit, sc, t, q, e);
}

extern "C" __global__ void __launch_bounds__(256) qmm_mx_to_ggml(const uint8_t* __restrict__ w, int n, int k,
                                                                 uint8_t* __restrict__ dst, int kc) {
  const int t = threadIdx.x;
  const long long u = blockIdx.x;
  const int row = (int)(u / kc) * qmm::kMxTile + (t & 31);
  const int blk = (int)(u % kc) * 8 + 2 * (t >> 6) + ((t >> 5) & 1);
  if (row >= n || blk >= k / 32) return;
  const uint8_t* p = w + u * qmm::kMxUnit;
  const qmm::mx_u32x4 q = *reinterpret_cast<const qmm::mx_u32x4*>(p + 16 * t);
  uint8_t* b = dst + ((long long)row * (k / 32) + blk) * qmm::kMxFp4Bytes;
  b[0] = p[qmm::kMxScaleOff + 4 * (t & 63) + (t >> 6)];
#pragma unroll
  for (int j = 0; j < 16; ++j)
    b[1 + j] = (uint8_t)((q[j >> 3] >> (4 * (j & 7)) & 15u) | (q[2 + (j >> 3)] >> (4 * (j & 7)) & 15u) << 4);
}

namespace qmm {
// Units -> dense [n, k], each value rounded once to the output type. A unit's values go
// through LDS so that a wave writes whole rows of it.
template <int T>
__device__ __forceinline__ void mx_dequantize(const uint8_t* __restrict__ w, int n, int k, void* __restrict__ dst,
                                              int kc) {
  __shared__ __attribute__((aligned(16))) float buf[kMxTile * kMxLdsRow];
  const int t = threadIdx.x;
  const long long u = blockIdx.x;
  const uint8_t* p = w + u * kMxUnit;
  const mx_u32x4 q = *reinterpret_cast<const mx_u32x4*>(p + 16 * t);
  const int e = p[kMxScaleOff + 4 * (t & 63) + (t >> 6)];
  float* o = buf + (t & 31) * kMxLdsRow + 64 * (t >> 6) + (t & 32);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    mx_f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mx_value(q[j >> 1] >> (16 * (j & 1) + 4 * i), e);
    *reinterpret_cast<mx_f32x4*>(o + 4 * j) = v;
  }
  __syncthreads();
  const int r0 = (int)(u / kc) * kMxTile, c = (int)(u % kc) * kMxChunk + 4 * (t & 63);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (t >> 6);
    if (r0 + r >= n || c >= k) continue;
    const mx_f32x4 v = *reinterpret_cast<const mx_f32x4*>(buf + r * kMxLdsRow + 4 * (t & 63));
    const long long at = (long long)(r0 + r) * k + c;
    if constexpr (T == kF32) {
      *reinterpret_cast<mx_f32x4*>(static_cast<float*>(dst) + at) = v;
    } else {
      *reinterpret_cast<mx_u32x2*>(static_cast<uint16_t*>(dst) + at) =
          mx_u32x2{mx_to16(v[0], T) | (uint32_t)mx_to16(v[1], T) << 16, mx_to16(v[2], T) | (uint32_t)mx_to16(v[3], T) << 16};
    }
  }
}

// 32 consecutive f32 values. `wide`: they start on a 16-byte boundary.
__device__ __forceinline__ uint32_t mx_load_block(const float* __restrict__ p, bool wide, float (&x)[32]) {
  uint32_t amax = 0;
  if (wide) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const mx_f32x4 v = reinterpret_cast<const mx_f32x4*>(p)[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * j + i] = v[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = p[j];
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) amax = max(amax, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
  return amax;
}

// This thread's block of a unit of digit planes.
__device__ __forceinline__ void mx_put_digits(uint8_t* __restrict__ unit, uint8_t (&sc)[256], int t, int e,
                                              const mx_u32x6& hi, const mx_u32x6& lo) {
  uint8_t* o = unit + (t >> 6) * kMxXStep + 16 * (t & 63);
  *reinterpret_cast<mx_u32x4*>(o) = mx_u32x4{hi[0], hi[1], hi[2], hi[3]};
  *reinterpret_cast<mx_u32x4*>(o + kMxXPart) = mx_u32x4{hi[4], hi[5], lo[0], lo[1]};
  *reinterpret_cast<mx_u32x4*>(o + 2 * kMxXPart) = mx_u32x4{lo[2], lo[3], lo[4], lo[5]};
  sc[4 * (t & 63) + (t >> 6)] = (uint8_t)e;
  __syncthreads();
  if (t < 64)
    *reinterpret_cast<uint32_t*>(unit + kMxXScaleOff + 4 * t) = *reinterpret_cast<const uint32_t*>(sc + 4 * t);
}

// Rows (row i: row src[i], or i) -> digit planes, a workgroup a unit; columns past k (up to the chunk's end) are zero.
template <int T>
__device__ __forceinline__ void mx_quantize_x(const void* __restrict__ x, long long ldx, int m, int k, int kc, int wide,
                                              const int* __restrict__ src, uint8_t* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) float buf[kMxTile * kMxLdsRow];
  __shared__ __attribute__((aligned(16))) uint8_t sc[256];
  const int t = threadIdx.x;
  const long long u = blockIdx.x;
  const int r0 = (int)(u / kc) * kMxTile, c0 = (int)(u % kc) * kMxChunk;
  const int rows = min(m - r0, kMxTile);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (t >> 6), c = 4 * (t & 63);
    mx_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r < rows && c0 + c < k) v = mx_load4<T>(x, (src ? src[r0 + r] : r0 + r) * ldx + c0 + c, wide != 0);
    *reinterpret_cast<mx_f32x4*>(buf + r * kMxLdsRow + c) = v;
  }
  __syncthreads();
  float v[32];
  const int e = mx_x_byte(mx_unit_block(buf, t, v));
  mx_u32x6 hi, lo;
  mx_digits(v, e, hi, lo);
  mx_put_digits(out + u * kMxXUnit, sc, t, e, hi, lo);
}
}  // namespace qmm

#define QMM_MX_TYPED(NAME, T)                                                                                     \
  extern "C" __global__ void __launch_bounds__(256) qmm_mx_dequantize_##NAME(                                     \
      const uint8_t* __restrict__ w, int n, int k, void* __restrict__ dst, int kc) {                              \
    qmm::mx_dequantize<T>(w, n, k, dst, kc);                                                                      \
  }                                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) qmm_mx_quantize_x_##NAME(                                     \
      const void* __restrict__ x, long long ldx, int m, int k, int kc, int wide, const int* __restrict__ src,     \
      uint8_t* __restrict__ out) {                                                                                \
    qmm::mx_quantize_x<T>(x, ldx, m, k, kc, wide, src, out);                                                      \
  }
QMM_MX_TYPED(f32, qmm::kF32)
QMM_MX_TYPED(f16, qmm::kF16)
QMM_MX_TYPED(bf16, qmm::kBF16)

// f32 rows -> 49-byte blocks (qmm_quantize_rows), and those -> digit planes.
extern "C" __global__ void __launch_bounds__(256) qmm_mx_quantize_rows(const float* __restrict__ x, long long ldx,
                                                                       int m, int k, int wide,
                                                                       uint8_t* __restrict__ xq) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int nb = k / 32;
  if (i >= (long long)m * nb) return;
  float v[32];
  qmm::mx_u32x6 hi, lo;
  const int e = qmm::mx_x_byte(qmm::mx_load_block(x + i / nb * ldx + 32 * (i % nb), wide != 0, v));
  qmm::mx_digits(v, e, hi, lo);
  uint8_t* o = xq + i * qmm::kMxFp6x2Bytes;
  o[0] = (uint8_t)e;
#pragma unroll
  for (int j = 0; j < 24; ++j) {
    o[1 + j] = (uint8_t)(hi[j >> 2] >> (8 * (j & 3)));
    o[25 + j] = (uint8_t)(lo[j >> 2] >> (8 * (j & 3)));
  }
}

extern "C" __global__ void __launch_bounds__(256) qmm_mx_blocks_to_planes(const uint8_t* __restrict__ xq, int m, int k,
                                                                          int kc, uint8_t* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) uint8_t sc[256];
  const int t = threadIdx.x;
  const long long u = blockIdx.x;
  const int row = (int)(u / kc) * qmm::kMxTile + (t & 31);
  const int b = (int)(u % kc) * 8 + 2 * (t >> 6) + ((t >> 5) & 1);
  qmm::mx_u32x6 d[2] = {(qmm::mx_u32x6)(0u), (qmm::mx_u32x6)(0u)};
  int e = 4;
  if (row < m && 32 * b < k) {
    const uint8_t* p = xq + ((long long)row * (k / 32) + b) * qmm::kMxFp6x2Bytes;
    e = p[0] < 4 ? qmm::kMxNan : p[0];  // (no quantizer writes one: the second digit's scale would be below 2^-127)
#pragma unroll
    for (int j = 0; j < 48; ++j) d[j / 24][j % 24 >> 2] |= (uint32_t)p[1 + j] << (8 * (j & 3));
  }
  qmm::mx_put_digits(out + u * qmm::kMxXUnit, sc, t, e, d[0], d[1]);
}

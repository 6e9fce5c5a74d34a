// Microscaled values: blocks of 32 that share a power-of-two scale byte e
// (E8M0: 2^(e - 127); 255 marks a block that is not a number).
//
//   MXFP4    weights: E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign).
//   MXFP6x2  activations: two E2M3 digits a value, x = 2^(e - 127) (hi + lo / 16).
//            E2M3 is sign, two exponent bits, three mantissa bits: steps of 1/8 up
//            to 2, 1/4 up to 4, 1/2 up to 7.5. The second digit leaves an error of
//            at most 2^-7 at a block maximum of 3.875 .. 7.75, 2^-9 of the maximum
//            or less (normal values: 1.1e-3 of their norm; one E4M3 or E2M3 digit
//            leaves 2.6e-2).
//
// Why two six-bit digits. The scaled matrix instruction multiplies either format at
// the four-bit rate (32x32x64: 8.4 PFLOP/s measured, against 4.7 with an 8-bit
// operand and 2.3 nominal in bf16), applies the scales of both operands itself,
// and sums f6 x f4 products exactly (64-bit check, K up to 4096: no difference
// while the blocks' scales lie within a few binades, 1.5e-7 of the absolute sum
// with scales over 2^24). With an E4M3 operand its sum loses bits below 2^-13 of
// the largest product: 4.9e-6 relative on normal data. So one product is two
// instructions, at 4.2 PFLOP/s, with an error of the activation's rounding only.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qmm {

// Device layout of an MXFP4 weight [n, k]: units of 32 rows x 256 columns, row
// tiles outermost (n and k padded with zero codes to whole units). In a unit, step
// s (64 columns) holds 64 lanes x 16 bytes, lane 32 h + r the codes of row r, block
// 2 s + h, two values a byte in order: the matrix instruction's operand as it is
// loaded, 1 KB contiguous a step. Then 64 lanes x 4 scale bytes, byte s the scale of
// block 2 s + h: one register serves four steps (the instruction selects the byte).
constexpr int kMxTile = 32;
constexpr int kMxChunk = 256;
constexpr int kMxStepBytes = 1024;
constexpr int kMxScaleOff = 4096;
constexpr int kMxUnit = 4352;
// Digit planes of activation rows: units of 32 rows x 256 columns in the same order, so
// that every operand load is contiguous. Step s holds three parts of 64 lanes x 16
// bytes: lane 32 h + r has the 48 bytes of block 2 s + h of row r, 24 of hi and 24 of
// lo, in the parts' order; then 64 lanes x 4 scale bytes. Rows past the last are left
// as they are: a column of the product reads its own row only.
constexpr int kMxXPart = 1024, kMxXStep = 3 * kMxXPart;
constexpr int kMxXScaleOff = 4 * kMxXStep;
constexpr int kMxXUnit = kMxXScaleOff + 256;
constexpr int kMxFp4Bytes = 17;   // GGML block: e, codes 0..15 in low nibbles, 16..31 in high ones
constexpr int kMxFp6x2Bytes = 49; // block of qmm_quantize_rows: e, hi[24], lo[24]
constexpr int kMxNan = 255;

typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned mx_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned mx_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned mx_u32x6 __attribute__((ext_vector_type(6)));
typedef unsigned mx_u32x8 __attribute__((ext_vector_type(8)));
typedef unsigned mx_u32x12 __attribute__((ext_vector_type(12)));

// Element types of typed rows: the C ABI's tags.
constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;

__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  return f != f ? (uint16_t)(u >> 16 | 64) : (uint16_t)((u + 0x7fff + (u >> 16 & 1)) >> 16);
}
__device__ __forceinline__ float mx_load(const void* p, int type, long long i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return type == kF16 ? (float)__builtin_bit_cast(_Float16, v) : bf16_to_f32(v);
}
__device__ __forceinline__ uint16_t mx_to16(float v, int type) {
  return type == kF16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : f32_to_bf16(v);
}
__device__ __forceinline__ void mx_store(void* p, int type, long long i, float v) {
  if (type == kF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = mx_to16(v, type);
}

// The scale byte of a block with the largest magnitude amax (as bits, sign clear):
// the smallest power of two at which amax does not round past the largest code, at
// least `least`. MAN: the mantissa from which it would (E2M1: 1.75, 7 -> 8; E2M3:
// 1.9375, 7.75 -> 8). An infinity or NaN gives 255.
template <uint32_t MAN>
__device__ __forceinline__ int mx_scale_byte(uint32_t amax, int least) {
  if (amax >= 0x7f800000u) return kMxNan;
  const int e = (int)(amax >> 23) - 2 + ((amax & 0x7fffffu) >= MAN ? 1 : 0);
  return max(e, least);
}
constexpr uint32_t kMxMan4 = 0x600000;  // .75
constexpr uint32_t kMxMan6 = 0x780000;  // .9375

__device__ __forceinline__ int mx_w_byte(uint32_t amax) { return amax == 0 ? 0 : mx_scale_byte<kMxMan4>(amax, 0); }
// (the second digit's scale is four binades lower)
__device__ __forceinline__ int mx_x_byte(uint32_t amax) { return mx_scale_byte<kMxMan6>(amax, 4); }

// 32 values (even ones in `a`, odd ones in `b`) as one E2M3 digit each. The instruction
// writes its first registers before it has read its last, and the compiler gives the
// result registers of an operand that ends here: the operands are kept past it.
__device__ __forceinline__ mx_u32x6 mx_to_digit(const mx_f32x16& a, const mx_f32x16& b) {
  const auto d = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, 1.0f);
  asm volatile("" ::"v"(a), "v"(b), "v"(d));
  return __builtin_bit_cast(mx_u32x6, d);
}
// and back, in order
typedef float mx_f32x32 __attribute__((ext_vector_type(32)));
__device__ __forceinline__ mx_f32x32 mx_from_digit(const mx_u32x6& d) {
  const mx_f32x32 v = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(d, 1.0f);
  asm volatile("" ::"v"(d), "v"(v));
  return v;
}

// Both digits of 32 values under scale byte e as 24 + 24 bytes. A block with e = 255
// gets zero digits (0 * NaN is NaN in the product).
__device__ __forceinline__ void mx_digits(const float (&x)[32], int e, mx_u32x6& hi, mx_u32x6& lo) {
  mx_f32x16 a, b;
  const int up = 127 - e;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    a[j] = e == kMxNan ? 0.0f : __builtin_ldexpf(x[2 * j], up);
    b[j] = e == kMxNan ? 0.0f : __builtin_ldexpf(x[2 * j + 1], up);
  }
  hi = mx_to_digit(a, b);
  const mx_f32x32 back = mx_from_digit(hi);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    a[j] = (a[j] - back[2 * j]) * 16.0f;
    b[j] = (b[j] - back[2 * j + 1]) * 16.0f;
  }
  lo = mx_to_digit(a, b);
}

// A lane's 48 bytes of a step. As one vector of 12 its two digits are the instruction's
// operands where the three loads put them, without a move.
__device__ __forceinline__ mx_u32x12 mx_x(const mx_u32x4& p0, const mx_u32x4& p1, const mx_u32x4& p2) {
  const mx_u32x8 a = __builtin_shufflevector(p0, p1, 0, 1, 2, 3, 4, 5, 6, 7);
  const mx_u32x8 b = __builtin_shufflevector(p2, p2, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11);
}
__device__ __forceinline__ mx_u32x6 mx_hi(const mx_u32x12& x) { return __builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5); }
__device__ __forceinline__ mx_u32x6 mx_lo(const mx_u32x12& x) { return __builtin_shufflevector(x, x, 6, 7, 8, 9, 10, 11); }

// Block (step s, lane place l) of a unit of digit planes.
__device__ __forceinline__ void mx_put_block(uint8_t* unit, int s, int l, int e, const mx_u32x6& hi, const mx_u32x6& lo) {
  uint8_t* o = unit + s * kMxXStep + 16 * l;
  *reinterpret_cast<mx_u32x4*>(o) = mx_u32x4{hi[0], hi[1], hi[2], hi[3]};
  *reinterpret_cast<mx_u32x4*>(o + kMxXPart) = mx_u32x4{hi[4], hi[5], lo[0], lo[1]};
  *reinterpret_cast<mx_u32x4*>(o + 2 * kMxXPart) = mx_u32x4{lo[2], lo[3], lo[4], lo[5]};
  unit[kMxXScaleOff + 4 * l + s] = (uint8_t)e;
}

// One step (64 columns) of a 32 x 32 tile by one digit: weights (A, rows of the result)
// times activations (B, columns). S: the byte of the scale registers.
template <int S>
__device__ __forceinline__ mx_f32x16 mx_mfma(const mx_u32x4& w, const mx_u32x6& x, mx_f32x16 c, int sw, int sx) {
  const mx_u32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const mx_u32x8 b = __builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_bit_cast(mx_i32x8, a), __builtin_bit_cast(mx_i32x8, b),
                                                         c, 4, 2, S, sw, S, sx);
}
// One step of 128 columns of a 16 x 16 tile: lane 16 g + r holds block g of row r, the
// result's column is lane & 15, its rows 4 (lane / 16) + register. The result must not
// share registers with an operand (the compiler allows it for this size; the sums were
// wrong): the operands are kept past it.
template <int S>
__device__ __forceinline__ mx_f32x4 mx_mfma16(const mx_u32x4& w, const mx_u32x6& x, mx_f32x4 c, int sw, int sx) {
  const mx_u32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const mx_u32x8 b = __builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, -1, -1);
  const mx_f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      __builtin_bit_cast(mx_i32x8, a), __builtin_bit_cast(mx_i32x8, b), c, 4, 2, S, sw, S, sx);
  asm volatile("" ::"v"(w), "v"(x), "v"(sw), "v"(sx), "v"(d));
  return d;
}
// (the second digit's scale is the first's less 4 in every byte)
constexpr int kMxLoScale = 0x04040404;
// (result: lane's column = lane & 31, register r its row 8 (r / 4) + 4 (lane / 32) + r % 4)

}  // namespace qmm

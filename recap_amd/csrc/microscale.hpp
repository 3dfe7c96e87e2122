// Microscaled rows: blocks of 32 values along a row that share a power of two, for the kernels that
// write or read them (microscale.hip, mx_linear.hip, capture.hip, attention.hip).
//
// A block whose largest magnitude is a has the scale byte s = e + 127 and the values code * 2^e:
//   fp4   e the smallest with a < 7 * 2^e: the largest value then rounds to at most 6, the largest
//         code, and every value is within half a step of its own.  Codes are sign, two exponent and
//         one mantissa bits (0, 0.5, 1, 1.5, 2, 3, 4, 6); two to a byte, the first in the low half.
//   int8  e the smallest with 64 a < 127.5 * 2^e; integers up to 127, each worth 2^(e - 6).  e stops at
//         127: from 127.5 * 2^121 on (1.992 * 2^127, of fp32 alone) values are cut off at 127 * 2^121.
// Both round to nearest, ties to the even code.  s = 255 marks a block that held an infinity or NaN:
// all of it reads as NaN.  Scales and products with them are exact, so the same values give the same
// codes on every path.
#pragma once

#include "rows.hpp"

namespace recap {

enum MxFormat { kMxFp4 = 1, kMxInt8 = 2 };

constexpr int kMxBlock = 32;
// Rows are filled up to this many values: whole blocks, and for the product (which reads fp4 rows
// only) whole steps of its reduction, so that it has no partial one.
__host__ __device__ constexpr int mx_fill(int format) { return format == kMxFp4 ? 256 : kMxBlock; }
__host__ __device__ constexpr int64_t mx_filled(int format, int64_t width) {
  return (width + mx_fill(format) - 1) / mx_fill(format) * mx_fill(format);
}
__host__ __device__ constexpr int64_t mx_row_bytes(int format, int64_t width) {
  return format == kMxFp4 ? mx_filled(format, width) / 2 : mx_filled(format, width);
}
__host__ __device__ constexpr int64_t mx_row_scales(int format, int64_t width) {
  return mx_filled(format, width) / kMxBlock;
}

constexpr unsigned kNotFinite = 0x7f800000u;  // magnitude bits of an infinity; of NaN: more

// Scale byte of a block from the bits of its largest magnitude.  A quarter (1 / 128 for int8) of the
// leading one added to the mantissa carries into the exponent from 1.75 (255 / 128) on.
template <int FORMAT>
__device__ inline unsigned mx_scale(unsigned bits) {
  unsigned s;
  if constexpr (FORMAT == kMxFp4) {
    s = (bits + 0x200000u) >> 23;
    s = s > 2 ? s - 2 : 0;
  } else {
    // A subnormal has no leading one of its own: its binade is half as long.  254 is the last power of
    // two; mx_int8_codes cuts off what rounds past 127 of it.
    s = min((bits + (bits < 0x800000u ? 0x8000u : 0x10000u)) >> 23, 254u);
  }
  return bits >= kNotFinite ? 255 : s;
}

// Largest magnitude's bits over the four lanes that share a block (8 values each).
__device__ inline unsigned quad_max(unsigned m) {
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, false));  // lane ^ 1
  return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
}

template <int N>
__device__ inline unsigned magnitude_bits(const float (&v)[N]) {
  unsigned m = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  return m;
}

// Eight fp4 codes of scale s.  The conversion takes the exponent of its scale operand.
__device__ inline unsigned mx_fp4_codes(const float (&v)[8], unsigned s) {
  const float unit = __uint_as_float(s << 23);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], unit, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], unit, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], unit, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], unit, 3);
  return s == 255 ? 0 : w;
}

// Eight int8 codes of scale s, in memory order.
__device__ inline u32x2 mx_int8_codes(const float (&v)[8], unsigned s) {
  const int up = 133 - (int)s;
  u32x2 w = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = fmaxf(fminf(rintf(ldexpf(v[e], up)), 127.0f), -127.0f);
    w[e >> 2] |= ((unsigned)(int)c & 0xff) << (8 * (e & 3));
  }
  return s == 255 ? u32x2{0, 0} : w;
}

__device__ inline float mx_nan() { return __uint_as_float(0x7fc00000u); }

__device__ inline void mx_fp4_values(unsigned w, unsigned s, float (&v)[8]) {
  const float unit = __uint_as_float(s << 23);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 3);
  const float x[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = s == 255 ? mx_nan() : x[e];
}

// Code e (0 .. 7, memory order) of eight, and what a code of a block with scale s is worth.
__device__ inline float mx_int8_code(u32x2 w, int e) {
  return (float)((int)(w[e >> 2] << (24 - 8 * (e & 3))) >> 24);
}
__device__ inline float mx_int8_unit(unsigned s) {
  return s == 255 ? mx_nan() : ldexpf(1.0f, (int)s - 133);
}

__device__ inline void mx_int8_values(u32x2 w, unsigned s, float (&v)[8]) {
  const float unit = mx_int8_unit(s);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = mx_int8_code(w, e) * unit;
}

}  // namespace recap

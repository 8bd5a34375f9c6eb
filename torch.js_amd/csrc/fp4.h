// Four-bit values: a sign and the number of a step of 0, 0.5, 1, 1.5, 2, 3, 4,
// 6 (one sign bit, two of an exponent, one of a fraction), times a float scale
// that several share.  The codes are those that gfx950 converts itself, two in
// one instruction, exactly, to floats or to bfloat16.  Device only.
#pragma once

#include "common.h"
#include "wave.h"

namespace tjh {
namespace fp4 {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float floatx2u __attribute__((ext_vector_type(2), aligned(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The eight values of a word, the lowest 4 bits first.
__device__ __forceinline__ void unpack(uint32_t w, float (&v)[8]) {
  const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0);
  const floatx2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
  const floatx2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2);
  const floatx2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// The same as a matrix operand.
__device__ __forceinline__ bf16x8 steps(uint32_t w) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// A float as three bfloat16 parts, eight bits of its significand each: every
// part is cut off, so that what is left is exact.  A part is the high half of a
// word; two are packed into one.
__device__ __forceinline__ float cut(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_high(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
}
// What is left of x; an infinity is its first part alone.
__device__ __forceinline__ float rest(float x) {
  const float h = cut(x);
  return x == h ? 0.f : x - h;
}
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&part)[3]) {
  uintx4 p[3];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float a = rest(x[2 * q]), b = rest(x[2 * q + 1]);
    p[0][q] = pack_high(x[2 * q], x[2 * q + 1]);
    p[1][q] = pack_high(a, b);
    p[2][q] = pack_high(a - cut(a), b - cut(b));
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) part[i] = __builtin_bit_cast(bf16x8, p[i]);
}
// The same of numbers that are no infinities.
__device__ __forceinline__ void split8_finite(const float (&x)[8], bf16x8 (&part)[3]) {
  uintx4 p[3];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float a = x[2 * q] - cut(x[2 * q]), b = x[2 * q + 1] - cut(x[2 * q + 1]);
    p[0][q] = pack_high(x[2 * q], x[2 * q + 1]);
    p[1][q] = pack_high(a, b);
    p[2][q] = pack_high(a - cut(a), b - cut(b));
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) part[i] = __builtin_bit_cast(bf16x8, p[i]);
}

// |x| as an integer in the order of magnitudes, NaN above infinity.
__device__ __forceinline__ uint32_t magnitude(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

// The scale of values whose largest magnitude is `top`: top / 6, 0 where they
// are held as zeros (under 2^-100, so that borders below stay normal floats),
// NaN where one of them is no number.
__device__ __forceinline__ float scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return top < 0x0d800000u ? 0.f : __uint_as_float(top) / 6.f;
}

// The code of x at a scale, by bisection.  A step is passed where |x| is above the
// border halfway to it, or on one whose upper step is even; the sign of |x| -
// border * scale is exact, as it is rounded once.
__device__ __forceinline__ uint32_t code_of(float x, float scale) {
  const float a = fabsf(x);
  const bool b4 = __builtin_fmaf(-1.75f, scale, a) >= 0.f;
  const bool b2 = __builtin_fmaf(b4 ? -3.5f : -0.75f, scale, a) >= 0.f;
  const float hi = b4 ? -5.f : -1.25f, lo = b4 ? -2.5f : -0.25f;
  const bool b1 = __builtin_fmaf(b2 ? hi : lo, scale, a) > 0.f;
  const uint32_t c = (b4 ? 4u : 0u) | (b2 ? 2u : 0u) | (b1 ? 1u : 0u);
  return (scale > 0.f ? c : 0u) | (x < 0.f ? 8u : 0u);
}

// Bytes of a cached position's codes.
__host__ __device__ inline int row_bytes(int D) { return (D + 31) / 32 * 16; }

}  // namespace fp4
}  // namespace tjh

// 8-bit rows: a row y stands as q = round(127 y / max|y|) (ties to even) and the scale max|y| / 127.
#pragma once
#include "common.h"

namespace k8s {
namespace q8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Below this a row's largest value is stored as zero.  Behind a norm that goes by y, and the h w that the integers are made of go
// down to kLeast, whose reciprocal times 127 is near fp32's end (with eps of 2^-40 and more y is below kTiny before that).
constexpr float kTiny = 0x1p-100f, kLeast = 0x1p-120f;

// max|y| as bits: a NaN is larger than the infinity, so that neither is lost on the way
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Step {
  float inv, rest;  // integers a unit of y, and what rounding it left
  float scale;      // what an integer stands for; NaN where the row holds a NaN or an infinity (its integers are zeros)
};
__device__ __forceinline__ Step row_step(uint32_t top, float least = kTiny) {
  const float t = __uint_as_float(top);
  if (top >= 0x7f800000u) return {0.f, 0.f, __uint_as_float(0x7fc00000u)};
  if (t < least) return {0.f, 0.f, 0.f};
  const float inv = 127.f / t;
  return {inv, fmaf(-inv, t, 127.f) / t, t / 127.f};
}

// 127 y / max to the nearest integer, ties to even, in the low byte: 1.5 2^23 puts the integer into the last bits of the sum.  The
// quotient is rounded to fp32 first, from 48 bits: a tie (short numbers make many) is met as one, where y times the rounded
// 127 / max alone would lie beside it for a whole row.
__device__ __forceinline__ uint32_t to_int8(float y, const Step& s) {
  float p = fmaf(y, s.inv, y * s.rest);
  asm("" : "+v"(p));  // (no fma with what follows)
  return __float_as_uint(p + 12582912.f);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return lo | hi;
}
__device__ __forceinline__ u32x2 pack8(const float (&y)[8], const Step& s) {
  uint32_t u[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] = to_int8(y[j], s);
  u32x2 r = {pack4(u[0], u[1], u[2], u[3]), pack4(u[4], u[5], u[6], u[7])};
  // (0 times an infinity or a NaN is a NaN, whose bits are no integer)
  if (s.inv == 0.f) r = u32x2{0, 0};
  return r;
}

// four int8 as two pairs of bf16: every int8 is one exactly
__device__ __forceinline__ u32x2 to_bf16x4(uint32_t v) {
  const float f0 = (float)(int8_t)v, f1 = (float)(int8_t)(v >> 8), f2 = (float)(int8_t)(v >> 16), f3 = (float)(int8_t)(v >> 24);
  return u32x2{__builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u),
               __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u)};
}
// eight int8 as a matrix operand
__device__ __forceinline__ bf16x8 to_bf16x8(uint32_t a, uint32_t b) {
  const u32x2 x = to_bf16x4(a), y = to_bf16x4(b);
  return __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
}

}  // namespace q8
}  // namespace k8s

// Rows in 8 bits with one fp32 scale each: the rules and device helpers that the kernels quantizing rows share
// (csrc/fp8.hip, csrc/int8.hip, csrc/norm.hip).
//
// e4m3: scale = absmax / 448 (the largest e4m3 value), element = x * (448 / absmax) in fp32, rounded to nearest even.  A row
// whose absmax is below 2^-118 -- all-zero rows, and rows so small that 448 / absmax would overflow fp32 (it does below
// 448 / FLT_MAX ~ 1.3e-36), turning 0 * inv into NaN -- is treated as a zero row: scale 1, inv 1 (its elements, all below
// 2^-118, round to +-0).  A row of
// the norm (csrc/norm.hip) that holds an infinity or a NaN has the scale NaN and elements 0, as in int8: an infinity in h makes
// 1 / rms and every other element zero, and a maximum that passed the NaN over would let the row read back as zeros.
// (csrc/fp8.hip quantizes rows as they are given: a NaN stays in its element, an infinity gives the scale infinity, and 0 times
// that reads back as NaN.)
//
// int8: scale = a / 127 with a = max(absmax, 2^-100), element = the whole number nearest to 127 x / a, ties to even.  The
// quotient is taken exactly: x = a / 2 lies on the border between 63 and 64 (common in bf16), and products by a rounded
// 127 / a fall on either side of it.  One fma adds the product to 1.5 * 2^23, which rounds it to a whole number in the low
// mantissa bits, a second one gives what was rounded away; where that is within 1e-4 of half a step (fp32 is off by less than
// 2e-5 steps), the element is compared with the border in 64 bits, where both sides are exact (24-bit values times at most
// 255).  A row that holds an infinity or a NaN has the scale NaN and elements 0.
#pragma once

#include "common.h"

namespace moe {

constexpr float kE4M3Max = 448.f;
constexpr float kQuantTiny = 0x1p-118f;  // smallest absmax quantized with its own e4m3 scale: 448 / 2^-118 < FLT_MAX
constexpr float kInt8Max = 127.f;
constexpr float kInt8Tiny = 0x1p-100f;   // smallest a of an int8 row: 127 / a stays far inside fp32

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void e4m3_row_scale(float amax, float& sc, float& inv) {
  const bool live = amax >= kQuantTiny;
  sc = live ? amax / kE4M3Max : 1.f;
  inv = live ? kE4M3Max / amax : 1.f;
}

struct E4M3Row {
  float scale, inv;
  uint32_t keep;  // all ones, or 0 for a row that holds an infinity or a NaN
};
__device__ __forceinline__ E4M3Row e4m3_row(uint32_t amax_bits) {
  E4M3Row r;
  const bool ok = amax_bits < 0x7f800000u;
  e4m3_row_scale(__uint_as_float(ok ? amax_bits : 0u), r.scale, r.inv);
  r.scale = ok ? r.scale : __uint_as_float(0x7fc00000u);
  r.keep = ok ? ~0u : 0u;
  return r;
}

__device__ __forceinline__ u32x2 e4m3_pack8(const float (&v)[8], const E4M3Row& r) {
  uint32_t lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * r.inv, v[1] * r.inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * r.inv, v[3] * r.inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * r.inv, v[5] * r.inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * r.inv, v[7] * r.inv, hi, true);
  return u32x2{lo & r.keep, hi & r.keep};
}

// Magnitude bits: their unsigned order is the order of the magnitudes, infinities and NaNs on top (fmaxf drops a NaN).
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Int8Row {
  float a, scale, inv;
  uint32_t keep;  // all ones, or 0 for a row that holds an infinity or a NaN
};
__device__ __forceinline__ Int8Row int8_row(uint32_t amax_bits) {
  Int8Row r;
  const bool ok = amax_bits < 0x7f800000u;
  r.a = fmaxf(__uint_as_float(ok ? amax_bits : 0u), kInt8Tiny);
  r.scale = ok ? r.a / kInt8Max : __uint_as_float(0x7fc00000u);
  r.inv = kInt8Max / r.a;
  r.keep = ok ? ~0u : 0u;
  return r;
}

constexpr float kInt8Magic = 12582912.f;  // 1.5 * 2^23: adding it leaves a whole number in the low mantissa bits

// The element next to a border: q steps, d = (127 x / a) - q to about 2e-5, |d| near 1/2.
__device__ __forceinline__ float int8_border(float v, float a, float q, float d) {
  const float up = d > 0.f ? q + 1.f : q - 1.f;
  const double side = 254.0 * (double)v - (double)(q + up) * (double)a;  // 2 (127 v - border a), exact
  const bool even_up = ((int)up & 1) == 0;
  const bool take = d > 0.f ? (side > 0.0 || (side == 0.0 && even_up)) : (side < 0.0 || (side == 0.0 && even_up));
  return take ? up : q;
}

// The low bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

__device__ __forceinline__ u32x2 int8_pack8(const float (&v)[8], const Int8Row& r) {
  float q[8], d[8], worst = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = fmaf(v[i], r.inv, kInt8Magic);
    d[i] = fmaf(v[i], r.inv, kInt8Magic - q[i]);
    worst = fmaxf(worst, fabsf(d[i]));
  }
  if (worst > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(d[i]) > 0.4999f) q[i] = int8_border(v[i], r.a, q[i] - kInt8Magic, d[i]) + kInt8Magic;
  }
  return u32x2{low_bytes(__float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3])) & r.keep,
               low_bytes(__float_as_uint(q[4]), __float_as_uint(q[5]), __float_as_uint(q[6]), __float_as_uint(q[7])) & r.keep};
}

}  // namespace moe

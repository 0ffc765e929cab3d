// MXFP4 matrices of the expert FFN: 4-bit (e2m1) elements, every 32 consecutive elements of a row with one shared
// power-of-two scale (OCP MX, E8M0).
//
// The values of e2m1 are 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives.  A block's scale is 2^e with e the smallest
// integer with absmax <= 6 * 2^e, so no element saturates, in [-124, 125]; its byte is e + 127.  With absmax = 1.m 2^p
// (6 = 1.5 * 2^2) that is e = p - 2 when 1.m <= 1.5 and p - 1 otherwise: an addition on the bits.  At the range's ends,
// what the largest values lose to saturation and the smallest to rounding keeps every value of a block a finite normal
// bf16 number (6 * 2^125 < 2^128, 2^-125 >= 2^-126), so a dequantized element is exact in bf16 and in fp32.  A block that
// holds an infinity or a NaN gets the byte 255 and stands for NaNs.
//
// k_quant_mxfp4    one read of the source: a lane holds 8 elements, the four lanes of a block share their absmax by two DPP
//                  moves, and v_cvt_scalef32_pk_fp4_f32 divides, rounds to nearest even and saturates two elements a time.
// k_dequant_mxfp4  the same shape backwards with v_cvt_scalef32_pk_bf16_fp4 / _f32_fp4.
// Both are bound by their bytes, 2.53 (bf16) or 4.53 (fp32) an element; a wave moves 2048 elements a step, four 16-byte (or
// eight, fp32) loads a lane in flight, and its four bytes a lane of 4-bit values and 64 bytes of scales are whole requests.
// bf16 [114688, 4096]: 194 us there (1.19 GB, 6.1 TB/s) and 170 back (7.0 TB/s); fp32 [768, 2048]: 2.9 and 3.4 us, a launch.
#include <algorithm>

#include "common.h"

namespace moe {
namespace {

constexpr int kQStep = 2048;  // elements of a wave's step: four pieces of 512, 8 a lane

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
  const u32x4 a = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    v[2 * m] = __uint_as_float(a[m] << 16);
    v[2 * m + 1] = __uint_as_float(a[m] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
  const f32x4 b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4));
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    v[m] = a[m];
    v[4 + m] = b[m];
  }
}

// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t mx4_byte(uint32_t amax) {
  // exponent field - 2, one more when the mantissa is above 1.5
  const int b = (int)((amax + 0x3fffffu) >> 23) - 2;
  return amax >= 0x7f800000u ? 255u : (uint32_t)min(max(b, 3), 252);
}

template <typename T>
__global__ __launch_bounds__(256) void k_quant_mxfp4(const T* __restrict__ src, int64_t n, uint32_t* __restrict__ q,
                                                    uint8_t* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t step = (int64_t)gridDim.x * 4 * kQStep;
  for (int64_t i0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kQStep; i0 < n; i0 += step) {
    float v[4][8];
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j * 512 + lane * 8;
      in[j] = i < n;  // n is a multiple of 32: the four lanes of a block agree
      load8(src + (in[j] ? i : 0), v[j]);
    }
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, abs_bits(v[j][k]));
      m = max(m, (uint32_t)row16_partner<0>((int)m));
      m = max(m, (uint32_t)row16_partner<1>((int)m));
      const uint32_t b = mx4_byte(m);
      mine = (lane & 3) == j ? b : mine;
      const float sc = __uint_as_float((b == 255u ? 127u : b) << 23);
      uint32_t w = 0;
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][0], v[j][1], sc, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][2], v[j][3], sc, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][4], v[j][5], sc, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][6], v[j][7], sc, 3);
      if (in[j]) q[(i0 + j * 512) / 8 + lane] = w;
    }
    // lane 4 b + j holds the byte of piece j's block b
    const int64_t blk = i0 / 32 + (lane & 3) * 16 + (lane >> 2);
    if (blk < n / 32) scale[blk] = (uint8_t)mine;
  }
}

__device__ __forceinline__ void store8(uint16_t* p, uint32_t w, float sc) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
  __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(p));
}
__device__ __forceinline__ void store8(float* p, uint32_t w, float sc) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
  __builtin_nontemporal_store(f32x4{a[0], a[1], b[0], b[1]}, reinterpret_cast<f32x4*>(p));
  __builtin_nontemporal_store(f32x4{c[0], c[1], d[0], d[1]}, reinterpret_cast<f32x4*>(p + 4));
}

template <typename T>
__global__ __launch_bounds__(256) void k_dequant_mxfp4(const uint32_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                      int64_t n, T* __restrict__ dst) {
  const int lane = threadIdx.x & 63;
  const int64_t step = (int64_t)gridDim.x * 4 * kQStep;
  for (int64_t i0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kQStep; i0 < n; i0 += step) {
    uint32_t w[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j * 512 + lane * 8;
      w[j] = q[i < n ? i / 8 : 0];
      b[j] = scale[i < n ? i / 32 : 0];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j * 512 + lane * 8;
      // the instruction takes the scale's exponent field: byte 0, as a float 0.0, is 2^-127, and 255 gives NaNs
      if (i < n) store8(dst + i, w[j], __uint_as_float(b[j] << 23));
    }
  }
}

bool al16m(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
unsigned mx_blocks(int64_t n) { return (unsigned)std::min<int64_t>(2048, (n + 4 * kQStep - 1) / (4 * kQStep)); }

}  // namespace

}  // namespace moe

using namespace moe;

static int mx_check(const char* what, int64_t rows, int64_t cols, int dtype) {
  if (rows < 0 || cols < 32 || cols % 32 || cols > INT32_MAX / 2 || rows > ((int64_t)1 << 46) / cols ||
      (dtype != MOE_BF16 && dtype != MOE_F32))
    return fail_arg("%s: bad arguments rows=%lld cols=%lld dtype=%d (need cols %% 32 == 0, bf16 or fp32)", what,
                    (long long)rows, (long long)cols, dtype);
  return 0;
}

extern "C" int moe_quant_mxfp4(const void* src, int src_dtype, int64_t rows, int64_t cols, void* q, void* scale,
                               void* stream) {
  if (int rc = mx_check("moe_quant_mxfp4", rows, cols, src_dtype)) return rc;
  if (rows == 0) return 0;
  if (!src || !q || !scale || !al16m(src) || !al16m(q)) return fail_arg("moe_quant_mxfp4: null or misaligned pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t n = rows * cols;
  if (src_dtype == MOE_BF16)
    MOE_LAUNCH("k_quant_mxfp4", k_quant_mxfp4<uint16_t>, dim3(mx_blocks(n)), dim3(256), 0, s,
               static_cast<const uint16_t*>(src), n, static_cast<uint32_t*>(q), static_cast<uint8_t*>(scale));
  else
    MOE_LAUNCH("k_quant_mxfp4", k_quant_mxfp4<float>, dim3(mx_blocks(n)), dim3(256), 0, s, static_cast<const float*>(src),
               n, static_cast<uint32_t*>(q), static_cast<uint8_t*>(scale));
  return check_launch("moe_quant_mxfp4");
}

extern "C" int moe_dequant_mxfp4(const void* q, const void* scale, int64_t rows, int64_t cols, void* dst, int dst_dtype,
                                 void* stream) {
  if (int rc = mx_check("moe_dequant_mxfp4", rows, cols, dst_dtype)) return rc;
  if (rows == 0) return 0;
  if (!q || !scale || !dst || !al16m(q) || !al16m(dst)) return fail_arg("moe_dequant_mxfp4: null or misaligned pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t n = rows * cols;
  if (dst_dtype == MOE_BF16)
    MOE_LAUNCH("k_dequant_mxfp4", k_dequant_mxfp4<uint16_t>, dim3(mx_blocks(n)), dim3(256), 0, s,
               static_cast<const uint32_t*>(q), static_cast<const uint8_t*>(scale), n, static_cast<uint16_t*>(dst));
  else
    MOE_LAUNCH("k_dequant_mxfp4", k_dequant_mxfp4<float>, dim3(mx_blocks(n)), dim3(256), 0, s,
               static_cast<const uint32_t*>(q), static_cast<const uint8_t*>(scale), n, static_cast<float*>(dst));
  return check_launch("moe_dequant_mxfp4");
}

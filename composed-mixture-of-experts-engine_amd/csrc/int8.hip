// Rows in int8 with one fp32 scale each, and 8-bit rows (int8 or e4m3) back to values.
//
//   a = max(absmax of the row, 2^-100), scale = a / 127, q = the whole number nearest to 127 x / a (ties to even; quant8.h)
//
// k_quant_rows_int8   one pass over memory: LPR lanes (a wave, or a block of four) hold a row of up to LPR * 64 elements in
//                     registers between its absmax and its quantization.  Longer rows are read twice.
// k_dequant_rows      value = q * scale in fp32, rounded to bf16 or kept.
//
// Both are bound by memory: 6 vector instructions an element against 3 bytes of traffic (bf16).
#include <algorithm>

#include "common.h"
#include "quant8.h"

namespace moe {
namespace {

constexpr int kQ8Threads = 256;

template <typename T>
__device__ __forceinline__ void row_load8(const T* p, u32x4 (&w)[sizeof(T) / 2]) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
}
__device__ __forceinline__ void row_get8(const u32x4 (&w)[1], float (&v)[8]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    v[2 * m] = __uint_as_float(w[0][m] << 16);
    v[2 * m + 1] = __uint_as_float(w[0][m] & 0xffff0000u);
  }
}
__device__ __forceinline__ void row_get8(const u32x4 (&w)[2], float (&v)[8]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    v[m] = __uint_as_float(w[0][m]);
    v[4 + m] = __uint_as_float(w[1][m]);
  }
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = row16_max_u32(v);
  v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return max(v, (uint32_t)__shfl_xor((int)v, 32));
}

// The absmax bits of a row over its LPR lanes: a wave, or the block's four waves through LDS.
template <int LPR>
__device__ __forceinline__ uint32_t row_absmax(uint32_t m, uint32_t* red) {
  m = wave_max_u32(m);
  if constexpr (LPR == kQ8Threads) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    __syncthreads();  // before the next row's
  }
  return m;
}

// NCH: 8-element pieces of a row that a lane holds; 0: any number, read twice.  Rows past *row_limit (if given) are left as
// they are.
template <typename T, int LPR, int NCH>
__global__ __launch_bounds__(kQ8Threads) void k_quant_rows_int8(const T* __restrict__ src, int64_t rows, int cols, int64_t ld,
                                                               uint8_t* __restrict__ dst, float* __restrict__ scale,
                                                               const int* __restrict__ row_limit) {
  __shared__ uint32_t red[4];
  const int l = threadIdx.x & (LPR - 1);
  const int64_t step = (int64_t)gridDim.x * (kQ8Threads / LPR);
  if (row_limit != nullptr) rows = min(rows, (int64_t)max(*row_limit, 0));
  for (int64_t r = (int64_t)blockIdx.x * (kQ8Threads / LPR) + threadIdx.x / LPR; r < rows; r += step) {
    const T* const s = src + r * ld;
    uint8_t* const d = dst + r * cols;
    uint32_t m = 0;
    float v[8];
    if constexpr (NCH > 0) {
      u32x4 w[NCH][sizeof(T) / 2];
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c = (l + LPR * j) * 8;
        if (c < cols) {
          row_load8(s + c, w[j]);
        } else {
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[j][i] = u32x4{0u, 0u, 0u, 0u};
        }
      }
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        row_get8(w[j], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
      }
      // the packed words are pinned: otherwise the unpacked floats of the first pass are kept for the second
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) __asm__ volatile("" : "+v"(w[j][i]));
      const Int8Row q = int8_row(row_absmax<LPR>(m, red));
      if (l == 0) scale[r] = q.scale;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c = (l + LPR * j) * 8;
        row_get8(w[j], v);
        const u32x2 o = int8_pack8(v, q);
        if (c < cols) *reinterpret_cast<u32x2*>(d + c) = o;
      }
    } else {
      u32x4 w[sizeof(T) / 2];
      for (int c = l * 8; c < cols; c += LPR * 8) {
        row_load8(s + c, w);
        row_get8(w, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
      }
      const Int8Row q = int8_row(row_absmax<LPR>(m, red));
      if (l == 0) scale[r] = q.scale;
      for (int c = l * 8; c < cols; c += LPR * 8) {
        row_load8(s + c, w);
        row_get8(w, v);
        *reinterpret_cast<u32x2*>(d + c) = int8_pack8(v, q);
      }
    }
  }
}

// Sixteen elements a lane, LPR lanes a row.
template <bool E4M3, typename T, int LPR>
__global__ __launch_bounds__(kQ8Threads) void k_dequant_rows(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                            int64_t rows, int cols, T* __restrict__ dst) {
  const int l = threadIdx.x & (LPR - 1);
  const int64_t step = (int64_t)gridDim.x * (kQ8Threads / LPR);
  for (int64_t r = (int64_t)blockIdx.x * (kQ8Threads / LPR) + threadIdx.x / LPR; r < rows; r += step) {
    const float sc = scale[r];
    const uint8_t* const s = q + r * cols;
    T* const d = dst + r * cols;
    for (int c = l * 16; c < cols; c += LPR * 16) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(s + c);
      float v[16];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if constexpr (E4M3) {
          v[4 * m] = __builtin_amdgcn_cvt_f32_fp8((int)w[m], 0) * sc;
          v[4 * m + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[m], 1) * sc;
          v[4 * m + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[m], 2) * sc;
          v[4 * m + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[m], 3) * sc;
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b) v[4 * m + b] = (float)(int8_t)(w[m] >> (8 * b)) * sc;
        }
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 o;
#pragma unroll
          for (int m = 0; m < 4; ++m) o[m] = pack2bf(v[8 * h + 2 * m], v[8 * h + 2 * m + 1]);
          __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(d + c) + h);
        }
      } else {
#pragma unroll
        for (int m = 0; m < 4; ++m)
          __builtin_nontemporal_store(f32x4{v[4 * m], v[4 * m + 1], v[4 * m + 2], v[4 * m + 3]},
                                      reinterpret_cast<f32x4*>(d + c) + m);
      }
    }
  }
}

bool al16_8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// enough blocks to fill the card several times over; the rest are strides
unsigned q8_blocks(int64_t rows, int lpr) {
  const int64_t per = kQ8Threads / lpr;
  return (unsigned)std::min<int64_t>(8192, std::max<int64_t>(1, (rows + per - 1) / per));
}

template <typename T, int LPR>
void launch_quant(const T* src, int64_t rows, int cols, int64_t ld, uint8_t* dst, float* scale, const int* lim, hipStream_t s) {
  const dim3 grid(q8_blocks(rows, LPR)), block(kQ8Threads);
  const int n = (cols + LPR * 8 - 1) / (LPR * 8);
#define MOE_Q8(NCH) MOE_LAUNCH("k_quant_rows_int8", (k_quant_rows_int8<T, LPR, NCH>), grid, block, 0, s, src, rows, cols, ld, dst, scale, lim)
  if (n <= 1) MOE_Q8(1);
  else if (n <= 2) MOE_Q8(2);
  else if (n <= 4) MOE_Q8(4);
  else if (n <= 8) MOE_Q8(8);
  else MOE_Q8(0);
#undef MOE_Q8
}
}  // namespace

int quant_rows_int8(const void* src, int src_dtype, int64_t rows, int64_t cols, int64_t ld, void* dst, float* scale,
                    const int* row_limit, hipStream_t s) {
  if (rows < 0 || cols < 16 || cols % 16 || ld < cols || ld % 8 || cols > INT32_MAX / 2 ||
      (src_dtype != MOE_BF16 && src_dtype != MOE_F32))
    return fail_arg("moe_quant_rows_int8: bad arguments rows=%lld cols=%lld ld=%lld (need cols %% 16 == 0, ld >= cols, "
                    "ld %% 8 == 0, bf16 or fp32)", (long long)rows, (long long)cols, (long long)ld);
  if (rows == 0) return 0;
  if (!src || !dst || !scale || !al16_8(src) || !al16_8(dst))
    return fail_arg("moe_quant_rows_int8: null or misaligned pointer");
  // a wave a row up to 1024 elements; a block a row past that
  const auto* bp = static_cast<const uint16_t*>(src);
  const auto* fp = static_cast<const float*>(src);
  auto* dp = static_cast<uint8_t*>(dst);
  if (src_dtype == MOE_BF16) {
    if (cols <= 1024) launch_quant<uint16_t, 64>(bp, rows, (int)cols, ld, dp, scale, row_limit, s);
    else launch_quant<uint16_t, 256>(bp, rows, (int)cols, ld, dp, scale, row_limit, s);
  } else {
    if (cols <= 1024) launch_quant<float, 64>(fp, rows, (int)cols, ld, dp, scale, row_limit, s);
    else launch_quant<float, 256>(fp, rows, (int)cols, ld, dp, scale, row_limit, s);
  }
  return check_launch("moe_quant_rows_int8");
}
}  // namespace moe

using namespace moe;

extern "C" int moe_quant_rows_int8(const void* src, int src_dtype, int64_t rows, int64_t cols, int64_t ld, void* dst,
                                   float* scale, void* stream) {
  return quant_rows_int8(src, src_dtype, rows, cols, ld, dst, scale, nullptr, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int moe_dequant_rows(const void* q, int q_format, const float* scale, int64_t rows, int64_t cols, void* dst,
                                int dst_dtype, void* stream) {
  if (rows < 0 || cols < 16 || cols % 16 || cols > INT32_MAX / 2 || (q_format != MOE_INT8 && q_format != MOE_E4M3) ||
      (dst_dtype != MOE_BF16 && dst_dtype != MOE_F32))
    return fail_arg("moe_dequant_rows: bad arguments rows=%lld cols=%lld (need cols %% 16 == 0, int8 or e4m3 rows, bf16 or "
                    "fp32 values)", (long long)rows, (long long)cols);
  if (rows == 0) return 0;
  if (!q || !scale || !dst || !al16_8(q) || !al16_8(dst)) return fail_arg("moe_dequant_rows: null or misaligned pointer");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto* qp = static_cast<const uint8_t*>(q);
#define MOE_DQ(F8, T, LPR)                                                                                             \
  MOE_LAUNCH("k_dequant_rows", (k_dequant_rows<F8, T, LPR>), dim3(q8_blocks(rows, LPR)), dim3(kQ8Threads), 0, s, qp, scale, \
             rows, (int)cols, static_cast<T*>(dst))
#define MOE_DQ_T(F8, LPR)                                       \
  do {                                                          \
    if (dst_dtype == MOE_BF16) MOE_DQ(F8, uint16_t, LPR);       \
    else MOE_DQ(F8, float, LPR);                                \
  } while (0)
  // lanes a row: 64, 128 or 256, by its 16-element pieces (65536 rows of 2048 e4m3: 256 lanes 101 us, 128 88)
  if (q_format == MOE_E4M3) {
    if (cols <= 1024) MOE_DQ_T(true, 64);
    else if (cols <= 2048) MOE_DQ_T(true, 128);
    else MOE_DQ_T(true, 256);
  } else {
    if (cols <= 1024) MOE_DQ_T(false, 64);
    else if (cols <= 2048) MOE_DQ_T(false, 128);
    else MOE_DQ_T(false, 256);
  }
#undef MOE_DQ_T
#undef MOE_DQ
  return check_launch("moe_dequant_rows");
}

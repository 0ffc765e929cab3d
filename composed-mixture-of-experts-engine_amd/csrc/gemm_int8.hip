// Products of int8 rows with int8 weights (a scale each row of either), whole or grouped by expert, and the SwiGLU experts
// on them.
//
//   y[m, n] = sx[m] sw[n] sum_k xq[m, k] wq[n, k]
//   experts: g, u = the gate and up products (fp32), act = silu(g) u rounded to bf16, quantized by row as any rows are
//            (csrc/int8.hip), y = its product with the down weights
//
// The sums are whole numbers in 32 bits (exact below K = 131072), so a row's result does not depend on the order of its sum,
// on the batch that it is in or on the form of the kernel.  Rows may be gathered: row m of the product is row
// row_slot[m] / top_k of xq (the dispatch plan's), so tokens are quantized once and never copied per expert.
//
// Few rows (k_i8_small): the weights' stream bounds the product.  A block owns 16 NF weight rows of one expert (gate/up: 8 NF
// gate rows and the matching up rows) and its NW waves each take every NW-th 128-byte column chunk of them, straight from
// memory into v_mfma_i32_16x16x64_i8 fragments (16 weight rows as the M operand, 16 tokens as the N operand): lane 16 q + r
// loads bytes [16 q, 16 q + 16) of a 64-byte half chunk of row r.  The k slot that a value lands in is free as long as both
// operands agree.  The waves' partial sums meet in LDS.  Every 64 rows of an expert are a pass of their own blocks over its
// weights.  Blocks start their chunks at different columns: rows lie a power of two apart, and blocks that walk them in step
// ask the same few memory channels.
#include <algorithm>

#include "common.h"
#include "quant8.h"

namespace moe {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct I8Args {
  const uint8_t* A;     // rows [T][K]
  const float* sa;      // their scales [T]
  const int* row_slot;  // row m of the product is row row_slot[m] / top_k of A; null: row m
  int top_k;
  int64_t T;            // rows of A
  const uint8_t* B;     // weights [E][N][K] (gate for the gate/up product)
  const uint8_t* B2;    // up weights
  const float* sb;      // their scales [E][N]
  const float* sb2;
  void* C;              // act [R][N] bf16 (gate/up) or y [R][N] bf16 / fp32
  const int* offsets;   // [E + 1]; null: one group of all R rows
  int64_t R;
  int K;                // bytes of a row of A and B
  int N;                // output columns
  int Tn;               // column tiles
  int E;
};

__device__ __forceinline__ i32x4 mma_i8(const u32x4& w, const u32x4& a, const i32x4& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, a), c, 0, 0, 0);
}
__device__ __forceinline__ float sig_i8(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// An expert's rows, kept inside the R that there are.
__device__ __forceinline__ int64_t seg(const I8Args& g, int e) {
  if (g.offsets == nullptr) return e == 0 ? 0 : g.R;
  return min(max((int64_t)g.offsets[e], (int64_t)0), g.R);
}
// The row of A behind row m of the product.
__device__ __forceinline__ int64_t source_row(const I8Args& g, int64_t m) {
  if (g.row_slot == nullptr) return m;
  return min((int64_t)max(g.row_slot[m] / g.top_k, 0), g.T - 1);
}

constexpr int kI8Pass = 64;  // rows of a pass

// One pass: rows [row0, row0 + min(rows, 16 MT)) of the segment against the block's 16 NF weight rows.
// GU: gate and up products and act; OT: the type of y (bf16 bits or fp32).
template <bool GU, typename OT, int NF, int NW, int MT>
__device__ __forceinline__ void i8_pass(const I8Args& g, int e, int64_t row0, int rows, int n0, uint32_t tile, int* red) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const uint32_t kb = (uint32_t)g.K;
  constexpr int RP = NF * 16 + 4;  // words a row of the partial sums
  const uint8_t* const base0 = g.B + (int64_t)e * g.N * g.K;
  const uint8_t* const base1 = GU ? g.B2 + (int64_t)e * g.N * g.K : nullptr;
  // fragment f of the 16 NF weight rows: GU: the first NF / 2 gate rows, the others up rows; rows past N repeat the last
  uint32_t wo[NF];
  const uint8_t* arow[MT];
#pragma unroll
  for (int f = 0; f < NF; ++f) wo[f] = (uint32_t)min(n0 + (GU ? f % (NF / 2) : f) * 16 + r, g.N - 1) * kb + q * 16;
#pragma unroll
  for (int m = 0; m < MT; ++m) arow[m] = g.A + source_row(g, row0 + min(m * 16 + r, rows - 1)) * g.K + q * 16;

  constexpr int AB = MT == 1 ? 2 : 1;  // chunks of token rows in flight or in use
  u32x4 wb[2][NF][2], ab[AB][MT][2];
  auto load_a = [&](int b, int c) {
    const uint32_t k0 = (uint32_t)c * 128;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bool in = k0 + s * 64 + q * 16 < kb;
      const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(in ? arow[m] + (k0 + s * 64) : arow[m] - q * 16);
        ab[b][m][s] = in ? v : z;
      }
    }
  };
  auto load = [&](int b, int c) {
    if constexpr (AB == 2) load_a(b, c);
    const uint32_t k0 = (uint32_t)c * 128;
    if (k0 + 128 <= kb) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int f = 0; f < NF; ++f)
          wb[b][f][s] = *reinterpret_cast<const u32x4*>((GU && f >= NF / 2 ? base1 : base0) + (wo[f] + (k0 + s * 64)));
    } else {  // the row's last, partial chunk: units past its end have any values (their tokens are zeros)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t k = k0 + s * 64 + q * 16 < kb ? k0 + s * 64 : 0u;
        const uint32_t at = k0 + s * 64 + q * 16 < kb ? 0u : q * 16;  // the row's first bytes for those
#pragma unroll
        for (int f = 0; f < NF; ++f)
          wb[b][f][s] = *reinterpret_cast<const u32x4*>((GU && f >= NF / 2 ? base1 : base0) + (wo[f] - at + k));
      }
    }
  };
  i32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[f][m] = i32x4{0, 0, 0, 0};
  auto mma = [&](int b, int c) {
    if constexpr (AB == 1) load_a(0, c);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[f][m] = mma_i8(wb[b][f][s], ab[AB == 2 ? b : 0][m][s], acc[f][m]);
  };
  const int nc = (g.K + 127) / 128;
  const int start = (int)__umulhi(tile * 0x9E3779B1u, (uint32_t)nc);
  auto at = [&](int i) {
    const int c = i + start;
    return c < nc ? c : c - nc;
  };
  int c = wv;
  if (c < nc) {
    load(0, at(c));
    for (;;) {
      if (c + NW < nc) load(1, at(c + NW));
      mma(0, at(c));
      c += NW;
      if (c >= nc) break;
      if (c + NW < nc) load(0, at(c + NW));
      mma(1, at(c));
      c += NW;
      if (c >= nc) break;
    }
  }

  // acc[f][m][j] of lane 16 q + r: weight row 16 f + 4 q + j, token row 16 m + r
  const float* const sb = g.sb + (int64_t)e * g.N;
  const float* const sb2 = GU ? g.sb2 + (int64_t)e * g.N : nullptr;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m * 16 >= rows) break;
    if (m > 0) __syncthreads();
#pragma unroll
    for (int f = 0; f < NF; ++f)
      *reinterpret_cast<i32x4*>(&red[(wv * 16 + r) * RP + f * 16 + q * 4]) = acc[f][m];
    __syncthreads();
    constexpr int PAIRS = GU ? NF * 4 : NF * 8;  // column pairs a row
    for (int u = tid; u < 16 * PAIRS; u += NW * 64) {
      const int mr = u / PAIRS, p = (u % PAIRS) * 2, n = n0 + p;
      if (m * 16 + mr >= rows || n >= g.N) continue;
      const int64_t row = row0 + m * 16 + mr;
      const float sx = g.sa[source_row(g, row)];
      int v[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const int2 s = *reinterpret_cast<const int2*>(&red[(x * 16 + mr) * RP + p]);
        v[0] += s.x;
        v[1] += s.y;
        if constexpr (GU) {
          const int2 t = *reinterpret_cast<const int2*>(&red[(x * 16 + mr) * RP + NF * 8 + p]);
          w[0] += t.x;
          w[1] += t.y;
        }
      }
      const float y0 = (float)v[0] * sx * sb[n], y1 = (float)v[1] * sx * sb[n + 1];
      if constexpr (GU) {
        const float u0 = (float)w[0] * sx * sb2[n], u1 = (float)w[1] * sx * sb2[n + 1];
        reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(g.C) + row * g.N + n)[0] =
            pack2bf(y0 * sig_i8(y0) * u0, y1 * sig_i8(y1) * u1);
      } else if constexpr (sizeof(OT) == 4) {
        *reinterpret_cast<float2*>(static_cast<float*>(g.C) + row * g.N + n) = float2{y0, y1};
      } else {
        reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(g.C) + row * g.N + n)[0] = pack2bf(y0, y1);
      }
    }
  }
}

template <bool GU, typename OT, int NF, int NW>
__global__ __launch_bounds__(NW * 64, 8 / NW) void k_i8_small(I8Args g) {
  __shared__ __attribute__((aligned(16))) int red[NW * 16 * (NF * 16 + 4)];
  const int slot = (int)(blockIdx.x / g.Tn), nt = (int)(blockIdx.x % g.Tn);
  int e = slot, pass = 0;
  if (slot >= g.E) {  // the (slot - E)-th of the passes past the experts' first ones
    const int lane = threadIdx.x & 63;
    int x = slot - g.E;
    for (int e0 = 0;; e0 += 64) {
      if (e0 >= g.E) return;
      const int i = e0 + lane;
      const int c = i < g.E ? max((int)(seg(g, i + 1) - seg(g, i) + kI8Pass - 1) / kI8Pass - 1, 0) : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        upto += lane >= o ? v : 0;
      }
      const unsigned long long past = __ballot(x < upto);
      if (past) {
        const int l = __builtin_ctzll(past);
        e = e0 + l;
        pass = x - (__shfl(upto, l) - __shfl(c, l)) + 1;
        break;
      }
      x -= __shfl(upto, 63);
    }
    e = __builtin_amdgcn_readfirstlane(e);
    pass = __builtin_amdgcn_readfirstlane(pass);
  }
  const int64_t m0 = seg(g, e) + (int64_t)pass * kI8Pass, hi = seg(g, e + 1);
  if (m0 >= hi) return;
  const int rows = (int)min(hi - m0, (int64_t)kI8Pass);
  const int n0 = nt * NF * (GU ? 8 : 16);
  const uint32_t tile = (uint32_t)(e * g.Tn + nt);
  if (rows > 32) i8_pass<GU, OT, NF, NW, 4>(g, e, m0, rows, n0, tile, red);
  else if (rows > 16) i8_pass<GU, OT, NF, NW, 2>(g, e, m0, rows, n0, tile, red);
  else i8_pass<GU, OT, NF, NW, 1>(g, e, m0, rows, n0, tile, red);
}

template <bool GU, typename OT>
int launch_small(const char* name, hipStream_t s, I8Args a) {
  const int64_t slots = a.E + a.R / kI8Pass;  // every expert's first pass, and as many more as R rows can need
  if (cdiv(a.N, GU ? 32 : 64) * (int64_t)a.E >= 512) {
    a.Tn = cdiv(a.N, GU ? 32 : 64);
    MOE_LAUNCH(name, (k_i8_small<GU, OT, 4, 4>), dim3((unsigned)(a.Tn * slots)), dim3(256), 0, s, a);
  } else {
    a.Tn = cdiv(a.N, GU ? 16 : 32);
    MOE_LAUNCH(name, (k_i8_small<GU, OT, 2, 8>), dim3((unsigned)(a.Tn * slots)), dim3(512), 0, s, a);
  }
  return check_launch(name);
}

template <bool GU, typename OT>
int product(const char* name, hipStream_t s, const I8Args& a) {
  return launch_small<GU, OT>(name, s, a);
}

bool al16_i8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

// Sizes that the kernels' 32-bit quantities hold: sums (127 * 127 K), row offsets inside an expert's matrix, block counts.
constexpr int64_t kI8MaxK = 131056;
bool i8_sizes(int64_t R, int64_t K, int64_t N, int64_t E) {
  return R >= 0 && R <= INT32_MAX / 2 && K >= 16 && K % 16 == 0 && K <= kI8MaxK && N >= 8 && N % 8 == 0 && E >= 1 && E <= 1024 &&
         N * K < ((int64_t)1 << 32) && (E + R / kI8Pass + 1) * ((N + 15) / 16) < INT32_MAX;
}
}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_matmul_int8(const void* xq, const float* sx, const void* wq, const float* sw, const int32_t* offsets,
                               int64_t R, int64_t K, int64_t N, int64_t E, void* y, int y_dtype, void* stream) {
  if (!i8_sizes(R, K, N, E) || (y_dtype != MOE_BF16 && y_dtype != MOE_F32) || (!offsets && E != 1))
    return fail_arg("moe_matmul_int8: bad arguments R=%lld K=%lld N=%lld E=%lld (need K %% 16 == 0, K <= %lld, N %% 8 == 0, "
                    "N K < 2^32, E <= 1024, bf16 or fp32 y; E == 1 without offsets)", (long long)R, (long long)K, (long long)N,
                    (long long)E, (long long)kI8MaxK);
  if (R == 0) return 0;
  if (!xq || !sx || !wq || !sw || !y || !al16_i8(xq) || !al16_i8(wq) || !al16_i8(y))
    return fail_arg("moe_matmul_int8: null or misaligned pointer");
  I8Args a{};
  a.A = static_cast<const uint8_t*>(xq);
  a.sa = sx;
  a.top_k = 1;
  a.T = R;
  a.B = static_cast<const uint8_t*>(wq);
  a.sb = sw;
  a.C = y;
  a.offsets = offsets;
  a.R = R;
  a.K = (int)K;
  a.N = (int)N;
  a.E = (int)E;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return y_dtype == MOE_BF16 ? product<false, uint16_t>("k_matmul_int8", s, a) : product<false, float>("k_matmul_int8", s, a);
}

// act (bf16), then act in int8 and its scales
extern "C" size_t moe_swiglu_fwd_int8_workspace(int64_t R, int64_t F) {
  if (R <= 0 || F <= 0) return 0;
  return up256((size_t)R * F * 2) + up256((size_t)R * F) + up256((size_t)R * 4);
}

extern "C" int moe_swiglu_fwd_int8(const void* xq, const float* sx, int64_t T, const int32_t* row_slot, int64_t top_k,
                                   const void* wg_q, const float* sg, const void* wu_q, const float* su, const void* wd_q,
                                   const float* sd, const int32_t* offsets, int64_t R, int64_t H, int64_t F, int64_t E, void* y,
                                   void* workspace, size_t ws_bytes, void* stream) {
  if (!i8_sizes(R, H, F, E) || !i8_sizes(R, F, H, E) || T < 0 || T > INT32_MAX / 2 || (row_slot ? top_k < 1 || top_k > INT32_MAX : T != R))
    return fail_arg("moe_swiglu_fwd_int8: bad arguments T=%lld R=%lld H=%lld F=%lld E=%lld top_k=%lld (need H %% 16 == 0, "
                    "F %% 16 == 0, H and F <= %lld, H F < 2^32, E <= 1024; T == R without row_slot)", (long long)T, (long long)R,
                    (long long)H, (long long)F, (long long)E, (long long)top_k, (long long)kI8MaxK);
  if (R == 0) return 0;
  if (T == 0) return fail_arg("moe_swiglu_fwd_int8: rows of no token");
  if (!xq || !sx || !wg_q || !sg || !wu_q || !su || !wd_q || !sd || !offsets || !y || !al16_i8(xq) || !al16_i8(wg_q) ||
      !al16_i8(wu_q) || !al16_i8(wd_q) || !al16_i8(y) || !al16_i8(workspace))
    return fail_arg("moe_swiglu_fwd_int8: null or misaligned pointer");
  if (!workspace || ws_bytes < moe_swiglu_fwd_int8_workspace(R, F))
    return set_error("moe_swiglu_fwd_int8: workspace %zu < %zu bytes", ws_bytes, moe_swiglu_fwd_int8_workspace(R, F)),
           MOE_EWORKSPACE;
  uint8_t* const act = static_cast<uint8_t*>(workspace);
  uint8_t* const aq = act + up256((size_t)R * F * 2);
  float* const as = reinterpret_cast<float*>(aq + up256((size_t)R * F));
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  I8Args a{};
  a.A = static_cast<const uint8_t*>(xq);
  a.sa = sx;
  a.row_slot = row_slot;
  a.top_k = row_slot ? (int)top_k : 1;
  a.T = T;
  a.B = static_cast<const uint8_t*>(wg_q);
  a.B2 = static_cast<const uint8_t*>(wu_q);
  a.sb = sg;
  a.sb2 = su;
  a.C = act;
  a.offsets = offsets;
  a.R = R;
  a.K = (int)H;
  a.N = (int)F;
  a.E = (int)E;
  if (int rc = product<true, uint16_t>("k_i8_gate_up", s, a)) return rc;
  if (int rc = quant_rows_int8(act, MOE_BF16, R, F, F, aq, as, offsets + E, s)) return rc;
  I8Args b{};
  b.A = aq;
  b.sa = as;
  b.top_k = 1;
  b.T = R;
  b.B = static_cast<const uint8_t*>(wd_q);
  b.sb = sd;
  b.C = y;
  b.offsets = offsets;
  b.R = R;
  b.K = (int)F;
  b.N = (int)H;
  b.E = (int)E;
  return product<false, uint16_t>("k_i8_down", s, b);
}

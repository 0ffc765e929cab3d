// Grouped SwiGLU expert products on MXFP4 weights (4-bit e2m1 elements, one E8M0 scale per 32 along the reduction) and
// bf16 rows, fp32 sums.
//
//   g = Wg x, u = Wu x, act = silu(g) u (rounded to bf16: the down projection's matrix instruction takes bf16), y = Wd act.
//
// A 4-bit value times its power-of-two scale is exact in bf16, and v_cvt_scalef32_pk_bf16_fp4 forms two of them in one
// instruction, so the products run on the bf16 matrix instructions with weights dequantized between the load and the MFMA
// and nothing lost: half a vector instruction a weight.  With r rows an expert costs 6 r F H flops over 1.59 F H bytes of
// weights.
//
// Few rows (k_mx_small): the weights' stream bounds both products.  A block owns 16 NF weight rows of one expert (gate/up
// product: 8 NF gate and the matching up rows) and its NW waves each take every NW-th 128-column chunk of them, straight
// from HBM into MFMA fragments: a lane's 16-byte load is one 32-element block of one row, with its one scale byte, and
// feeds four v_mfma_f32_16x16x32_bf16, 8 elements each.  The k slot that a value lands in is free as long as both operands
// agree: lane 16 q + r holds block 4 c + q of row r, and takes elements 128 c + 32 q + 8 s + [0, 8) of token row r for the
// s-th of the four.  The waves' partial sums meet in LDS in wave order.
#include <algorithm>

#include "common.h"

namespace moe {
namespace {

struct MxArgs {
  const uint16_t* A;   // rows [R][K] bf16
  const uint8_t* B;    // weights [E][N][K / 2] (gate for the gate/up product)
  const uint8_t* B2;   // up weights
  const uint8_t* S;    // scales [E][N][K / 32]
  const uint8_t* S2;
  uint16_t* C;         // act [R][F] / y [R][N]
  uint16_t* C2;        // hgu [R][2F] (gate/up product; null for inference)
  const int* offsets;  // [E+1]
  int K;               // reduction length
  int N;               // output columns: F (gate/up) or H
  int Tn;              // column tiles
  int E;
};

__device__ __forceinline__ float sig_mx(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// 8 consecutive 4-bit elements to bf16.
__device__ __forceinline__ bf16x8 mx_frag(uint32_t w, float sc) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
  return __builtin_bit_cast(bf16x8, r);
}

// One pass: rows [row0, row0 + min(rows, 16 MT)) of the segment against the block's 16 NF weight rows.
template <bool GU, int NF, int NW, int MT>
__device__ __forceinline__ void mx_pass(const MxArgs& g, int e, int64_t row0, int rows, int n0, uint32_t tile, float* red) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int nb = g.K / 32;          // blocks of a row
  constexpr int RP = NF * 16 + 4;   // floats a row of the partial sums
  const int64_t eb = (int64_t)e * g.N * nb;  // blocks before this expert
  const uint8_t* const wb[2] = {g.B + eb * 16, GU ? g.B2 + eb * 16 : nullptr};
  const uint8_t* const sb[2] = {g.S + eb, GU ? g.S2 + eb : nullptr};
  // fragment f of the 16 NF weight rows: GU: the first NF / 2 gate rows, the others up rows; rows past N repeat the last
  uint32_t wo[NF], ao[MT];  // in blocks of 32 elements
#pragma unroll
  for (int f = 0; f < NF; ++f)
    wo[f] = (uint32_t)min(n0 + (GU ? f % (NF / 2) : f) * 16 + r, g.N - 1) * (uint32_t)nb;
#pragma unroll
  for (int m = 0; m < MT; ++m) ao[m] = (uint32_t)min(m * 16 + r, rows - 1) * (uint32_t)nb;
  const uint16_t* const arow = g.A + row0 * g.K;

  u32x4 w[2][NF], a[2][MT][4];
  uint32_t sc[2][NF];
  auto load = [&](int b, int c) {
    const bool in = c * 4 + q < nb;  // blocks past the row's end are zeros on both sides
    const uint32_t blk = in ? c * 4 + q : 0;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int o = GU && f >= NF / 2;
      w[b][f] = *reinterpret_cast<const u32x4*>(wb[o] + (int64_t)(wo[f] + blk) * 16);
      sc[b][f] = sb[o][wo[f] + blk];
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        a[b][m][s] = *reinterpret_cast<const u32x4*>(arow + (int64_t)(ao[m] + blk) * 32 + s * 8);
    if (!in) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        w[b][f] = u32x4{0u, 0u, 0u, 0u};
        sc[b][f] = 127u;
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int s = 0; s < 4; ++s) a[b][m][s] = u32x4{0u, 0u, 0u, 0u};
    }
  };
  f32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto mma = [&](int b) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const bf16x8 wf = mx_frag(w[b][f][s], __uint_as_float(sc[b][f] << 23));
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[f][m] = mfma16x16x32(wf, __builtin_bit_cast(bf16x8, a[b][m][s]), acc[f][m]);
      }
  };
  const int nc = (nb + 3) / 4;
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
      mma(0);
      c += NW;
      if (c >= nc) break;
      if (c + NW < nc) load(0, at(c + NW));
      mma(1);
      c += NW;
      if (c >= nc) break;
    }
  }

  // acc[f][m][j] of lane 16 q + r: weight row 16 f + 4 q + j, token row 16 m + r
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m * 16 >= rows) break;
    if (m > 0) __syncthreads();
#pragma unroll
    for (int f = 0; f < NF; ++f)
      *reinterpret_cast<f32x4*>(&red[(wv * 16 + r) * RP + f * 16 + q * 4]) = acc[f][m];
    __syncthreads();
    constexpr int PAIRS = GU ? NF * 4 : NF * 8;  // column pairs a row
    for (int u = tid; u < 16 * PAIRS; u += NW * 64) {
      const int mr = u / PAIRS, p = (u % PAIRS) * 2;
      const int n = n0 + p;
      if (m * 16 + mr >= rows || n >= g.N) continue;
      const int64_t row = row0 + m * 16 + mr;
      float v[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const float2 s = *reinterpret_cast<const float2*>(&red[(x * 16 + mr) * RP + p]);
        v[0] += s.x;
        v[1] += s.y;
        if constexpr (GU) {
          const float2 o = *reinterpret_cast<const float2*>(&red[(x * 16 + mr) * RP + NF * 8 + p]);
          t[0] += o.x;
          t[1] += o.y;
        }
      }
      if constexpr (GU) {
        *reinterpret_cast<uint32_t*>(g.C + row * g.N + n) = pack2bf(v[0] * sig_mx(v[0]) * t[0], v[1] * sig_mx(v[1]) * t[1]);
        if (g.C2 != nullptr) {
          uint16_t* h = g.C2 + row * 2 * (int64_t)g.N + n;
          *reinterpret_cast<uint32_t*>(h) = pack2bf(v[0], v[1]);
          *reinterpret_cast<uint32_t*>(h + g.N) = pack2bf(t[0], t[1]);
        }
      } else {
        *reinterpret_cast<uint32_t*>(g.C + row * g.N + n) = pack2bf(v[0], v[1]);
      }
    }
  }
}

constexpr int kMxPass = 32;  // rows of a pass

template <bool GU, int NF, int NW>
__global__ __launch_bounds__(NW * 64) void k_mx_small(MxArgs g) {
  __shared__ __attribute__((aligned(16))) float red[NW * 16 * (NF * 16 + 4)];
  const int slot = (int)(blockIdx.x / g.Tn), nt = (int)(blockIdx.x % g.Tn);
  int e = slot, pass = 0;
  if (slot >= g.E) {  // the (slot - E)-th of the passes past the experts' first ones
    const int lane = threadIdx.x & 63;
    int x = slot - g.E;
    for (int e0 = 0;; e0 += 64) {
      if (e0 >= g.E) return;
      const int i = e0 + lane;
      const int c = i < g.E ? max((g.offsets[i + 1] - g.offsets[i] + kMxPass - 1) / kMxPass - 1, 0) : 0;
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
  const int m0 = g.offsets[e] + pass * kMxPass, hi = g.offsets[e + 1];
  if (m0 >= hi) return;
  const int n0 = nt * NF * (GU ? 8 : 16);
  const uint32_t tile = (uint32_t)(e * g.Tn + nt);
  if (hi - m0 > 16) mx_pass<GU, NF, NW, 2>(g, e, m0, min(kMxPass, hi - m0), n0, tile, red);
  else mx_pass<GU, NF, NW, 1>(g, e, m0, hi - m0, n0, tile, red);
}

template <bool GU>
int launch_small(const char* name, hipStream_t s, MxArgs a, int64_t E, int64_t R) {
  a.E = (int)E;
  const int64_t slots = E + R / kMxPass;  // every expert's first pass, and as many more as R rows can need
  a.Tn = cdiv(a.N, GU ? 32 : 64);
  if (a.Tn * slots > INT32_MAX) return fail_arg("%s: too many tiles", name);
  MOE_LAUNCH(name, (k_mx_small<GU, 4, 4>), dim3((unsigned)(a.Tn * slots)), dim3(256), 0, s, a);
  return check_launch(name);
}

bool al16x(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t al256x(size_t v) { return (v + 255) & ~(size_t)255; }

int mx_shape(const char* what, int64_t R, int64_t H, int64_t F, int64_t E) {
  const int64_t lim = INT32_MAX;
  if (R < 0 || R > lim || H < 32 || F < 32 || E < 1 || E > 1024 || H % 32 || F % 32 || H > lim / 64 || F > lim / 64 ||
      H * F > lim * 16)
    return fail_arg("%s: bad shape R=%lld H=%lld F=%lld E=%lld (need H%%32==0, F%%32==0, E<=1024)", what, (long long)R,
                    (long long)H, (long long)F, (long long)E);
  return 0;
}
}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_swiglu_fwd_mxfp4_workspace(int64_t R, int64_t H, int64_t F, int64_t E) {
  (void)H;
  if (R <= 0 || F <= 0 || E <= 0) return 0;
  return moe_swiglu_workspace(E) + al256x((size_t)R * F * 2);
}

extern "C" int moe_swiglu_fwd_mxfp4(const void* xp, const void* wg_q, const void* sg, const void* wu_q, const void* su,
                                    const void* wd_q, const void* sd, const int32_t* offsets, int64_t R, int64_t H,
                                    int64_t F, int64_t E, void* hgu, void* y, void* workspace, size_t ws_bytes,
                                    void* stream) {
  if (int rc = mx_shape("moe_swiglu_fwd_mxfp4", R, H, F, E)) return rc;
  if (R == 0) return 0;
  if (!xp || !wg_q || !sg || !wu_q || !su || !wd_q || !sd || !offsets || !y || !al16x(xp) || !al16x(wg_q) || !al16x(wu_q) ||
      !al16x(wd_q) || (hgu && !al16x(hgu)) || !al16x(y))
    return fail_arg("moe_swiglu_fwd_mxfp4: null or misaligned pointer");
  if (ws_bytes < moe_swiglu_fwd_mxfp4_workspace(R, H, F, E) || !workspace || !al16x(workspace))
    return set_error("moe_swiglu_fwd_mxfp4: workspace"), MOE_EWORKSPACE;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint16_t* act = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + moe_swiglu_workspace(E));
  MxArgs a{};
  a.offsets = offsets;
  a.A = static_cast<const uint16_t*>(xp);
  a.B = static_cast<const uint8_t*>(wg_q);
  a.B2 = static_cast<const uint8_t*>(wu_q);
  a.S = static_cast<const uint8_t*>(sg);
  a.S2 = static_cast<const uint8_t*>(su);
  a.C = act;
  a.C2 = static_cast<uint16_t*>(hgu);
  a.K = (int)H;
  a.N = (int)F;
  if (int rc = launch_small<true>("k_mx_small_fwd1", s, a, E, R)) return rc;
  MxArgs b{};
  b.offsets = offsets;
  b.A = act;
  b.B = static_cast<const uint8_t*>(wd_q);
  b.S = static_cast<const uint8_t*>(sd);
  b.C = static_cast<uint16_t*>(y);
  b.K = (int)F;
  b.N = (int)H;
  return launch_small<false>("k_mx_small_fwd2", s, b, E, R);
}

// ---- backward to the rows ----

extern "C" size_t moe_swiglu_bwd_mxfp4_workspace(int64_t R, int64_t H, int64_t F, int64_t E) {
  if (R <= 0 || H <= 0 || F <= 0 || E <= 0) return 0;
  return moe_swiglu_workspace(E) + moe_swiglu_split_workspace(R, H, F, E) + al256x((size_t)R * F * 4) +
         2 * al256x((size_t)E * F * H * 2);
}

extern "C" int moe_swiglu_bwd_mxfp4(const void* dy, const void* hgu, const void* wg_q, const void* sg, const void* wu_q,
                                    const void* su, const void* wd_q, const void* sd, const int32_t* offsets, int64_t R,
                                    int64_t H, int64_t F, int64_t E, void* dxp, void* workspace, size_t ws_bytes,
                                    void* stream) {
  if (int rc = mx_shape("moe_swiglu_bwd_mxfp4", R, H, F, E)) return rc;
  if (R == 0) return 0;
  if (!dy || !hgu || !wg_q || !sg || !wu_q || !su || !wd_q || !sd || !offsets || !dxp || !al16x(dy) || !al16x(hgu) ||
      !al16x(wg_q) || !al16x(wu_q) || !al16x(wd_q) || !al16x(dxp))
    return fail_arg("moe_swiglu_bwd_mxfp4: null or misaligned pointer");
  if (ws_bytes < moe_swiglu_bwd_mxfp4_workspace(R, H, F, E) || !workspace || !al16x(workspace))
    return set_error("moe_swiglu_bwd_mxfp4: workspace"), MOE_EWORKSPACE;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t gemm_ws = moe_swiglu_workspace(E) + moe_swiglu_split_workspace(R, H, F, E);
  char* ws = static_cast<char*>(workspace);
  void* dh = ws + gemm_ws;
  char* w0 = ws + gemm_ws + al256x((size_t)R * F * 4);
  char* w1 = w0 + al256x((size_t)E * F * H * 2);
  const int64_t n = E * F * H;
  if (int rc = dequant_mxfp4_bf16(wd_q, sd, n, w0, s)) return rc;
  if (int rc = swiglu_tiles(offsets, E, workspace, s)) return rc;
  if (int rc = swiglu_dact(dy, hgu, w0, offsets, R, H, F, E, dh, workspace, s)) return rc;
  if (int rc = dequant_mxfp4_bf16(wg_q, sg, n, w0, s)) return rc;
  if (int rc = dequant_mxfp4_bf16(wu_q, su, n, w1, s)) return rc;
  return swiglu_dxp(dh, w0, w1, offsets, R, H, F, E, dxp, workspace, gemm_ws, s);
}

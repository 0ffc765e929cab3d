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
// product: 8 NF gate and the matching up rows) and its NW waves each take every NW-th unit of 256 columns of them.  Lane
// 16 q + r of v_mfma_f32_16x16x32_bf16 wants row r's block 4 j + q, but sixteen rows' blocks side by side in a load are 64
// cache accesses of 16 bytes, about one a clock, and the vector cache then bounds the kernel (measured: 0.9 of one a clock).  So
// eight lanes fetch a row's 128-byte line, two units ahead, and the unit passes through the wave's own LDS, with no barrier.
// The k slot that a value lands in is free as long as both operands agree: a lane's block feeds four MFMAs, 8 elements each,
// and takes elements 8 s + [0, 8) of the same 32 of its token row for the s-th.  The waves' partial sums meet in LDS in wave
// order.  16 tokens, two experts each, E 8, H 4096, F 14336: 92 us for the gate/up product (500 MB, 5.4 TB/s) and 52 for the
// down projection (4.8 TB/s), where loads in the lanes' own order took 116 and 60.
//
// Many rows (k_mx_tile): 64, 128 or 256 rows of an expert by 256 weight rows.  The rows go through LDS in 64-wide slices, two
// at a time; a wave has weight rows of its own, dequantizes them between registers and feeds v_mfma_f32_32x32x16_bf16, half a
// conversion to 2, 4 or 8 row fragments.  64 rows read a weight so rarely that the vector cache bounds them too: their weights
// come by whole lines through the wave's LDS (1002 rows at the sizes above, tiles of 64 rows: 600 -> 500 us); after that
// LDS moves 7/8 of what it can by count, and the MFMAs are 46% busy.  128 and 256 rows load in the lanes' own order, whose accesses the matrix instructions
// cover; what bounds them is the matrix instructions' power (16384 rows: 4.76 ms, 5.77 TFLOP, 1210 TFLOP/s at 1.6 GHz).
#include <algorithm>
#include <utility>

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
  const int* tile_off; // [E+1] row-tile prefix (tiled form)
  float* part;         // partial tiles of a split last round (tiled down projection; null: no split)
  int npart;           // ... and how many of them an XCD has room for
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

struct __attribute__((packed)) MxBytes8 { uint32_t v[2]; };

// A wave's LDS: a unit of the block's 16 NF weight rows (128 bytes of each, swizzled) and their eight scale bytes.
constexpr int mx_stage(int NF) { return NF * 16 * 136; }

// One pass: rows [row0, row0 + min(rows, 16 MT)) of the segment against the block's 16 NF weight rows.
template <bool GU, int NF, int NW, int MT>
__device__ __forceinline__ void mx_pass(const MxArgs& g, int e, int64_t row0, int rows, int n0, uint32_t tile, uint8_t* stage,
                                        float* red) {
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int nb = g.K / 32;          // blocks of a row
  constexpr int RP = NF * 16 + 4;   // floats a row of the partial sums
  constexpr int NP = NF * 2;        // pieces of a unit: 8 weight rows each, GU: the first half gate rows, the others up rows
  const int64_t eb = (int64_t)e * g.N * nb;  // blocks before this expert
  const uint8_t* const wb[2] = {g.B + eb * 16, (GU ? g.B2 : g.B) + eb * 16};
  const uint8_t* const sb[2] = {g.S + eb, (GU ? g.S2 : g.S) + eb};
  // the weight row of row x of the block's; rows past N repeat the last
  auto wrow = [&](int x) { return (uint32_t)min(n0 + (GU ? x % (NF * 8) : x), g.N - 1) * (uint32_t)nb; };
  uint32_t wo[NP], ao[MT];  // the row's first block, and the token row's first byte
#pragma unroll
  for (int p = 0; p < NP; ++p) wo[p] = wrow(p * 8 + (lane >> 3));
  const uint32_t so = wrow(lane % (NF * 16));
  const bool sup = GU && lane % (NF * 16) >= NF * 8;
#pragma unroll
  for (int m = 0; m < MT; ++m) ao[m] = (uint32_t)min(m * 16 + r, rows - 1) * (uint32_t)g.K * 2u;
  const uint8_t* const arow = reinterpret_cast<const uint8_t*>(g.A + row0 * g.K);

  // A unit: 256 columns, one 128-byte line of 4-bit values of each weight row.  Eight lanes fetch a line; the matrix
  // instruction wants a row's blocks four lanes of sixteen apart, so the unit passes through the wave's own LDS.
  constexpr int AB = MT == 1 ? 2 : 1;  // units of token rows in flight or in use
  u32x4 w[2][NP], a[AB][MT][2][4];
  uint32_t sc[2][2];
  auto load_w = [&](int b, int u) {
    const int c = lane & 7;
    if (u * 8 + 8 <= nb) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
        w[b][p] = *reinterpret_cast<const u32x4*>(wb[GU && p >= NF] + u * 128 + (wo[p] + (uint32_t)c) * 16u);
      const MxBytes8 s = *reinterpret_cast<const MxBytes8*>((sup ? sb[1] : sb[0]) + u * 8 + so);
      sc[b][0] = s.v[0];
      sc[b][1] = s.v[1];
    } else {  // the row's last, partial unit: blocks past its end have any values and a scale of 1 (their tokens are zeros)
#pragma unroll
      for (int p = 0; p < NP; ++p)
        w[b][p] = *reinterpret_cast<const u32x4*>(wb[GU && p >= NF] + (wo[p] + (uint32_t)min(u * 8 + c, nb - 1)) * 16u);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sc[b][j] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int blk = u * 8 + j * 4 + k;
          const uint32_t s = (sup ? sb[1] : sb[0])[so + (uint32_t)min(blk, nb - 1)];
          sc[b][j] |= (blk < nb ? s : 127u) << (8 * k);
        }
      }
    }
  };
  auto put_w = [&](int b) {
    __asm__ volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int row = p * 8 + (lane >> 3);
      *reinterpret_cast<u32x4*>(stage + row * 128 + (((lane & 7) ^ ((row >> 1) & 7)) << 4)) = w[b][p];
    }
    if (lane < NF * 16) *reinterpret_cast<uint2*>(stage + NF * 16 * 128 + lane * 8) = uint2{sc[b][0], sc[b][1]};
    __asm__ volatile("" ::: "memory");
  };
  auto load_a = [&](int b, int u) {
    if (u * 8 + 8 <= nb) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            a[b][m][j][s] = *reinterpret_cast<const u32x4*>(arow + u * 512 + j * 256 + s * 16 + (ao[m] + (uint32_t)q * 64u));
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int blk = u * 8 + j * 4 + q;
        const bool in = blk < nb;
        const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(arow + (ao[m] + (in ? (uint32_t)blk * 64u : 0u) + s * 16u));
            a[b][m][j][s] = in ? v : z;
          }
      }
    }
  };
  f32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto mma = [&](int b) {
    uint2 sv[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) sv[f] = *reinterpret_cast<const uint2*>(stage + NF * 16 * 128 + (f * 16 + r) * 8);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4 wv4[NF];
      float sf[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int row = f * 16 + r;
        wv4[f] = *reinterpret_cast<const u32x4*>(stage + row * 128 + (((4 * j + q) ^ ((row >> 1) & 7)) << 4));
        sf[f] = __uint_as_float((((j ? sv[f].y : sv[f].x) >> (8 * q)) & 0xffu) << 23);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const bf16x8 wf = mx_frag(wv4[f][s], sf[f]);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[f][m] = mfma16x16x32(wf, __builtin_bit_cast(bf16x8, a[b][m][j][s]), acc[f][m]);
        }
    }
  };
  // the waves take every NW-th unit, from one on that differs between blocks
  const int nu = (nb + 7) / 8;
  const int start = (int)__umulhi(tile * 0x9E3779B1u, (uint32_t)nu);
  auto at = [&](int i) {
    const int u = i + start;
    return u < nu ? u : u - nu;
  };
  if (wv < nu) {
    load_w(0, at(wv));
    load_a(0, at(wv));
    if (wv + NW < nu) {
      load_w(1, at(wv + NW));
      if constexpr (AB == 2) load_a(1, at(wv + NW));
    }
    auto unit = [&](auto b_c, int u) {
      constexpr int b = decltype(b_c)::value;
      put_w(b);
      if constexpr (AB == 2) {
        if (u + 2 * NW < nu) load_w(b, at(u + 2 * NW));
        mma(b);
        if (u + 2 * NW < nu) load_a(b, at(u + 2 * NW));
      } else {
        __builtin_amdgcn_sched_barrier(0);
        mma(0);
        __builtin_amdgcn_sched_barrier(0);
        if (u + NW < nu) load_a(0, at(u + NW));
        if (u + 2 * NW < nu) load_w(b, at(u + 2 * NW));
      }
    };
    for (int u = wv;;) {
      unit(std::integral_constant<int, 0>{}, u);
      u += NW;
      if (u >= nu) break;
      unit(std::integral_constant<int, 1>{}, u);
      u += NW;
      if (u >= nu) break;
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
__global__ __launch_bounds__(NW * 64, 2) void k_mx_small(MxArgs g) {
  __shared__ __attribute__((aligned(16))) float red[NW * 16 * (NF * 16 + 4)];
  __shared__ __attribute__((aligned(16))) uint8_t stages[NW * mx_stage(NF)];
  uint8_t* const stage = stages + (threadIdx.x >> 6) * mx_stage(NF);
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
  if (hi - m0 > 16) mx_pass<GU, NF, NW, 2>(g, e, m0, min(kMxPass, hi - m0), n0, tile, stage, red);
  else mx_pass<GU, NF, NW, 1>(g, e, m0, hi - m0, n0, tile, stage, red);
}

// 64 weight rows and four waves a block; two waves where a row has few units for them; where that leaves fewer than 256 blocks
// with rows, 32 rows and eight waves.  Down projection, us, (4, 4) | (4, 2) | (2, 8), rows of all experts: one token at
// H 4096, F 14336 (128 blocks, 56 units a row) 20 | 27 | 14; 16 tokens (512 blocks) 52 | 57 | 55; 512 rows of E 128, H 2048, F 768
// (4608 blocks, 3 units) 26 | 23 | 57; both products, 512 rows of E 64, H 4096, F 1536 (6 units) 140 | 132.
template <bool GU>
int launch_small(const char* name, hipStream_t s, MxArgs a, int64_t E, int64_t R) {
  a.E = (int)E;
  const int64_t slots = E + R / kMxPass;  // every expert's first pass, and as many more as R rows can need
  const bool wide = cdiv(a.N, GU ? 32 : 64) * std::min(E, R) >= 256;
  a.Tn = cdiv(a.N, (GU ? 16 : 32) * (wide ? 2 : 1));
  if (a.Tn * slots > INT32_MAX) return fail_arg("%s: too many tiles", name);
  if (wide && a.K <= 6 * 256) MOE_LAUNCH(name, (k_mx_small<GU, 4, 2>), dim3((unsigned)(a.Tn * slots)), dim3(128), 0, s, a);
  else if (wide) MOE_LAUNCH(name, (k_mx_small<GU, 4, 4>), dim3((unsigned)(a.Tn * slots)), dim3(256), 0, s, a);
  else MOE_LAUNCH(name, (k_mx_small<GU, 2, 8>), dim3((unsigned)(a.Tn * slots)), dim3(512), 0, s, a);
  return check_launch(name);
}

// ---- many rows ----
template <int P>
__device__ __forceinline__ uint32_t mx_pair(uint32_t w, float sc) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, P));
}

// The expert of logical tile L: the experts whose tiles all come before it.
__device__ __forceinline__ int mx_expert(const MxArgs& g, int L, int lane) {
  int e = 0;
  for (int e0 = 0; e0 < g.E; e0 += 64) {
    const int i = e0 + lane;
    const int n = __popcll(__ballot(i < g.E && g.tile_off[min(i, g.E - 1) + 1] * g.Tn <= L));
    e += n;
    if (n < 64) break;
  }
  return __builtin_amdgcn_readfirstlane(e);
}

// Blocks of a tiled product that an XCD's 32 CUs hold at once.
__host__ __device__ constexpr int mx_resident(int bm) { return bm == 256 ? 32 : 64; }

// The last round of a product: an XCD's n tiles run `resident` at a time, and its last n % resident leave the rest of it
// idle; with few rows that round is all there is.  Those tiles are split over their slices, in rounds of G, into `parts`
// blocks each, whose fp32 tiles go to memory and are added in order by k_mx_reduce.  parts (1 to 8) is the one with the
// least estimated time in slices: the rounds that the parts take, plus `over` slices a part for writing and reading back its
// tile, plus the reduction's launch.  Every block computes it from the device's tile count, and the reduction again.
struct MxSplit {
  int full, rest, parts;  // whole tiles; split tiles; blocks of each
};
__device__ __forceinline__ MxSplit mx_split(int n, int ns, int npart, int resident, int G, int over = 16) {
  MxSplit s{0, 0, 1};
  if (n <= 0) return s;
  s.rest = n % resident;
  s.full = n - s.rest;
  int cost = ns;
  for (int S = 2; s.rest > 0 && S <= 8; ++S) {
    if (s.rest * S > npart || S * G > ns) break;
    const int c = (s.rest * S + resident - 1) / resident * ((ns + S - 1) / S + over) + 5;
    if (c < cost) {
      cost = c;
      s.parts = S;
    }
  }
  return s;
}

// BM: rows of a tile.  MW: 32-row weight fragments of a wave (the block's four waves lie side by side on the weights).
// G: 64-wide slices of weights in flight or in use (a slice's registers are loaded with slice i + G as soon as slice i is
// converted).  XD: slices of the rows on their way from memory to LDS.
template <int BM, int MW, int G, int XD, bool GU>
__global__ __launch_bounds__(256, BM * MW >= 512 ? 1 : 2) void k_mx_tile(MxArgs g) {
  constexpr bool EVEN = BM == 256;                  // K % 128 == 0: rounds of two whole slices, nothing to mask
  constexpr int NB = BM / 32;                       // token fragments, and 16-byte pieces of a thread's share of a slice
  constexpr int BN = 128 * MW;                      // weight rows of the tile
  constexpr int CW = GU ? BN / 2 : BN;              // output columns of the tile
  constexpr int WC = CW / 4;                        // ... and of a wave
  constexpr int SLICE = BM * 128;                   // LDS bytes of a 64-wide slice of the rows
  constexpr int CP = BN + 8;                        // pitch of the output tile (bf16)
  constexpr bool VIA = BM == 64;                     // weights by whole 128-byte lines and through the wave's own LDS
  constexpr int WST = VIA ? mx_stage(4) : 0;        // ... a round of 64 rows and their scales
  static_assert(!VIA || (MW == 2 && G == 4));
  constexpr int SMEM = std::max(2 * SLICE + 4 * WST, BM * CP * 2);
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i32 = lane & 31, h = lane >> 5;

  // XCD-contiguous logical order over a 1-D grid sized for the most tiles any routing can produce: the tiles that there
  // are, split into 8 contiguous ranges (blockIdx mod 8), row tiles of a column tile next to each other
  const int total = g.tile_off[g.E] * g.Tn;
  const int chunk = (total + 7) >> 3, xcd = (int)(blockIdx.x & 7);
  int slot = (int)(blockIdx.x >> 3);
  int b0 = 0, b1 = (g.K + 63) / 64;   // the block's slices of the reduction
  float* part_out = nullptr;
  if constexpr (!GU) {
    if (g.part != nullptr) {
      const MxSplit sp = mx_split(min(chunk, total - xcd * chunk), b1, g.npart, mx_resident(BM), G);
      if (sp.parts > 1 && slot >= sp.full) {
        const int j = slot - sp.full, t = j / sp.parts, p = j - t * sp.parts;
        if (t >= sp.rest) return;
        slot = sp.full + t;
        b0 = __builtin_amdgcn_readfirstlane(b1 / G * p / sp.parts * G);
        b1 = __builtin_amdgcn_readfirstlane(p + 1 == sp.parts ? b1 : b1 / G * (p + 1) / sp.parts * G);
        part_out = g.part + (int64_t)(xcd * g.npart + j) * (BM * BN);
      }
    }
  }
  const int L = xcd * chunk + slot;
  if (slot >= chunk || L >= total) return;
  const int e = mx_expert(g, L, lane);
  const int cnt = g.tile_off[e + 1] - g.tile_off[e], local = L - g.tile_off[e] * g.Tn;
  const int nt = local / cnt, mt = local - nt * cnt;
  const int mbase = g.offsets[e] + mt * BM, mlen = min(BM, g.offsets[e + 1] - mbase);
  const int n0 = nt * CW;
  const int K = g.K, nb = K / 32;

  // Slices: if K is no multiple of 64, slice 0 holds a row's last 32 values (its loads are the checked ones) and slice i the
  // 64 from 64 (i - 1) on.  The loop takes them in rounds of G; a slice behind the last, ns, is zeros.
  // A part of a split tile starts at slice b0.
  const int lead = b0 > 0 ? 0 : (K + 63) / 64 - K / 64, ns = b1 - b0;  // ns - lead >= 2: K >= 128, parts have rounds of G
  const int first = b0 > 0 ? b0 - ((K + 63) / 64 - K / 64) : 0;         // whole slices of the row in front of the block's

  // rows: instruction j = NB wv + p of a slice fills rows 8 j + lane / 8; a row's eight 16-byte chunks are swizzled so that
  // the 16 rows a fragment read touches at once lie in distinct banks
  const uint8_t* const xbase = reinterpret_cast<const uint8_t*>(g.A + (int64_t)mbase * K + first * 64);
  uint32_t xo[NB];  // the piece's row and chunk, in bytes
#pragma unroll
  for (int p = 0; p < NB; ++p) {
    const int row = 8 * (NB * wv + p) + (lane >> 3);
    xo[p] = ((uint32_t)min(row, mlen - 1) * (uint32_t)K + (uint32_t)(((lane & 7) ^ ((row >> 1) & 7)) * 8)) * 2u;
  }
  // weights: the wave's MW fragments of 32 rows, straight to registers; GU: gate rows, then the same up rows
  const int64_t eb = (int64_t)e * g.N * nb;
  auto wbase = [&](int m) { return (GU && m >= MW / 2 ? g.B2 : g.B) + eb * 16 + first * 32; };
  auto sbase = [&](int m) { return (GU && m >= MW / 2 ? g.S2 : g.S) + eb + first * 2; };
  uint32_t wo[MW];  // the row's first block
#pragma unroll
  for (int m = 0; m < MW; ++m)
    wo[m] = (uint32_t)min(n0 + wv * WC + (GU ? m % (MW / 2) : m) * 32 + i32, g.N - 1) * (uint32_t)nb;

  // scale bytes: of a slice (G == 2), or of two slices in one word; a lane's byte is 8 h (+ 16) bits up
  constexpr int SJ = G == 2 ? 1 : 2;
  u32x4 xs[XD][NB], w[G][MW];
  uint32_t sw[G / SJ][MW];
  auto load_x = [&](int slot, int i, int p) {
    xs[slot][p] = *reinterpret_cast<const u32x4*>(xbase + (int64_t)(min(i, ns - 1) - lead) * 128 + xo[p]);
  };
  auto load_x_first = [&](int p) {
    const int row = 8 * (NB * wv + p) + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
    const bool in = lead == 0 || c < 4;
    const u32x4 v = *reinterpret_cast<const u32x4*>(
        xbase + (in ? xo[p] + (lead ? (uint32_t)(K - 32) * 2u : 0u) : xo[p] - (uint32_t)c * 16u));
    xs[0][p] = in ? v : u32x4{0u, 0u, 0u, 0u};
  };
  auto write_x = [&](int slot, int i, int p) {
    const uint32_t keep = EVEN || i < ns ? ~0u : 0u;
    __asm__ volatile("" ::: "memory");
    *reinterpret_cast<u32x4*>(smem + (i & 1) * SLICE + (NB * wv + p) * 1024 + lane * 16) = xs[slot][p] & keep;
    __asm__ volatile("" ::: "memory");
  };
  struct __attribute__((packed)) Bytes4 { uint32_t v; };
  struct __attribute__((packed)) Bytes2 { uint16_t v; };
  // slice i's weights; those behind the last slice are never used
  auto load_w = [&](int slot, int i) {
    const int at = min(i, ns - 1) - lead;
#pragma unroll
    for (int m = 0; m < MW; ++m)
      w[slot][m] = *reinterpret_cast<const u32x4*>(wbase(m) + (int64_t)at * 32 + (wo[m] + (uint32_t)h) * 16u);
  };
  // the scales of slices [i, i + SJ); of the last slice alone, those of the last two
  auto load_s = [&](int slot, int i) {
    const int at = min(i, ns - SJ) - lead;
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      const uint8_t* const s = sbase(m) + (int64_t)at * 2 + wo[m];
      sw[slot][m] = SJ == 2 ? reinterpret_cast<const Bytes4*>(s)->v : (uint32_t)reinterpret_cast<const Bytes2*>(s)->v;
    }
  };
  // both of the first round, in which slice 0 may be half a slice (its second half: any weights, a finite scale)
  auto load_w_first = [&](int l) {
    const bool in = l < ns && (l >= lead || h == 0);
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      const uint32_t o = wo[m] + (uint32_t)(!in ? 0 : l >= lead ? 2 * (l - lead) + h : nb - 1);
      w[l][m] = *reinterpret_cast<const u32x4*>(wbase(m) + o * 16u);
      const uint32_t s = (in ? (uint32_t)*(sbase(m) + o) : 127u) << (16 * (l % SJ) + 8 * h);
      sw[l / SJ][m] = l % SJ == 0 ? s : sw[l / SJ][m] | s;
    }
  };
  // VIA: a round of four slices of the wave's 64 rows.  Eight lanes fetch a row's 128 bytes (piece p: rows 8 p + lane / 8), a
  // lane the scales of row `lane`; a row's chunks are swizzled in LDS as the token rows' are.
  uint8_t* const wst = smem + 2 * SLICE + wv * WST;
  u32x4(&wr)[G * MW] = reinterpret_cast<u32x4(&)[G * MW]>(w);
  uint32_t sr[2];
  // (N % 32 == 0: a fragment's 32 rows lie inside the matrix or past it; those past it repeat the last ones)
  auto row0 = [&](int m) { return min(n0 + wv * WC + (GU ? 0 : m * 32), g.N - 32); };
  auto piece = [&](int p) { return wbase(p / 4) + (int64_t)(row0(p / 4) + p % 4 * 8) * nb * 16; };
  const uint32_t wp = (uint32_t)(lane >> 3) * (uint32_t)nb;
  const uint32_t sp = (uint32_t)(lane < 32 ? row0(0) : row0(MW - 1)) * (uint32_t)nb + (uint32_t)i32 * (uint32_t)nb;
  const uint8_t* const srow = lane < 32 ? sbase(0) : sbase(MW - 1);
  auto load_round = [&](int i) {  // slices [i, i + 4); those behind the last one again
    const int at = min(i + ((lane & 7) >> 1), ns - 1) - lead;
    const uint32_t o = (wp + (uint32_t)(2 * at + (lane & 1))) * 16u;
#pragma unroll
    for (int p = 0; p < 8; ++p) wr[p] = *reinterpret_cast<const u32x4*>(piece(p) + o);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      sr[k] = reinterpret_cast<const Bytes4*>(srow + (int64_t)(min(i + 2 * k, ns - 2) - lead) * 2 + sp)->v;
  };
  auto load_round_first = [&] {
    auto block = [&](int l, int hh) {
      return (uint32_t)(l >= ns || (l < lead && hh) ? 0 : l >= lead ? 2 * (l - lead) + hh : nb - 1);
    };
#pragma unroll
    for (int p = 0; p < 8; ++p)
      wr[p] = *reinterpret_cast<const u32x4*>(piece(p) + (wp + block((lane & 7) >> 1, lane & 1)) * 16u);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sr[k] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int l = 2 * k + b / 2, hh = b & 1;
        const uint32_t v = srow[sp + block(l, hh)];
        sr[k] |= (l < lead && hh ? 127u : v) << (8 * b);
      }
    }
  };
  auto put_round = [&](int i) {
    __asm__ volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int row = p * 8 + (lane >> 3);
      *reinterpret_cast<u32x4*>(wst + row * 128 + (((lane & 7) ^ ((row >> 1) & 7)) << 4)) = wr[p];
    }
    // (the last slice alone comes with the one in front of it)
    const uint32_t s0 = i > 0 && i == ns - 1 ? sr[0] >> 16 : sr[0], s1 = i > 0 && i + 2 == ns - 1 ? sr[1] >> 16 : sr[1];
    *reinterpret_cast<uint2*>(wst + 64 * 128 + lane * 8) = uint2{s0, s1};
    __asm__ volatile("" ::: "memory");
  };
  u32x4 wl[MW];     // the slice in use
  uint32_t sl[MW];  // its scale bytes
  auto take = [&](auto l_c) {  // slice l of the round in LDS
    constexpr int l = decltype(l_c)::value;
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      const int row = m * 32 + i32;
      wl[m] = *reinterpret_cast<const u32x4*>(wst + row * 128 + (((2 * l + h) ^ ((row >> 1) & 7)) << 4));
      sl[m] = wst[64 * 128 + row * 8 + 2 * l + h];
    }
    __asm__ volatile("" ::: "memory");
  };
  float sf[MW];  // the scales of the slice whose weights are used next (finite behind the last one)
  auto scales = [&](int l, int i) {
    const int up = 16 * (l % SJ) + (SJ == 2 && l % 2 == 0 && i >= G && i == ns - 1 ? 16 : 0);
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      const uint32_t b = VIA ? sl[m] << 23 : ((sw[l / SJ][m] >> (up + 8 * h)) & 0xffu) << 23;
      sf[m] = __uint_as_float(EVEN || i < ns ? b : 0x3f800000u);
    }
  };
  auto frag = [&](int i, int s, int n) {
    const int row = n * 32 + i32;
    return *reinterpret_cast<const bf16x8*>(smem + (i & 1) * SLICE + row * 128 + (((4 * h + s) ^ ((row >> 1) & 7)) << 4));
  };

  f32x16 acc[MW][NB];
#pragma unroll
  for (int m = 0; m < MW; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[m][n][j] = 0.f;
  bf16x8 fb0[NB], fb1[NB];
  u32x4 wf0[MW], wf1[MW];

  // One 16-wide step of slice i: MW NB MFMAs, and between them the next step's token fragments, its weights' conversion and
  // refill pieces [PLO, PHI) (slice i + 1 to LDS, i + 1 + XD from memory)
  auto step = [&](auto plo_c, auto phi_c, auto ns_c, const bf16x8(&cb)[NB], const u32x4(&cw)[MW], bf16x8(&nb_)[NB],
                  u32x4(&nw)[MW], int ni, auto nl_c, auto xl_c, int i) {
    constexpr int PLO = decltype(plo_c)::value, PHI = decltype(phi_c)::value;
    constexpr int NS = decltype(ns_c)::value, NL = decltype(nl_c)::value, XL = decltype(xl_c)::value;
    constexpr int SLOTS = MW * NB, CV = MW * 4;
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (([&] {
         constexpr int n = I / MW, m = I % MW;
         acc[m][n] = mfma32x32x16(__builtin_bit_cast(bf16x8, cw[m]), cb[n], acc[m][n]);
         __builtin_amdgcn_sched_barrier(0);
         if constexpr (I < NB) nb_[I] = frag(ni, NS, I);
         constexpr int C0 = I * CV / SLOTS, C1 = (I + 1) * CV / SLOTS;
         [&]<int... C>(std::integer_sequence<int, C...>) {
           ((nw[(C0 + C) / 4][(C0 + C) % 4] = mx_pair<(C0 + C) % 4>(VIA ? wl[(C0 + C) / 4][NS] : w[NL][(C0 + C) / 4][NS],
                                                                     sf[(C0 + C) / 4])), ...);
         }(std::make_integer_sequence<int, C1 - C0>{});
         constexpr int p = PLO + I - NB;
         if constexpr (I >= NB && p < PHI) {
           write_x(XL, i + 1, p);
           load_x(XL, i + 1 + XD, p);
         }
         __builtin_amdgcn_sched_barrier(0);
       }()), ...);
    }(std::make_integer_sequence<int, SLOTS>{});
  };
  constexpr int P1 = (NB + 2) / 3, P2 = (2 * NB + 2) / 3;
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  using IP1 = std::integral_constant<int, P1>;
  using IP2 = std::integral_constant<int, P2>;
  using IPN = std::integral_constant<int, NB>;
  // slice i, at position J of a round of G
  auto slice = [&](auto j_c, int i) {
    constexpr int J = decltype(j_c)::value;
    using NJ = std::integral_constant<int, (J + 1) % G>;
    using X = std::integral_constant<int, (J + 1) % XD>;
    step(I0{}, IP1{}, I1{}, fb0, wf0, fb1, wf1, i, j_c, X{}, i);
    if constexpr (VIA && J == G - 1) put_round(i + 1);
    step(IP1{}, IP2{}, I2{}, fb1, wf1, fb0, wf0, i, j_c, X{}, i);
    step(IP2{}, IPN{}, I3{}, fb0, wf0, fb1, wf1, i, j_c, X{}, i);
    if constexpr (VIA) {
      if constexpr (J == G - 1) load_round(i + 1 + G);
      take(NJ{});
    } else {
      load_w(J, i + G);
      if constexpr (SJ == 1) load_s(J, i + G);
      else if constexpr (J % 2 == 1) load_s(J / 2, i - 1 + G);
    }
    lds_sync();  // every wave's pieces of slice i + 1 are written and its reads of slice i done
    scales(NJ::value, i + 1);
    __builtin_amdgcn_sched_barrier(0);
    step(I0{}, I0{}, I0{}, fb1, wf1, fb0, wf0, i + 1, NJ{}, X{}, i);
  };
#pragma unroll
  for (int p = 0; p < NB; ++p) load_x_first(p);
  if constexpr (VIA) {
    load_round_first();
  } else {
#pragma unroll
    for (int l = 0; l < G; ++l) load_w_first(l);
  }
#pragma unroll
  for (int p = 0; p < NB; ++p) write_x(0, 0, p);
#pragma unroll
  for (int x = 1; x <= XD; ++x)
#pragma unroll
    for (int p = 0; p < NB; ++p) load_x(x % XD, x, p);
  if constexpr (VIA) {
    put_round(0);
    load_round(G);
    take(I0{});
  }
  __syncthreads();
  scales(0, 0);
#pragma unroll
  for (int n = 0; n < NB; ++n) fb0[n] = frag(0, 0, n);
#pragma unroll
  for (int m = 0; m < MW; ++m) wf0[m] = __builtin_bit_cast(u32x4, mx_frag(VIA ? wl[m][0] : w[0][m][0], sf[m]));
  for (int i = 0; i < ns; i += G) {
    [&]<int... J>(std::integer_sequence<int, J...>) {
      (slice(std::integral_constant<int, J>{}, i + J), ...);
    }(std::make_integer_sequence<int, G>{});
  }
  __syncthreads();

  if constexpr (!GU) {
    if (part_out != nullptr) {
      f32x4* const o = reinterpret_cast<f32x4*>(part_out) + wv * (MW * NB * 256) + lane;
#pragma unroll
      for (int m = 0; m < MW; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            o[((m * NB + n) * 4 + q) * 64] =
                f32x4{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
      return;
    }
  }

  // acc[m][n][j]: weight row 32 m + (j & 3) + 8 (j >> 2) + 4 h of the wave's, token row 32 n + i32.  The tile goes through
  // LDS so that its rows leave as whole segments.
  uint16_t* const ct = reinterpret_cast<uint16_t*>(smem);
  auto put = [&](int n, int col, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(ct + (n * 32 + i32) * CP + col + 4 * h) = uint2{pack2bf(a, b), pack2bf(c, d)};
  };
  auto out = [&](auto cols_c, auto at) {
    constexpr int UR = decltype(cols_c)::value / 8;  // 16-byte units of a row
    __syncthreads();
    for (int u = tid; u < BM * UR; u += 256) {
      const int row = u / UR, c = (u % UR) * 8;
      uint16_t* const dst = at(row, c);
      if (row < mlen && dst != nullptr) *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(ct + row * CP + c);
    }
  };
  if constexpr (GU) {
#pragma unroll
    for (int m = 0; m < MW / 2; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float a[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = acc[m][n][4 * q + j];
            a[j] = x * sig_mx(x) * acc[MW / 2 + m][n][4 * q + j];
          }
          put(n, wv * WC + m * 32 + q * 8, a[0], a[1], a[2], a[3]);
        }
    out(std::integral_constant<int, CW>{}, [&](int row, int c) {
      return n0 + c < g.N ? g.C + (int64_t)(mbase + row) * g.N + n0 + c : nullptr;
    });
    if (g.C2 == nullptr) return;
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < MW; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        put(n, (GU ? m / (MW / 2) * CW + m % (MW / 2) * 32 : m * 32) + wv * WC + q * 8, acc[m][n][4 * q],
            acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]);
  out(std::integral_constant<int, BN>{}, [&](int row, int c) -> uint16_t* {
    if constexpr (GU) {
      const int f = n0 + c % CW;
      return f < g.N ? g.C2 + (int64_t)(mbase + row) * 2 * g.N + (c < CW ? f : g.N + f) : nullptr;
    } else {
      return n0 + c < g.N ? g.C + (int64_t)(mbase + row) * g.N + n0 + c : nullptr;
    }
  });
}

// The split tiles' sums: blockIdx = (XCD, split tile), blockIdx.y an eighth of its 32 x 32 blocks.
template <int BM, int MW, int G>
__global__ __launch_bounds__(256) void k_mx_reduce(MxArgs g) {
  constexpr int NB = BM / 32, BN = 128 * MW, RES = mx_resident(BM), U = BM * BN / 4, BLOCKS = BM * BN / 1024;
  constexpr int BP = 36;  // pitch of a 32 x 32 block (bf16): 8-byte writes, rows 18 banks apart
  __shared__ __attribute__((aligned(16))) uint16_t blk[2][32 * BP];
  const int tid = threadIdx.x, lane = tid & 63, q = tid >> 6;
  const int xcd = (int)blockIdx.x / RES, t = (int)blockIdx.x % RES;
  const int total = g.tile_off[g.E] * g.Tn, chunk = (total + 7) >> 3;
  const MxSplit sp = mx_split(min(chunk, total - xcd * chunk), (g.K + 63) / 64, g.npart, RES, G);
  if (sp.parts == 1 || t >= sp.rest) return;
  const int L = xcd * chunk + sp.full + t, e = mx_expert(g, L, lane);
  const int cnt = g.tile_off[e + 1] - g.tile_off[e], local = L - g.tile_off[e] * g.Tn;
  const int nt = local / cnt, mt = local - nt * cnt;
  const int mbase = g.offsets[e] + mt * BM, mlen = min(BM, g.offsets[e + 1] - mbase);
  const f32x4* const src = reinterpret_cast<const f32x4*>(g.part + (int64_t)(xcd * g.npart + t * sp.parts) * (BM * BN));
  int buf = 0;
  for (int b = (int)blockIdx.y * (BLOCKS / 8); b < (int)(blockIdx.y + 1) * (BLOCKS / 8); ++b) {
    const int n = b % NB, m = b / NB;  // m: 32 weight rows of all waves'
    const int rb = n * 32, cb = nt * BN + m * 32;
    if (rb >= mlen || cb >= g.N) continue;  // the same for the whole block
    f32x4 s = src[b * 256 + q * 64 + lane];
    for (int p = 1; p < sp.parts; ++p) s += src[(int64_t)p * U + b * 256 + q * 64 + lane];
    *reinterpret_cast<uint2*>(&blk[buf][(lane & 31) * BP + q * 8 + (lane >> 5) * 4]) =
        uint2{pack2bf(s[0], s[1]), pack2bf(s[2], s[3])};
    __syncthreads();  // between a buffer's readers and its next writers lies the other buffer's barrier
    const int r = tid >> 3, c = (tid & 7) * 4;
    if (rb + r < mlen)  // N % 32 == 0
      *reinterpret_cast<uint2*>(g.C + (int64_t)(mbase + rb + r) * g.N + cb + c) =
          *reinterpret_cast<const uint2*>(&blk[buf][r * BP + c]);
    buf ^= 1;
  }
}

template <int BM, int MW, int G, int XD, bool GU>
int launch_tile_as(const char* name, hipStream_t s, MxArgs a, int64_t E, int64_t R) {
  a.E = (int)E;
  a.Tn = cdiv(a.N, GU ? 64 * MW : 128 * MW);
  const int64_t blocks = ((R + BM - 1) / BM + E) * a.Tn;
  if (blocks > INT32_MAX - 8) return fail_arg("%s: too many tiles", name);
  const int64_t more = a.part ? 8 * a.npart : 0;
  MOE_LAUNCH(name, (k_mx_tile<BM, MW, G, XD, GU>), dim3((unsigned)((blocks + 7) / 8 * 8 + more)), dim3(256), 0, s, a);
  if constexpr (!GU) {
    if (a.part != nullptr)
      MOE_LAUNCH("k_mx_reduce", (k_mx_reduce<BM, MW, G>), dim3(8 * mx_resident(BM), 8), dim3(256), 0, s, a);
  }
  return check_launch(name);
}
template <int BM, bool GU>
int launch_tile(const char* name, hipStream_t s, MxArgs a, int64_t E, int64_t R) {
  if constexpr (BM == 256) return launch_tile_as<256, 2, 2, 1, GU>(name, s, a, E, R);
  else if constexpr (BM == 128) return launch_tile_as<128, 2, 4, 1, GU>(name, s, a, E, R);
  else return launch_tile_as<64, 2, 4, 2, GU>(name, s, a, E, R);
}

// Rows of a tile (0: the few-row form), by the rows an expert has on average (the host does not know more) and by the gate/up
// product's tiles, which have to fill the chip: 512 blocks of 64 or 128 rows are resident at once, 256 of 256 rows.  The tiled
// loop takes reductions of 128 and more, and with 256 rows only multiples of 128.  Both products, us, by rows an expert
// (routed; few-row form | 64 | 128 | 256 rows):
//   E 8,   H 4096, F 14336   8: 160 | 237 | 342 | 539   16: 226 | 240 | 346 | 539   48: 519 | 245 | 361 | 555
//                            96: 882 | 387 | 387 | 576  256: - | 816 | 807 | 893    512: - | 1480 | 1370 | 1381
//   E 128, H 2048, F 768     8: 85 | 105 | 145 | 242    16: 113 | 108 | 148 | 253   48: 248 | 130 | 158 | 259
//                            96: 440 | 192 | 170 | 269  256: - | 425 | 382 | 430    512: - | 782 | 684 | 703
//   E 8,   H 1024, F 4096    16: 29 | 42 | 50 | 66      32: 38 | 44 | 53 | 68       64: 62 | 55 | 58 | 73
//                            128: - | 68 | 79 | 80      256: - | 91 | 102 | 119     512: - | 151 | 143 | 160
// A batch that goes to one expert pays for the average, as each 32 rows read its weights again (all rows to one expert, few-row
// form | the same in tiles of 64): 128 rows of E 8, H 4096, F 14336: 171 | 106; 2048 rows of E 128, H 2048, F 768: 71 | 45; 1200
// rows of E 76, H 4096, F 14336: 1166 | 448 (spread evenly the same batches take 188, 86 and 1699 in the few-row form).
int mx_rows(int64_t R, int64_t H, int64_t F, int64_t E) {
  if (H < 128 || F < 128) return 0;
  const bool even = H % 128 == 0 && F % 128 == 0;
  const int64_t tn = (F + 127) / 128;
  if (R <= (E * tn < 512 ? 40 : 16) * E) return 0;
  if (even && R > 512 * E && R / 256 * tn >= 1024) return 256;
  return R > 160 * E && std::max(R / 128, E) * tn >= 1024 ? 128 : 64;
}

// Room for the partial tiles of an XCD (tiles of bm rows, 256 columns): two rounds of parts, 8 a tile.  None for products of
// 16 rounds of tiles and more, of which the last is too little to pay for the reduction.
int mx_parts(int bm, int64_t R, int64_t E, int64_t N) {
  if (bm == 0) return 0;
  const int64_t tiles = ((R + bm - 1) / bm + E) * ((N + 255) / 256);
  if (R / bm * ((N + 255) / 256) >= 16 * 8 * mx_resident(bm)) return 0;
  return (int)std::min<int64_t>(2 * mx_resident(bm), 8 * ((tiles + 7) / 8));
}
size_t mx_part_bytes(int bm, int64_t R, int64_t E, int64_t N) {
  return (size_t)8 * mx_parts(bm, R, E, N) * bm * 256 * sizeof(float);
}

bool al16x(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t al256x(size_t v) { return (v + 255) & ~(size_t)255; }

int mx_shape(const char* what, int64_t R, int64_t H, int64_t F, int64_t E) {
  const int64_t lim = INT32_MAX;
  if (R < 0 || R > lim || H < 32 || F < 32 || E < 1 || E > 1024 || H % 32 || F % 32 || H > lim / 512 || F > lim / 512 ||
      H * F > lim * 2)
    return fail_arg("%s: bad shape R=%lld H=%lld F=%lld E=%lld (need H%%32==0, F%%32==0, E<=1024)", what, (long long)R,
                    (long long)H, (long long)F, (long long)E);
  return 0;
}
}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_swiglu_fwd_mxfp4_workspace(int64_t R, int64_t H, int64_t F, int64_t E) {
  if (R <= 0 || H <= 0 || F <= 0 || E <= 0) return 0;
  return moe_swiglu_workspace(E) + al256x((size_t)R * F * 2) + mx_part_bytes(mx_rows(R, H, F, E), R, E, H);
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
  const int bm = mx_rows(R, H, F, E);
  a.tile_off = static_cast<const int*>(workspace);
  if (bm > 0)
    if (int rc = swiglu_tiles(offsets, E, bm, workspace, s)) return rc;
  if (int rc = bm == 256   ? launch_tile<256, true>("k_mx_tile_fwd1", s, a, E, R)
               : bm == 128 ? launch_tile<128, true>("k_mx_tile_fwd1", s, a, E, R)
               : bm == 64  ? launch_tile<64, true>("k_mx_tile_fwd1", s, a, E, R)
                           : launch_small<true>("k_mx_small_fwd1", s, a, E, R))
    return rc;
  MxArgs b{};
  b.tile_off = a.tile_off;
  b.offsets = offsets;
  b.A = act;
  b.B = static_cast<const uint8_t*>(wd_q);
  b.S = static_cast<const uint8_t*>(sd);
  b.C = static_cast<uint16_t*>(y);
  b.K = (int)F;
  b.N = (int)H;
  b.npart = mx_parts(bm, R, E, H);
  if (b.npart > 0)
    b.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + moe_swiglu_workspace(E) + al256x((size_t)R * F * 2));
  return bm == 256   ? launch_tile<256, false>("k_mx_tile_fwd2", s, b, E, R)
         : bm == 128 ? launch_tile<128, false>("k_mx_tile_fwd2", s, b, E, R)
         : bm == 64  ? launch_tile<64, false>("k_mx_tile_fwd2", s, b, E, R)
                     : launch_small<false>("k_mx_small_fwd2", s, b, E, R);
}

// ---- backward to the rows ----

namespace moe {
namespace {
struct BkArgs {
  const uint16_t* A;   // dy [R][K] / dh [R][K]
  const uint8_t* B;    // weights [E][Ks][N / 2]: the reduction runs down their rows, their blocks lie along the columns
  const uint8_t* B2;   // ... and those of the reduction's rows from Ks on (up weights)
  const uint8_t* S;    // scales [E][Ks][N / 32]
  const uint8_t* S2;
  uint16_t* C;         // dh [R][2N] / dxp [R][N]
  const uint16_t* X;   // hgu [R][2N] (product with Wd)
  const int* offsets;  // [E+1]
  const int* tile_off; // [E+1] row-tile prefix
  int K;               // reduction length: Ks or 2 Ks
  int Ks;
  int N;               // output columns
  int Tn;              // column tiles
  int E;
  float* part;         // partial tiles of a split last round (null: no split) ...
  int npart;           // ... and how many of them an XCD has room for
};

constexpr int kBkCols = 256;  // columns of a tile

// NF consecutive columns of a row of bf16.
template <int NF>
struct __attribute__((aligned(NF * 2))) BkCols {
  uint32_t d[NF / 2];
};
// They leave: dxp as they are; dh = [da u silu'(g) | da silu(g)] from fp32 da and the pre-activations.
template <bool DACT, int NF>
__device__ __forceinline__ void bk_store(const BkArgs& g, int64_t row, int col, const float (&v)[NF]) {
  if constexpr (DACT) {
    const uint16_t* const pre = g.X + row * 2 * (int64_t)g.N + col;
    const BkCols<NF> gv = *reinterpret_cast<const BkCols<NF>*>(pre), uv = *reinterpret_cast<const BkCols<NF>*>(pre + g.N);
    BkCols<NF> dg, du;
#pragma unroll
    for (int d = 0; d < NF / 2; ++d) {
      float o[2], p[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = __uint_as_float(h ? gv.d[d] & 0xffff0000u : gv.d[d] << 16);
        const float u = __uint_as_float(h ? uv.d[d] & 0xffff0000u : uv.d[d] << 16);
        const float sg = sig_mx(x), t = v[2 * d + h] * sg;
        o[h] = t * u * (1.f + x * (1.f - sg));
        p[h] = t * x;
      }
      dg.d[d] = pack2bf(o[0], o[1]);
      du.d[d] = pack2bf(p[0], p[1]);
    }
    const int64_t at = row * 2 * (int64_t)g.N + col;
    *reinterpret_cast<BkCols<NF>*>(g.C + at) = dg;
    *reinterpret_cast<BkCols<NF>*>(g.C + at + g.N) = du;
  } else {
    BkCols<NF> o;
#pragma unroll
    for (int d = 0; d < NF / 2; ++d) o.d[d] = pack2bf(v[2 * d], v[2 * d + 1]);
    *reinterpret_cast<BkCols<NF>*>(g.C + row * g.N + col) = o;
  }
}

// Where a product's tile L lies.
struct BkTile {
  int e, nt, mbase, mlen;
};
template <int BM>
__device__ __forceinline__ BkTile bk_tile(const BkArgs& g, int L, int lane) {
  MxArgs m{};
  m.E = g.E;
  m.Tn = g.Tn;
  m.tile_off = g.tile_off;
  BkTile t;
  t.e = mx_expert(m, L, lane);
  const int cnt = g.tile_off[t.e + 1] - g.tile_off[t.e], local = L - g.tile_off[t.e] * g.Tn;
  t.nt = local / cnt;
  t.mbase = g.offsets[t.e] + (local - t.nt * cnt) * BM;
  t.mlen = min(BM, g.offsets[t.e + 1] - t.mbase);
  return t;
}
// The backward's products reduce down the weights' rows, across their blocks: every reduction row of a block has a scale of its
// own, and the matrix instruction wants pairs of reduction rows in a word.  So a lane loads NF consecutive columns of eight rows
// (a scale a row), dequantizes them along the columns, two a instruction, and turns the words of two rows over with one v_perm
// a word: a vector instruction a weight, twice the forward's, and no pass through LDS.  Column NF i + j of the wave's goes to
// fragment j, lane i, which leaves each lane NF consecutive columns of the result: fp32 da meets the pre-activations in
// registers, and rows leave in whole segments.  The rows go through LDS in 64-wide slices, as in k_mx_tile: fetched by the lanes
// that use them they are 64 cache accesses a load, and those bounded the products (5.4 ms for dxp below).
//
// What bounds them: with 256 rows no one part of the loop (one wave a SIMD, MFMA busy 62% at 1.77 GHz).  In a copy that leaves a
// part out at a time dxp takes, of 3.10 ms: without the conversions 2.79, the weights' loads 2.74, the rows' refills of LDS
// 2.60, the scales 3.00, all four 2.10 (each a little flattered, as constant operands draw less power); dact, of 1.95 ms:
// 1.81, 1.65, 1.68, 1.79 and 1.16, with its epilogue's 1.9 GB, which two blocks a CU run under each other's loops, inside.
// 16384 rows, E 8, H 4096, F 14336: dact 1.95-2.2 ms, dxp 3.1-3.35 ms (1.92 TFLOP and 3.85: 920-985 and 1150-1240 TFLOP/s);
// the products on bf16 weights 2.01 and 3.35.

// A form: a wave has 32 TF rows by 32 NF columns, a block's four waves lie WT on the rows, WF on the columns and KS along the
// reduction.
template <int TF_, int NF_, int WT_, int WF_, int KS_>
struct BkForm {
  static constexpr int TF = TF_, NF = NF_, WT = WT_, WF = WF_, KS = KS_, BM = 32 * TF_ * WT_;
  static constexpr int BLOCKS = TF * NF > 8 ? 1 : 2;  // of a CU
  static_assert(WT * WF * KS == 4 && WF * NF == 8);
};
// The split of an XCD's last round.  With KS waves along the reduction a block's slices pass KS times as fast, and its tile is
// as much smaller.
template <class Form>
__device__ __forceinline__ MxSplit bk_split(const BkArgs& g, int n) {
  constexpr int KS = Form::KS;
  return mx_split(n, (g.K / 32 + 2 * KS - 1) / (2 * KS), g.npart, 32 * Form::BLOCKS, 2, 16 / KS);
}

template <class Form, bool DACT>
__global__ __launch_bounds__(256, Form::BLOCKS) void k_mx_back(BkArgs g) {
  constexpr int TF = Form::TF, NF = Form::NF, WT = Form::WT, WF = Form::WF, KS = Form::KS, BM = Form::BM;
  constexpr int NP = BM / (8 * WT * WF);  // 16-byte pieces of a thread's share of a slice of the rows
  constexpr int SL = TF * NF;     // MFMAs of a 16-wide step
  constexpr int SLICE = BM * 128; // LDS bytes of a 64-wide slice of the rows
  constexpr int PB = NF;          // blocks of a wave's columns
  constexpr int SR = 36;          // a block's scales of 32 reduction rows (padded: blocks lie in distinct banks)
  constexpr int SP = PB * SR;     // ... and a wave's
  constexpr int SMEM = std::max(2 * KS * SLICE, 4 * (KS - 1) * 8192);
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];
  __shared__ __attribute__((aligned(16))) float scl[4 * SP];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i32 = lane & 31, h = lane >> 5;

  const int total = g.tile_off[g.E] * g.Tn;
  const int chunk = (total + 7) >> 3, xcd = (int)(blockIdx.x & 7);
  int slot = (int)(blockIdx.x >> 3);
  int b0 = 0, b1 = g.K / 32;  // the block's units of 32 of the reduction
  float* part_out = nullptr;
  {
    const MxSplit sp = bk_split<Form>(g, min(chunk, total - xcd * chunk));
    if (sp.parts > 1 && slot >= sp.full) {
      const int j = slot - sp.full, t = j / sp.parts, p = j - t * sp.parts;
      if (t >= sp.rest) return;
      slot = sp.full + t;
      const int units = b1;
      b0 = units * p / sp.parts;
      b1 = units * (p + 1) / sp.parts;
      part_out = g.part + (int64_t)(xcd * g.npart + j) * (BM * kBkCols);
    }
  }
  const int L = xcd * chunk + slot;
  if (slot >= chunk || L >= total) return;
  const BkTile tl = bk_tile<BM>(g, L, lane);
  const int gw = wv % (WT * WF), tw = gw % WT, fw = gw / WT, kw = wv / (WT * WF);
  const int n0 = tl.nt * kBkCols + fw * (32 * NF);
  const int w0 = __builtin_amdgcn_readfirstlane(b0 + (b1 - b0) * kw / KS);
  const int w1 = __builtin_amdgcn_readfirstlane(b0 + (b1 - b0) * (kw + 1) / KS);
  // Slices of 64: an odd number of units has a unit of zeros in front.  The KS shares run as many slices as the longest.
  const int lead = (w1 - w0) & 1, ns = (w1 - w0 + lead) >> 1;
  const int rounds = ((b1 - b0 + KS - 1) / KS + 1) >> 1;
  // unit 2 i + half of the share; behind the share's last one (and in front of its first) any unit there is
  const int units = g.K / 32;
  auto unit = [&](int i, int half) { return max(min(w0 - lead + 2 * i + half, min(w1, units) - 1), 0); };
  auto live = [&](int i, int half) { return i < ns && (half == 1 || lead == 0 || i > 0); };

  const int N = g.N, nbk = N / 32, rowb = N / 2;
  // rows: piece p of a slice is rows 8 (NP gw + p) + lane / 8 of the share's; a row's eight 16-byte chunks are swizzled so
  // that the 16 rows a fragment read touches at once lie in distinct banks
  const uint8_t* const xbase = reinterpret_cast<const uint8_t*>(g.A + (int64_t)tl.mbase * g.K);
  uint8_t* const xs_lds = smem + kw * (2 * SLICE);
  uint32_t xo[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int row = 8 * (NP * gw + p) + (lane >> 3);
    xo[p] = (uint32_t)min(row, tl.mlen - 1) * (uint32_t)g.K * 2u;
  }
  const buf_rsrc_t xr = buf_rsrc(xbase, -1);
  u32x4 xs[NP];
  auto load_x = [&](int i, int p) {
    const int row = 8 * (NP * gw + p) + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
    // (behind the share's last slice any two units there are: they are written as zeros)
    const int at = max(min(w0 - lead + 2 * i, units - 2), 0);
    xs[p] = __builtin_bit_cast(
        u32x4, __builtin_amdgcn_raw_buffer_load_b128(xr, (int)(xo[p] + (uint32_t)(units > 1 ? c : c & 3) * 16u), at * 64, 0));
  };
  auto load_x_first = [&](int p) {
    const int row = 8 * (NP * gw + p) + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
    xs[p] = *reinterpret_cast<const u32x4*>(xbase + (int64_t)unit(0, c >> 2) * 64 + xo[p] + (c & 3) * 16);
    if (!live(0, c >> 2)) xs[p] = u32x4{0u, 0u, 0u, 0u};
  };
  auto write_x = [&](int i, int p, bool first) {
    const uint32_t keep = KS == 1 || first || i < ns ? ~0u : 0u;  // (KS == 1: no one reads what is behind the last slice)
    __asm__ volatile("" ::: "memory");
    *reinterpret_cast<u32x4*>(xs_lds + (i & 1) * SLICE + (NP * gw + p) * 1024 + lane * 16) = xs[p] & keep;
    __asm__ volatile("" ::: "memory");
  };
  auto frag = [&](int i, int s, int t) {
    const int row = tw * (32 * TF) + t * 32 + i32;
    return *reinterpret_cast<const bf16x8*>(xs_lds + (i & 1) * SLICE + row * 128 + (((2 * s + h) ^ ((row >> 1) & 7)) << 4));
  };

  // weights: lane 32 h + i has columns NF i + [0, NF) of rows 16 s + 8 h + [0, 8); columns past N repeat the last.  Buffer
  // loads: a lane offset that stays, and a uniform one that moves.
  const int64_t eb = (int64_t)tl.e * g.Ks;
  const uint32_t bo = (uint32_t)(8 * h) * (uint32_t)rowb + (uint32_t)min(n0 / NF + i32, N / NF - 1) * (NF / 2u);
  // scales: lane 32 h + i loads blocks PB / 2 h + [0, PB / 2) of row i, as a word that ends inside the array
  const uint32_t so = (uint32_t)i32 * (uint32_t)nbk + (uint32_t)(n0 / 32 + PB / 2 * h);
  const uint32_t slim = (uint32_t)min((int64_t)INT32_MAX, (int64_t)(g.E - tl.e) * g.Ks * nbk - 4);
  struct __attribute__((packed)) Bytes4 { uint32_t v; };
  typedef f32x4 __attribute__((may_alias)) f32x4a;
  uint32_t w[4][8];         // [step][row]
  uint32_t sw[2], sh[2];    // a unit's word, and how many of its bits are other blocks'
  float* const sl = scl + wv * SP;
  auto second = [&](int u) { return u * 32 >= g.Ks; };
  const uint8_t* const wb = g.B + eb * rowb;
  const uint8_t* const wb2 = g.B2 + eb * rowb;
  typedef const __attribute__((address_space(1))) uint8_t gbyte;
  gbyte* sb = (gbyte*)(g.S + eb * nbk);
  gbyte* sb2 = (gbyte*)(g.S2 + eb * nbk);
  __asm__("" : "+s"(sb), "+s"(sb2));  // in registers: not loaded again in the loop
  auto wsrc = [&](int u) {
    return buf_rsrc(second(u) ? wb2 : wb, -1);
  };
  auto woff = [&](int u, int x) { return (u * 32 + 16 * x - (second(u) ? g.Ks : 0)) * rowb; };
  auto load_w = [&](int s, int j, buf_rsrc_t b, int off) {
    if constexpr (NF == 8) w[s][j] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(b, (int)bo, off + j * rowb, 0);
    else w[s][j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(b, (int)bo, off + j * rowb, 0);
  };
  auto load_s = [&](int half, int u) {
    const uint32_t at = (uint32_t)(u * 32 - (second(u) ? g.Ks : 0)) * (uint32_t)nbk + so, in = min(at, slim);
    sw[half] = ((const __attribute__((address_space(1))) Bytes4*)((second(u) ? sb2 : sb) + in))->v;
    sh[half] = min((at - in) * 8u, 31u);
  };
  auto put_s = [&](int i, int half) {
    const uint32_t v = live(i, half) ? sw[half] >> sh[half] : 0x7f7f7f7fu;
    __asm__ volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < PB / 2; ++j) sl[(PB / 2 * h + j) * SR + i32] = __uint_as_float(((v >> (8 * j)) & 0xffu) << 23);
    __asm__ volatile("" ::: "memory");
  };
  f32x4 sc[2][2];  // the scales of the rows of a unit's two steps
  auto get_s = [&](int x) {
    const float* const at = sl + i32 * NF / 32 * SR + 16 * x + 8 * h;
    sc[x][0] = *reinterpret_cast<const f32x4a*>(at);
    sc[x][1] = *reinterpret_cast<const f32x4a*>(at + 4);
    __asm__ volatile("" ::: "memory");
  };

  f32x16 acc[TF][NF];
#pragma unroll
  for (int t = 0; t < TF; ++t)
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[t][j][v] = 0.f;
  u32x4 f0[NF], f1[NF];  // fragment j: column NF i + j of the wave's, 16 reduction rows
  bf16x8 x0[TF], x1[TF];

  // Piece c of a step's conversion: rows 2 t, 2 t + 1, columns 2 p, 2 p + 1 become words t of fragments 2 p, 2 p + 1.
  constexpr int P = NF / 2, PIECES = 4 * P;
  uint32_t cx[2], cy[2];
  auto conv_a = [&](auto c_c, const uint32_t(&r)[8], const f32x4(&s)[2]) {
    constexpr int c = decltype(c_c)::value, t = c / P, p = c % P;
    cx[c & 1] = mx_pair<p>(r[2 * t], s[t / 2][t % 2 * 2]);
    cy[c & 1] = mx_pair<p>(r[2 * t + 1], s[t / 2][t % 2 * 2 + 1]);
  };
  auto conv_b = [&](auto c_c, u32x4(&f)[NF]) {
    constexpr int c = decltype(c_c)::value, t = c / P, p = c % P;
    f[2 * p][t] = __builtin_amdgcn_perm(cy[c & 1], cx[c & 1], 0x05040100u);
    f[2 * p + 1][t] = __builtin_amdgcn_perm(cy[c & 1], cx[c & 1], 0x07060302u);
  };

  // Step s of slice i: TF NF MFMAs, and between them the next step's row fragments, its conversion (a piece's transposition a
  // slot behind its dequantization), each pair of its rows followed by the loads of the same rows of the next slice, and in
  // the first three the slice's share of refill pieces (slice i + 1 to LDS, i + 2 from memory).
  auto step = [&](auto s_c, const bf16x8(&cx_)[TF], const u32x4(&cf)[NF], bf16x8(&nx)[TF], u32x4(&nf)[NF], int i) {
    constexpr int s = decltype(s_c)::value, sn = (s + 1) % 4, x = s & 1, half = s >> 1;
    const int in = s == 3 ? i + 1 : i;                 // the next step's slice
    const int un = unit(in + 1, sn >> 1);
    const buf_rsrc_t bn = wsrc(un);
    const int wn = woff(un, sn & 1);
    constexpr int P0 = s == 3 ? 0 : (s * NP + 2) / 3, P1 = s == 3 ? 0 : ((s + 1) * NP + 2) / 3;
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (([&] {
         constexpr int t = I / NF, j = I % NF, EVERY = SL / PIECES, c = I / EVERY;
         acc[t][j] = mfma32x32x16(cx_[t], __builtin_bit_cast(bf16x8, cf[j]), acc[t][j]);
         __builtin_amdgcn_sched_barrier(0);
         if constexpr (I < TF) nx[I] = frag(in, sn, I);
         if constexpr (I % EVERY == 0) {
           conv_a(std::integral_constant<int, c>{}, w[sn], sc[1 - x]);
           if constexpr (c > 0) conv_b(std::integral_constant<int, c - 1>{}, nf);
           if constexpr (c % P == P - 1) {
             load_w(sn, 2 * (c / P), bn, wn);
             load_w(sn, 2 * (c / P) + 1, bn, wn);
           }
         }
         if constexpr (x == 0 && I == SL * 5 / 16) put_s(half == 0 ? i : i + 1, 1 - half);
         if constexpr (x == 0 && I == SL * 7 / 16) load_s(1 - half, unit(half == 0 ? i + 1 : i + 2, 1 - half));
         if constexpr (I == SL * 11 / 16) get_s(x);
         constexpr int PE = SL / 8, p = P0 + (I - 5 * PE) / PE;
         if constexpr (I >= 5 * PE && I % PE == 0 && p < P1) {
           write_x(i + 1, p, false);
           load_x(i + 2, p);
         }
         __builtin_amdgcn_sched_barrier(0);
       }()), ...);
    }(std::make_integer_sequence<int, SL>{});
    conv_b(std::integral_constant<int, PIECES - 1>{}, nf);
    __builtin_amdgcn_sched_barrier(0);
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  using S3 = std::integral_constant<int, 3>;
#pragma unroll
  for (int p = 0; p < NP; ++p) load_x_first(p);
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) load_w(s, j, wsrc(unit(0, s >> 1)), woff(unit(0, s >> 1), s & 1));
  load_s(0, unit(0, 0));
  load_s(1, unit(0, 1));
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    write_x(0, p, true);
    load_x(1, p);
  }
  put_s(0, 0);
  get_s(0);
  get_s(1);
  load_s(0, unit(1, 0));
  __syncthreads();
#pragma unroll
  for (int t = 0; t < TF; ++t) x0[t] = frag(0, 0, t);
  [&]<int... I>(std::integer_sequence<int, I...>) {
    ((conv_a(std::integral_constant<int, I>{}, w[0], sc[0]), conv_b(std::integral_constant<int, I>{}, f0)), ...);
  }(std::make_integer_sequence<int, PIECES>{});
#pragma unroll
  for (int j = 0; j < 8; ++j) load_w(0, j, wsrc(unit(1, 0)), woff(unit(1, 0), 0));
  // (a second use of the loaded words, or the loop would carry them as 16 bits, widen them at its top and wait for them there)
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) __asm__ volatile("" ::"v"(w[s][j]));
  const int col = n0 + i32 * NF;
  for (int i = 0; i < rounds; ++i) {
    step(S0{}, x0, f0, x1, f1, i);
    step(S1{}, x1, f1, x0, f0, i);
    step(S2{}, x0, f0, x1, f1, i);
    lds_sync();  // every wave's pieces of slice i + 1 are written and its reads of slice i done
    step(S3{}, x1, f1, x0, f0, i);
  }
  __syncthreads();

  // acc[t][j][v]: row 32 t + (v & 3) + 8 (v >> 2) + 4 h, column NF i + j: a lane has NF consecutive columns of a row, and
  // 32 lanes a whole segment of it.  c = 16 t + v.
  struct __attribute__((aligned(16))) Cols { float v[NF]; };
  auto cols = [&](int c) {
    Cols o;
#pragma unroll
    for (int j = 0; j < NF; ++j) o.v[j] = acc[c / 16][j][c % 16];
    return o;
  };
  auto partial = [&](int c, const Cols& o) {
    reinterpret_cast<Cols*>(part_out)[((tw * WF + fw) * (16 * TF) + c) * 64 + lane] = o;
  };
  auto leave = [&](int c, const Cols& o) {
    const int r = tw * (32 * TF) + (c >> 4) * 32 + (c & 3) + ((c >> 2) & 3) * 8 + 4 * h;
    if (r < tl.mlen && col < N) bk_store<DACT, NF>(g, tl.mbase + r, col, o.v);
  };
  if constexpr (KS == 1) {
    if (part_out != nullptr) {
#pragma unroll
      for (int c = 0; c < 16 * TF; ++c) partial(c, cols(c));
      return;
    }
#pragma unroll
    for (int t = 0; t < TF; ++t) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int r = tw * (32 * TF) + t * 32 + (v & 3) + (v >> 2) * 8 + 4 * h;
        if (r < tl.mlen && col < N) bk_store<DACT, NF>(g, tl.mbase + r, col, cols(16 * t + v).v);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    // The KS waves of the same rows and columns meet in LDS, each for a KS-th of the c, in rounds of 32 values a lane.
    constexpr int PC = 16 * TF / KS, Q = 32 / NF;
    Cols* const rd = reinterpret_cast<Cols*>(smem) + (wv % (WT * WF)) * (KS * (KS - 1) * Q * 64) + lane;
#pragma unroll
    for (int q0 = 0; q0 < PC; q0 += Q) {
      if (q0 > 0) __syncthreads();
#pragma unroll
      for (int o = 0; o < KS; ++o) {  // owner
        if (o == kw) continue;
#pragma unroll
        for (int q = 0; q < Q; ++q) rd[((o * (KS - 1) + (kw < o ? kw : kw - 1)) * Q + q) * 64] = cols(o * PC + q0 + q);
      }
      __syncthreads();
#pragma unroll
      for (int o = 0; o < KS; ++o) {
        if (o != kw) continue;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int c = o * PC + q0 + q;
          Cols sum;
#pragma unroll
          for (int x = 0; x < KS; ++x) {  // in the order of the reduction
            const Cols y = x == o ? cols(c) : rd[((o * (KS - 1) + (x < o ? x : x - 1)) * Q + q) * 64];
#pragma unroll
            for (int j = 0; j < NF; ++j) sum.v[j] = x == 0 ? y.v[j] : sum.v[j] + y.v[j];
          }
          if (part_out != nullptr) partial(c, sum);
          else leave(c, sum);
        }
      }
    }
  }
}

// The split tiles' sums: blockIdx.x = (XCD, split tile), blockIdx.y an eighth of the tile's (wave, c) pairs.
template <class Form, bool DACT>
__global__ __launch_bounds__(256) void k_mx_back_reduce(BkArgs g) {
  constexpr int NF = Form::NF, BM = Form::BM, PAIRS = BM * kBkCols / (64 * NF), WC = 16 * Form::TF;
  const int tid = threadIdx.x, lane = tid & 63;
  constexpr int RES = 32 * Form::BLOCKS;
  const int xcd = (int)blockIdx.x / RES, t = (int)blockIdx.x % RES;
  const int total = g.tile_off[g.E] * g.Tn, chunk = (total + 7) >> 3;
  const MxSplit sp = bk_split<Form>(g, min(chunk, total - xcd * chunk));
  if (sp.parts == 1 || t >= sp.rest) return;
  const BkTile tl = bk_tile<BM>(g, xcd * chunk + sp.full + t, lane);
  struct __attribute__((aligned(16))) Cols { float v[NF]; };
  const Cols* const src = reinterpret_cast<const Cols*>(g.part + (int64_t)(xcd * g.npart + t * sp.parts) * (BM * kBkCols));
  for (int wc = (int)blockIdx.y * (PAIRS / 8) + (tid >> 6); wc < (int)(blockIdx.y + 1) * (PAIRS / 8); wc += 4) {
    const int c = wc % WC, wave = wc / WC, tw = wave / Form::WF, fw = wave % Form::WF;
    const int r = tw * (2 * WC) + (c >> 4) * 32 + (c & 3) + ((c >> 2) & 3) * 8 + 4 * (lane >> 5);
    const int col = tl.nt * kBkCols + fw * (32 * NF) + (lane & 31) * NF;
    if (r >= tl.mlen || col >= g.N) continue;
    Cols sum = src[wc * 64 + lane];
    for (int p = 1; p < sp.parts; ++p) {
      const Cols y = src[(int64_t)p * (PAIRS * 64) + wc * 64 + lane];
#pragma unroll
      for (int j = 0; j < NF; ++j) sum.v[j] += y.v[j];
    }
    bk_store<DACT, NF>(g, tl.mbase + r, col, sum.v);
  }
}

// Rows of a product's tile, by the rows an expert has on average and by the tiles there are (N: its output columns).  Both
// products, us, by rows an expert (routed; 64 rows | 128 | 256 for dxp alone):
//   E 8,   H 4096, F 14336   16: 252 | 366 | 524   64: 399 | 393 | 542   256: 920 | 942 | 993   2048: 7323 | 5742 | 5380
//   E 128, H 2048, F 768     16: 161 | 175 | 255   64: 244 | 196 | 274   256: 633 | 454 | 502   2048: 4358 | 2787 | 2715
//   E 8,   H 1024, F 4096    16: 57 | 69 | 83      64: 68 | 83 | 103     256: 137 | 116 | 126   2048: 825 | 533 | 541
// 256 rows for the product with Wd as well cost 4% at 2048 rows: one block a CU leaves nothing to run under its epilogue.
int bk_rows(bool dact, int64_t R, int64_t N, int64_t F, int64_t E) {
  if (R < 64 * E || std::max(R / 128, E) * ((F + 255) / 256) < 256) return 64;
  return !dact && R >= 1024 * E && R / 256 * ((N + 255) / 256) >= 512 ? 256 : 128;
}
int bk_parts(int bm, int64_t R, int64_t E, int64_t N) {
  const int64_t tiles = ((R + bm - 1) / bm + E) * ((N + kBkCols - 1) / kBkCols);
  return (int)std::min<int64_t>(bm == 128 ? 128 : 64, 8 * ((tiles + 7) / 8));
}
size_t bk_part_bytes(int bm, int64_t R, int64_t E, int64_t N) {
  return (size_t)8 * bk_parts(bm, R, E, N) * bm * kBkCols * sizeof(float);
}

template <class Form, bool DACT>
int launch_back_as(const char* name, hipStream_t s, BkArgs a, int64_t E, int64_t R) {
  a.E = (int)E;
  a.Tn = cdiv(a.N, kBkCols);
  const int64_t blocks = ((R + Form::BM - 1) / Form::BM + E) * a.Tn;
  if (blocks > INT32_MAX / 2) return fail_arg("%s: too many tiles", name);
  MOE_LAUNCH(name, (k_mx_back<Form, DACT>), dim3((unsigned)((blocks + 7) / 8 * 8 + 8 * a.npart)), dim3(256), 0, s, a);
  MOE_LAUNCH("k_mx_back_reduce", (k_mx_back_reduce<Form, DACT>), dim3(8 * 32 * Form::BLOCKS, 8), dim3(256), 0, s, a);
  return check_launch(name);
}
template <bool DACT>
int launch_back(const char* name, hipStream_t s, const BkArgs& a, int64_t E, int64_t R, int bm) {
  if constexpr (!DACT) {
    if (bm == 256) return launch_back_as<BkForm<4, 4, 2, 2, 1>, DACT>(name, s, a, E, R);
  }
  return bm == 128 ? launch_back_as<BkForm<2, 4, 2, 2, 1>, DACT>(name, s, a, E, R)
                   : launch_back_as<BkForm<2, 8, 1, 1, 4>, DACT>(name, s, a, E, R);
}
}  // namespace
}  // namespace moe

extern "C" size_t moe_swiglu_bwd_mxfp4_workspace(int64_t R, int64_t H, int64_t F, int64_t E) {
  if (R <= 0 || H <= 0 || F <= 0 || E <= 0) return 0;
  return moe_swiglu_workspace(E) + al256x((size_t)R * F * 4) +
         std::max(bk_part_bytes(bk_rows(true, R, F, F, E), R, E, F), bk_part_bytes(bk_rows(false, R, H, F, E), R, E, H));
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
  const int da = bk_rows(true, R, F, F, E), dx = bk_rows(false, R, H, F, E);
  uint16_t* const dh = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + moe_swiglu_workspace(E));
  if (int rc = swiglu_tiles(offsets, E, da, workspace, s)) return rc;
  BkArgs a{};
  a.offsets = offsets;
  a.tile_off = static_cast<const int*>(workspace);
  a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(dh) + al256x((size_t)R * F * 4));
  BkArgs b = a;
  // dh = epilogue(dy . Wd): Wd's rows are the reduction
  a.A = static_cast<const uint16_t*>(dy);
  a.B = a.B2 = static_cast<const uint8_t*>(wd_q);
  a.S = a.S2 = static_cast<const uint8_t*>(sd);
  a.C = dh;
  a.X = static_cast<const uint16_t*>(hgu);
  a.K = a.Ks = (int)H;
  a.N = (int)F;
  a.npart = bk_parts(da, R, E, F);
  if (int rc = launch_back<true>("k_mx_back_dact", s, a, E, R, da)) return rc;
  // dxp = dh . [Wg ; Wu]
  if (dx != da)
    if (int rc = swiglu_tiles(offsets, E, dx, workspace, s)) return rc;
  b.A = dh;
  b.B = static_cast<const uint8_t*>(wg_q);
  b.S = static_cast<const uint8_t*>(sg);
  b.B2 = static_cast<const uint8_t*>(wu_q);
  b.S2 = static_cast<const uint8_t*>(su);
  b.C = static_cast<uint16_t*>(dxp);
  b.K = (int)(2 * F);
  b.Ks = (int)F;
  b.N = (int)H;
  b.npart = bk_parts(dx, R, E, H);
  return launch_back<false>("k_mx_back_dxp", s, b, E, R, dx);
}

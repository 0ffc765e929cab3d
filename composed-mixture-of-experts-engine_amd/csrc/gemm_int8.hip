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
#include <utility>

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

// ---- many rows ----
typedef __attribute__((address_space(1))) const u32x4 g_u32x4;
__device__ __forceinline__ u32x4 ldg16(const uint8_t* p) {
  return *reinterpret_cast<g_u32x4*>(reinterpret_cast<uintptr_t>(p));
}
struct __attribute__((packed, aligned(4))) Scale4 { float v[4]; };
__device__ __attribute__((aligned(16))) const uint8_t g_i8_zero[16] = {0};

// One tile of BM rows of an expert by BN weight rows (GU: BN / 2 gate rows and the matching up rows, 32 by 32), four waves
// WR x WC of MI x NI fragments of v_mfma_i32_32x32x32_i8.  Both operands go through LDS in slices of 128 bytes of a row (whole
// cache lines), two slices at a time, a row's eight 16-byte chunks swizzled so that the 16 rows a fragment read touches at
// once lie in distinct banks.  While slice kt is computed, each wave writes its share of slice kt + 1 (in registers since the
// slice before) into the free half and loads its share of slice kt + 2 into the same registers, one 16-byte piece a lane at a
// time between the matrix instructions; one barrier a slice.
template <bool GU, typename OT, int WR, int MI, int NI>
__global__ __launch_bounds__(256, MI * NI <= 4 ? 2 : 1) void k_i8_tile(I8Args g) {
  constexpr int WC = 4 / WR;
  constexpr int BM = WR * MI * 32, BN = WC * NI * 32;
  constexpr int SA = BM * 128, SB = BN * 128;          // LDS bytes of a slice of either operand
  constexpr int QA = BM / 32, QB = BN / 32, NP = QA + QB;  // 16-byte pieces of a wave's share of a slice
  constexpr int CW = GU ? BN / 2 : BN;                 // output columns of the tile
  constexpr int WCOLS = CW / WC;                       // ... and of a wave
  constexpr int CP = GU ? (WCOLS + 8) / 2 : WCOLS + 4; // words a row of a wave's output strip of 32 rows
  constexpr int SMEM = std::max(2 * (SA + SB), 4 * 32 * CP * 4);
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm0 = wv / WC * (MI * 32), wn0 = wv % WC * (NI * 32);
  const int i32 = lane & 31, h = lane >> 5;

  // XCD-contiguous logical order over a 1-D grid sized for the most tiles any routing can produce: the tiles that there are,
  // split into 8 contiguous ranges (blockIdx mod 8)
  auto row_tiles = [&](int e) {
    return e < g.E ? (int)((seg(g, e + 1) - seg(g, e) + BM - 1) / BM) : 0;
  };
  int sum = 0;
  for (int e0 = 0; e0 < g.E; e0 += 64) sum += max(row_tiles(e0 + lane), 0);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  const int total = __builtin_amdgcn_readfirstlane(sum) * g.Tn;
  const int chunk = (total + 7) >> 3, slot = (int)(blockIdx.x >> 3), L = (int)(blockIdx.x & 7) * chunk + slot;
  if (slot >= chunk || L >= total) return;
  int e = 0, before = 0, cnt = 0;  // row tiles of the experts before e, and of e
  for (int e0 = 0;; e0 += 64) {
    const int c = max(row_tiles(e0 + lane), 0);
    int upto = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      upto += lane >= o ? v : 0;
    }
    const unsigned long long past = __ballot(L < (before + upto) * g.Tn);
    if (past) {
      const int l = __builtin_ctzll(past);
      e = e0 + l;
      cnt = __shfl(c, l);
      before += __shfl(upto, l) - cnt;
      break;
    }
    before += __shfl(upto, 63);
  }
  e = __builtin_amdgcn_readfirstlane(e);
  cnt = __builtin_amdgcn_readfirstlane(cnt);
  const int local = L - __builtin_amdgcn_readfirstlane(before) * g.Tn;
  constexpr int GM = 8;
  const int grp = local / (GM * g.Tn), rest = local - grp * GM * g.Tn, gm = min(cnt - grp * GM, GM);
  const int nt = rest / gm, mt = grp * GM + rest - nt * gm;
  const int64_t mbase = seg(g, e) + (int64_t)mt * BM;
  const int mlen = (int)min(seg(g, e + 1) - mbase, (int64_t)BM);
  const int n0 = nt * CW, K = g.K, nk = (K + 127) / 128;

  // piece p of a wave's share: instruction j fills rows 8 j + lane / 8 of its operand's tile, slot lane % 8 of the row
  const uint8_t* const b_base[2] = {g.B + (int64_t)e * g.N * K, GU ? g.B2 + (int64_t)e * g.N * K : g.B + (int64_t)e * g.N * K};
  const uint8_t* a_src[QA];
  uint32_t b_off[QB];
  auto chunk_of = [&](int j) { return (lane & 7) ^ ((4 * j + (lane >> 4)) & 7); };
#pragma unroll
  for (int q = 0; q < QA; ++q) {
    const int j = QA * wv + q;
    a_src[q] = g.A + source_row(g, mbase + min(8 * j + (lane >> 3), mlen - 1)) * K + chunk_of(j) * 16;
  }
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int j = QB * wv + q, i = 8 * j + (lane >> 3);
    const int n = GU ? n0 + (i >> 6) * 32 + (i & 31) : n0 + i;
    b_off[q] = (uint32_t)min(n, g.N - 1) * (uint32_t)K + chunk_of(j) * 16;
  }
  u32x4 st[NP];
  // piece p of slice kt; past the row's end A is zeros and B anything
  auto gload = [&](int kt, int p, bool full) {
    if (p < QA) {
      const uint8_t* s = a_src[p] + kt * 128;
      if (!full) s = kt * 128 + chunk_of(QA * wv + p) * 16 < K ? s : g_i8_zero;
      st[p] = ldg16(s);
    } else {
      const int q = p - QA, j = QB * wv + q;
      const uint8_t* const base = b_base[GU ? (8 * j >> 5) & 1 : 0];
      uint32_t o = b_off[q];
      if (full) {
        st[p] = ldg16(base + (uint32_t)kt * 128u + o);
      } else {
        const int k = kt * 128 + chunk_of(j) * 16;
        st[p] = ldg16(base + (o - chunk_of(j) * 16) + (k < K ? (uint32_t)k : 0u));
      }
    }
  };
  auto half = [&](int kt) { return smem + (kt & 1) * (SA + SB); };
  auto lwrite = [&](int kt, int p) {
    uint8_t* const d = half(kt) + (p < QA ? (QA * wv + p) * 1024 : SA + (QB * wv + p - QA) * 1024);
    __asm__ volatile("" ::: "memory");
    *reinterpret_cast<u32x4*>(d + lane * 16) = st[p];
    __asm__ volatile("" ::: "memory");
  };
  auto frag = [&](const uint8_t* t, int row, int ks) {
    return *reinterpret_cast<const i32x4*>(t + row * 128 + (((2 * ks + h) ^ ((row >> 1) & 7)) << 4));
  };
  auto read_frag = [&](int kt, int ks, int f, i32x4(&fa)[MI], i32x4(&fb)[NI]) {
    if (f < MI) fa[f] = frag(half(kt), wm0 + f * 32 + i32, ks);
    else fb[f - MI] = frag(half(kt) + SA, wn0 + (f - MI) * 32 + i32, ks);
  };

  i32x16 acc[MI][NI];
#pragma unroll
  for (int mi = 0; mi < MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[mi][ni][j] = 0;

  // One 32-wide quarter of slice kt: MI NI matrix instructions, after each at most a fragment read of the next quarter (the
  // first ones) and a refill piece of [PLO, PHI) (the last ones).  MODE 0: write slice kt + 1, load the whole slice kt + 2;
  // 1: the slice loaded may end inside; 2: write only; 3: neither.
  constexpr int SLOTS = MI * NI;
  auto quarter = [&](auto mode_c, auto plo_c, auto phi_c, const i32x4(&ca)[MI], const i32x4(&cb)[NI], int nkt, int nks,
                     bool read_next, i32x4(&na)[MI], i32x4(&nb)[NI], int kt, bool lfull) {
    constexpr int MODE = decltype(mode_c)::value, PLO = decltype(plo_c)::value, PHI = decltype(phi_c)::value;
    static_assert(PHI - PLO <= SLOTS && MI + NI <= SLOTS);
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (([&] {
         constexpr int mi = I / NI, ni = I % NI;
         acc[mi][ni] = __builtin_amdgcn_mfma_i32_32x32x32_i8(cb[ni], ca[mi], acc[mi][ni], 0, 0, 0);
         __builtin_amdgcn_sched_barrier(0);
         if constexpr (I < MI + NI) {
           if (read_next) read_frag(nkt, nks, I, na, nb);
         }
         constexpr int p = PHI - SLOTS + I;
         if constexpr (MODE < 3 && p >= PLO) {
           lwrite(kt + 1, p);
           if constexpr (MODE == 0) gload(kt + 2, p, true);
           else if constexpr (MODE == 1) gload(kt + 2, p, lfull);
         }
         __builtin_amdgcn_sched_barrier(0);
       }()), ...);
    }(std::make_integer_sequence<int, SLOTS>{});
  };
  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, (NP + 2) / 3>;
  using P2 = std::integral_constant<int, (2 * NP + 2) / 3>;
  using P3 = std::integral_constant<int, NP>;
  using M3 = std::integral_constant<int, 3>;
  i32x4 fa0[MI], fb0[NI], fa1[MI], fb1[NI];
  const int whole = K / 128;  // whole slices
  auto slice = [&](auto mode_c, int kt) {
    const bool lfull = kt + 2 < whole;
    quarter(mode_c, P0{}, P1{}, fa0, fb0, kt, 1, true, fa1, fb1, kt, lfull);
    quarter(mode_c, P1{}, P2{}, fa1, fb1, kt, 2, true, fa0, fb0, kt, lfull);
    quarter(mode_c, P2{}, P3{}, fa0, fb0, kt, 3, true, fa1, fb1, kt, lfull);
    lds_sync();  // this wave's pieces of slice kt + 1 are written and its reads of slice kt done, and every other wave's
    __builtin_amdgcn_sched_barrier(0);
    quarter(M3{}, P3{}, P3{}, fa1, fb1, kt + 1, 0, kt + 1 < nk, fa0, fb0, kt, true);
  };
  for (int p = 0; p < NP; ++p) gload(0, p, 0 < whole);
  for (int p = 0; p < NP; ++p) lwrite(0, p);
  if (nk > 1) {
    for (int p = 0; p < NP; ++p) gload(1, p, 1 < whole);
  }
  __syncthreads();
  for (int f = 0; f < MI + NI; ++f) read_frag(0, 0, f, fa0, fb0);
  int kt = 0;
  for (; kt + 2 < whole; ++kt) slice(std::integral_constant<int, 0>{}, kt);
  for (; kt + 2 < nk; ++kt) slice(std::integral_constant<int, 1>{}, kt);
  if (kt + 1 < nk) slice(std::integral_constant<int, 2>{}, kt++);
  if (kt < nk) slice(M3{}, kt);
  __syncthreads();

  // The matrix instructions take the weights as their M operand, so a lane holds one row of C and, in each four accumulators,
  // four columns in a row: acc[mi][ni][j] = C[wm0 + 32 mi + lane % 32][wn0 + 32 ni + 8 (j / 4) + 4 (lane / 32) + j % 4].  Each
  // wave turns its strips of 32 rows over through LDS of its own, so that rows leave in whole lines.
  uint32_t* const cs = reinterpret_cast<uint32_t*>(smem) + wv * 32 * CP;
  const int c0 = n0 + wv % WC * WCOLS;  // the wave's first column
  const float* const sb = g.sb + (int64_t)e * g.N;
  const float* const sb2 = GU ? g.sb2 + (int64_t)e * g.N : nullptr;
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int r0 = wm0 + mi * 32;  // the strip's first row of the tile
    if (r0 >= mlen) break;
    const float sx = g.sa[source_row(g, mbase + min(r0 + i32, mlen - 1))];
    __asm__ volatile("" ::: "memory");
    if constexpr (GU) {
#pragma unroll
      for (int pr = 0; pr < NI / 2; ++pr)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int c = pr * 32 + v * 8 + h * 4, n = min(c0 + c, g.N - 4);
          const Scale4 sg = *reinterpret_cast<const Scale4*>(sb + n), su = *reinterpret_cast<const Scale4*>(sb2 + n);
          float o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float gv = (float)acc[mi][2 * pr][4 * v + j] * sx * sg.v[j];
            o[j] = gv * sig_i8(gv) * ((float)acc[mi][2 * pr + 1][4 * v + j] * sx * su.v[j]);
          }
          *reinterpret_cast<uint2*>(cs + i32 * CP + c / 2) = uint2{pack2bf(o[0], o[1]), pack2bf(o[2], o[3])};
        }
    } else {
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int c = ni * 32 + v * 8 + h * 4, n = min(c0 + c, g.N - 4);
          const Scale4 s = *reinterpret_cast<const Scale4*>(sb + n);
          f32x4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = (float)acc[mi][ni][4 * v + j] * sx * s.v[j];
          *reinterpret_cast<f32x4*>(cs + i32 * CP + c) = o;
        }
    }
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    constexpr int PER = GU || sizeof(OT) == 2 ? 8 : 4;  // columns of a 16-byte store
    constexpr int LPR = WCOLS / PER;                    // lanes a row
#pragma unroll
    for (int u = 0; u < 32 * LPR / 64; ++u) {
      const int r = u * (64 / LPR) + lane / LPR, c = lane % LPR * PER;
      u32x4 o;
      if constexpr (GU) {
        o = *reinterpret_cast<const u32x4*>(cs + r * CP + c / 2);
      } else if constexpr (sizeof(OT) == 4) {
        o = *reinterpret_cast<const u32x4*>(cs + r * CP + c);
      } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(cs + r * CP + c), hi = *reinterpret_cast<const f32x4*>(cs + r * CP + c + 4);
        o = u32x4{pack2bf(lo[0], lo[1]), pack2bf(lo[2], lo[3]), pack2bf(hi[0], hi[1]), pack2bf(hi[2], hi[3])};
      }
      if (r0 + r < mlen && c0 + c < g.N)
        *reinterpret_cast<u32x4*>(static_cast<OT*>(g.C) + (mbase + r0 + r) * g.N + c0 + c) = o;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <bool GU, typename OT, int WR, int MI, int NI>
int launch_tile(const char* name, hipStream_t s, I8Args a) {
  constexpr int BM = WR * MI * 32, CW = (4 / WR) * NI * 32 / (GU ? 2 : 1);
  a.Tn = cdiv(a.N, CW);
  const int64_t tiles = (a.offsets ? a.R / BM + a.E : cdiv(a.R, BM)) * a.Tn;  // the most that any routing can produce
  MOE_LAUNCH(name, (k_i8_tile<GU, OT, WR, MI, NI>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(256), 0, s, a);
  return check_launch(name);
}

template <bool GU, typename OT>
int product(const char* name, hipStream_t s, const I8Args& a) {
  const int64_t r = a.R / a.E;
  const int form = r <= 24 ? 0 : r <= 64 ? 1 : r <= 192 ? 2 : 3;
  if (form == 0) return launch_small<GU, OT>(name, s, a);
  if (form == 1) return launch_tile<GU, OT, 1, 2, 2>(name, s, a);
  if (form == 2) return launch_tile<GU, OT, 2, 2, 4>(name, s, a);
  return launch_tile<GU, OT, 2, 4, 4>(name, s, a);
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

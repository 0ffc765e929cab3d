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
// ask the same few memory channels.  One token, two experts, H 4096, F 14336: 24 us for the down projection (117 MB, 5.0 TB/s),
// 19 us on the experts of the call before, which the 256 MB cache still holds in part; 4096 x 4096, 16, 32, 64 rows: 7, 10, 14 us,
// where a block's start and its waves' meeting count.
//
// More rows (k_i8_tile): both operands from memory straight to LDS.  That token's gate and up products: 40 us (235 MB, 5.9
// TB/s), 38 us on the same experts again.  128 rows on 8 experts of that layer: 145 us for gate and up (940 MB, 6.5 TB/s: all the
// card reads), 75 for the down projection; 1002 rows: 235 and 98 us (4.0 and 4.8 TB/s), between the weights' stream and the matrix
// instructions; 16384 rows: 1.83 ms for gate and up (3.85 Tops, 2.1 Pops/s) and 0.87 ms (2.2), where the matrix instructions' power
// sets the clock (8192^3: 2.39 Pops/s, a library's product 2.41).
#include <algorithm>
#include <type_traits>
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
  bool scan;            // k_i8_small: blocks for the passes that there are alone
  bool tails;           // tiles: experts' last rows behind all whole tiles
  int parts;            // tiles: blocks that a tile's reduction is split over; their sums go to C as int32 [parts][R][columns]
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
  // Block slots: every expert's first pass, then the passes past those.  With far fewer rows than experts (g.scan) the slots are
  // the passes that there are, experts one after the other: E 128, 8 rows 32 -> 21 us, but 64 rows 56 -> 63.
  int e = slot, pass = 0;
  const int lane = threadIdx.x & 63, skip = g.scan ? 0 : 1;
  if (g.scan || slot >= g.E) {
    int x = g.scan ? slot : slot - g.E;
    for (int e0 = 0;; e0 += 64) {
      if (e0 >= g.E) return;
      const int i = e0 + lane;
      const int c = i < g.E ? max((int)((seg(g, i + 1) - seg(g, i) + kI8Pass - 1) / kI8Pass) - skip, 0) : 0;
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
        pass = x - (__shfl(upto, l) - __shfl(c, l)) + skip;
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
int launch_small(hipStream_t s, I8Args a) {
  constexpr const char* name = GU ? "k_i8_small_gu" : "k_i8_small";
  const int64_t live = std::min<int64_t>(a.E, a.R);  // experts with rows, at most
  a.scan = a.R * 4 <= a.E;
  const int64_t slots = (a.scan ? live : a.E) + a.R / kI8Pass;  // the most passes that any routing can take
  if (cdiv(a.N, GU ? 32 : 64) * live >= 512) {
    a.Tn = cdiv(a.N, GU ? 32 : 64);
    MOE_LAUNCH(name, (k_i8_small<GU, OT, 4, 4>), dim3((unsigned)(a.Tn * slots)), dim3(256), 0, s, a);
  } else if (GU || cdiv(a.N, 32) * live >= 256) {
    a.Tn = cdiv(a.N, GU ? 16 : 32);
    MOE_LAUNCH(name, (k_i8_small<GU, OT, 2, 8>), dim3((unsigned)(a.Tn * slots)), dim3(512), 0, s, a);
  } else if constexpr (!GU) {
    a.Tn = cdiv(a.N, 16);
    MOE_LAUNCH(name, (k_i8_small<GU, OT, 1, 8>), dim3((unsigned)(a.Tn * slots)), dim3(512), 0, s, a);
  }
  return check_launch(name);
}

// ---- many rows ----
//
// A tile (i8_tile): up to 256 rows of an expert by 256 weight rows (GU: 128 gate rows and the matching up rows, 32 by 32) on
// v_mfma_i32_32x32x32_i8, four waves, one a SIMD.  Both operands go from memory straight to LDS (global_load_lds) in slices of
// 128 bytes of a row, whole cache lines, a row's eight 16-byte chunks swizzled so that the 16 rows a fragment read touches at
// once lie in distinct banks.
struct I8Place {
  int e;
  int64_t mbase;  // the tile's first row
  int mlen, n0;   // its rows; its first output column
  int k0, klen;   // the columns of A and B to sum over
  int part;
  int turn;       // TURN: the eighth of the reduction that it starts with
};

__device__ __attribute__((aligned(16))) const uint8_t g_i8_zero[16] = {0};
struct __attribute__((packed, aligned(4))) Scale4 { float v[4]; };
typedef __attribute__((address_space(3))) void lds_i8_t;

// s_waitcnt vmcnt(n), and lgkmcnt(0) or unconstrained.
template <int N, bool LGKM0>
__device__ __forceinline__ void i8_wait() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (LGKM0 ? 0 : 15 << 8));
}

// LDS of a tile of WR MI 32 rows: NS stages of a slice of both operands.
template <int WR, int MI, int NI>
constexpr int i8_stage() { return (WR * MI + 4 / WR * NI) * 32 * 128; }

// WR x (4 / WR) waves of MI x NI fragments.  The ring holds NS slices: while slice kt is multiplied the next NS - 1 are on their
// way.  A slice is four 32-wide quarters of MI NI matrix instructions, each followed by at most a fragment read of the next
// quarter and a refill piece or two (16 bytes a lane).  The slice's one barrier lies inside its last quarter, when the wave's
// own LDS reads of the slice have long drained under matrix instructions: behind it slice kt + 1 is complete and slice kt's
// stage is free for slice kt + NS.
template <bool GU, typename OT, int WR, int MI, int NI, int NS, bool NT, bool TURN>
__device__ __forceinline__ void i8_tile(const I8Args& g, const I8Place& at, uint8_t* smem) {
  constexpr int WC = 4 / WR, BM = WR * MI * 32, BN = WC * NI * 32;
  constexpr int SA = BM * 128, STAGE = i8_stage<WR, MI, NI>();
  constexpr int QA = BM / 32, QB = BN / 32, NP = QA + QB;  // 16-byte pieces of a wave's share of a slice
  constexpr bool PART = std::is_same_v<OT, int>;           // int32 sums of a part of the reduction
  constexpr int CW = GU ? BN / 2 : BN, WCOLS = CW / WC;    // output columns of the tile and of a wave
  constexpr int CP = (WCOLS * (int)sizeof(OT) + 16) / 4;   // words a row of a wave's output strip of 32 rows
  static_assert(!(GU && PART), "gate and up sums meet in one block");
  static_assert(4 * 32 * CP * 4 <= NS * STAGE, "the output strips reuse the ring");
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm0 = wv / WC * (MI * 32), wn0 = wv % WC * (NI * 32);
  const int i32 = lane & 31, h = lane >> 5;
  const int K = at.klen, nk = (K + 127) / 128, whole = K / 128;
  const int turn = TURN && whole == nk ? at.turn * (nk / 8) : 0;

  // piece p of a wave's share: instruction j fills rows 8 j + lane / 8 of its operand's tile, slot lane % 8 of the row.  Rows
  // past the tile repeat the last one.  A lane's address is a scalar base and an offset of 32 bits of its own that no slice
  // changes; the instruction's own offset moves both the address and the place in LDS, so four pieces share m0 (the offsets are
  // off by as much, and kBias keeps them positive).
  constexpr uint32_t kBias = 3 * 1024;
  const int64_t eb = (int64_t)at.e * g.N * g.K + at.k0;
  const uint8_t* const b_base[2] = {g.B + eb, (GU ? g.B2 : g.B) + eb};
  const uint8_t* const a_base = g.A + (g.row_slot == nullptr ? at.mbase * g.K : (int64_t)0) + at.k0;
  uint32_t a_off[QA], b_off[QB];
  auto chunk_of = [&](int j) { return (lane & 7) ^ ((4 * j + (lane >> 4)) & 7); };
#pragma unroll
  for (int q = 0; q < QA; ++q) {
    const int j = QA * wv + q, r = min(8 * j + (lane >> 3), at.mlen - 1);
    a_off[q] = (uint32_t)(g.row_slot == nullptr ? (int64_t)r : source_row(g, at.mbase + r)) * (uint32_t)g.K + chunk_of(j) * 16 +
               (kBias - q % 4 * 1024);
  }
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int j = QB * wv + q, i = 8 * j + (lane >> 3);
    const int n = GU ? at.n0 + (i >> 6) * 32 + (i & 31) : at.n0 + i;
    b_off[q] = (uint32_t)min(n, g.N - 1) * (uint32_t)g.K + chunk_of(j) * 16 + (kBias - q % 4 * 1024);
  }
  // Piece p of slice kt to the stage at byte s; past the row's end A is zeros and B the row's first bytes.  Issued from asm: the
  // compiler would make every LDS read that it cannot tell apart wait for all of them; the waits are the loop's own.  (m0 is
  // written by the scalar unit: one wait state.)
  auto fill = [&](int kt, int s, auto p_c, bool full) {
    constexpr int p = decltype(p_c)::value;
    constexpr bool IS_A = p < QA;
    constexpr int q = IS_A ? p : p - QA;
    const int j = (IS_A ? QA : QB) * wv + q;
    const uint8_t* const base = IS_A ? a_base : b_base[GU ? (8 * j >> 5) & 1 : 0];
    uint32_t off;
    if constexpr (IS_A) off = a_off[q];
    else off = b_off[q];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_i8_t*)(smem + s + (IS_A ? 0 : SA) + (j - q % 4) * 1024);
    if (full) {
      const int kr = !TURN || kt + turn < nk ? kt + turn : kt + turn - nk;
      const uint8_t* const at_kt = base - kBias + (int64_t)kr * 128;
      if constexpr (NT && !IS_A)
        __asm__ volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%2 nt" : : "v"(off), "s"(at_kt), "n"(q % 4 * 1024), "{m0}"(lds) : "memory");
      else
        __asm__ volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%2" : : "v"(off), "s"(at_kt), "n"(q % 4 * 1024), "{m0}"(lds) : "memory");
    } else {
      const int k = kt * 128 + chunk_of(j) * 16;
      const uint8_t* const row = base + (off - (kBias - q % 4 * 1024) - chunk_of(j) * 16);
      const uint8_t* const src = k < K ? row + k : IS_A ? g_i8_zero : row;
      __asm__ volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "{m0}"(lds + q % 4 * 1024) : "memory");
    }
  };
  // fragment f of quarter ks of the slice in stage s, in the order in which the quarter's matrix instructions need them
  auto read_frag = [&](int s, int ks, int f, i32x4(&fa)[MI], i32x4(&fb)[NI]) {
    const bool is_a = f == 0 || f > NI;
    const int x = is_a ? (f ? f - NI : 0) : f - 1, row = (is_a ? wm0 : wn0) + x * 32 + i32;
    const i32x4 v = *reinterpret_cast<const i32x4*>(smem + s + (is_a ? 0 : SA) + row * 128 +
                                                    (((2 * ks + h) ^ ((row >> 1) & 7)) << 4));
    if (is_a) fa[x] = v;
    else fb[x] = v;
  };

  i32x16 acc[MI][NI];
#pragma unroll
  for (int mi = 0; mi < MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[mi][ni][j] = 0;

  // Refill pieces: the first PD from the barrier on, the others in the next slice's first quarter.
  constexpr int SLOTS = MI * NI, NF = MI + NI, SLACK = std::max(std::min(SLOTS - NF, 4), 0), PD = std::min(NP, SLOTS - SLACK);
  // FILL 0: none; 1: whole slices; 2: the slice may end inside.  PLO, PHI: pieces, spread over the slots from RLO on.  VM: loads
  // that may still be on their way at the barrier (-1: no barrier).
  auto quarter = [&](auto fill_c, auto plo_c, auto phi_c, auto rlo_c, auto vm_c, const i32x4(&ca)[MI], const i32x4(&cb)[NI],
                     int ns, int nks, bool read_next, i32x4(&na)[MI], i32x4(&nb)[NI], int fkt, int fs) {
    constexpr int FILL = decltype(fill_c)::value, PLO = decltype(plo_c)::value, PHI = decltype(phi_c)::value;
    constexpr int RLO = decltype(rlo_c)::value, VM = decltype(vm_c)::value;
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (([&] {
         constexpr int mi = I / NI, ni = I % NI;
         if constexpr (VM >= 0 && I == RLO) {
           i8_wait<VM, true>();
           __asm__ volatile("" ::: "memory");
           __builtin_amdgcn_s_barrier();
           __asm__ volatile("" ::: "memory");
           __builtin_amdgcn_sched_barrier(0);
         }
         acc[mi][ni] = __builtin_amdgcn_mfma_i32_32x32x32_i8(cb[ni], ca[mi], acc[mi][ni], 0, 0, 0);
         __builtin_amdgcn_sched_barrier(0);
         // (reads: one a slot, or as many as it takes to end with the quarter)
         if constexpr (I >= RLO) {
           constexpr int N = SLOTS - RLO, R0 = N >= NF ? std::min(I - RLO, NF) : NF * (I - RLO) / N;
           constexpr int R1 = N >= NF ? std::min(I - RLO + 1, NF) : NF * (I - RLO + 1) / N;
           if (read_next) {
             [&]<int... X>(std::integer_sequence<int, X...>) {
               (read_frag(ns, nks, R0 + X, na, nb), ...);
             }(std::make_integer_sequence<int, R1 - R0>{});
           }
         }
         if constexpr (FILL > 0 && I >= RLO) {
           constexpr int P0 = PLO + (PHI - PLO) * (I - RLO) / (SLOTS - RLO), P1 = PLO + (PHI - PLO) * (I - RLO + 1) / (SLOTS - RLO);
           [&]<int... P>(std::integer_sequence<int, P...>) {
             (fill(fkt, fs, std::integral_constant<int, P0 + P>{}, FILL == 1 || fkt < whole), ...);
           }(std::make_integer_sequence<int, P1 - P0>{});
         }
         __builtin_amdgcn_sched_barrier(0);
       }()), ...);
    }(std::make_integer_sequence<int, SLOTS>{});
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
  using C2 = std::integral_constant<int, 2>;
  using CN = std::integral_constant<int, -1>;
  using CD = std::integral_constant<int, PD>;
  using CP_ = std::integral_constant<int, NP>;
  using CS = std::integral_constant<int, SLACK>;
  i32x4 fa0[MI], fb0[NI], fa1[MI], fb1[NI];
  auto next = [&](int s) { return s + STAGE == NS * STAGE ? 0 : s + STAGE; };
  auto prev = [&](int s) { return s == 0 ? (NS - 1) * STAGE : s - STAGE; };
  // Slice kt, in stage s.  F0: fills of the rest of slice kt + NS - 1, F1: of the first of slice kt + NS; VM as above.
  auto slice = [&](auto f0, auto f1, auto vm, int kt, int s) {
    quarter(f0, CD{}, CP_{}, C0{}, CN{}, fa0, fb0, s, 1, true, fa1, fb1, kt + NS - 1, prev(s));
    quarter(C0{}, C0{}, C0{}, C0{}, CN{}, fa1, fb1, s, 2, true, fa0, fb0, 0, 0);
    quarter(C0{}, C0{}, C0{}, C0{}, CN{}, fa0, fb0, s, 3, true, fa1, fb1, 0, 0);
    quarter(f1, C0{}, CD{}, CS{}, vm, fa1, fb1, next(s), 0, kt + 1 < nk, fa0, fb0, kt + NS, s);
  };
  // nothing of the compiler's own may be on its way in the loop: it would wait there for everything that is
  i8_wait<0, true>();
  for (int t = 0; t < NS && t < nk; ++t) {
    [&]<int... P>(std::integer_sequence<int, P...>) {
      ((P < PD || t < NS - 1 ? fill(t, t * STAGE, std::integral_constant<int, P>{}, t < whole) : void()), ...);
    }(std::make_integer_sequence<int, NP>{});
  }
  if (nk >= NS) i8_wait<(NS - 2) * NP + PD, false>();  // slice 0 is there
  else i8_wait<0, false>();
  lds_sync();
  for (int f = 0; f < NF; ++f) read_frag(0, 0, f, fa0, fb0);
  int kt = 0, s = 0;
  using CV = std::integral_constant<int, (NS - 2) * NP>;
  for (; kt + NS < whole; ++kt, s = next(s)) slice(C1{}, C1{}, CV{}, kt, s);
  for (; kt + NS < nk; ++kt, s = next(s)) slice(C2{}, C2{}, CV{}, kt, s);
  if (kt + NS - 1 < nk) {
    slice(C2{}, C0{}, CV{}, kt, s);
    ++kt, s = next(s);
  }
  for (; kt < nk; ++kt, s = next(s)) slice(C0{}, C0{}, C0{}, kt, s);
  __syncthreads();

  // The matrix instructions take the weights as their M operand, so a lane holds one row of C and, in each four accumulators,
  // four columns in a row: acc[mi][ni][j] = C[wm0 + 32 mi + lane % 32][wn0 + 32 ni + 8 (j / 4) + 4 (lane / 32) + j % 4].  Each
  // wave turns its strips of 32 rows over through LDS of its own, so that rows leave in whole lines.
  uint32_t* const cs = reinterpret_cast<uint32_t*>(smem) + wv * 32 * CP;
  const int c0 = at.n0 + wv % WC * WCOLS;  // the wave's first column
  const float* const sb = g.sb + (int64_t)at.e * g.N;
  const float* const sb2 = GU ? g.sb2 + (int64_t)at.e * g.N : nullptr;
  // the lane's scales, all asked for before the first is used: [0] of every accumulator column (GU: of the gate), [1] of the up
  constexpr int NS4 = GU ? NI * 2 : NI * 4;
  Scale4 sc[GU ? 2 : 1][NS4];
  float sx[MI];
  if constexpr (!PART) {
#pragma unroll
    for (int u = 0; u < NS4; ++u) {
      const int n = min(c0 + u * 8 + h * 4, g.N - 4);
      sc[0][u] = *reinterpret_cast<const Scale4*>(sb + n);
      if constexpr (GU) sc[1][u] = *reinterpret_cast<const Scale4*>(sb2 + n);
    }
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) sx[mi] = g.sa[source_row(g, at.mbase + min(wm0 + mi * 32 + i32, at.mlen - 1))];
  }
  OT* const out = static_cast<OT*>(g.C) + (PART ? (int64_t)at.part * g.R * g.N : 0);
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int r0 = wm0 + mi * 32;  // the strip's first row of the tile
    if (r0 >= at.mlen) break;
    __asm__ volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < NS4; ++u) {
      const int c = u * 8 + h * 4, v = u % 4;  // the lane's column of the strip
      if constexpr (PART) {
        const i32x16& t = acc[mi][u / 4];
        *reinterpret_cast<i32x4*>(cs + i32 * CP + c) = i32x4{t[4 * v], t[4 * v + 1], t[4 * v + 2], t[4 * v + 3]};
      } else {
        f32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (GU) {
            const float gv = (float)acc[mi][u / 4 * 2][4 * v + j] * sx[mi] * sc[0][u].v[j];
            o[j] = gv * sig_i8(gv) * ((float)acc[mi][u / 4 * 2 + 1][4 * v + j] * sx[mi] * sc[1][u].v[j]);
          } else {
            o[j] = (float)acc[mi][u / 4][4 * v + j] * sx[mi] * sc[0][u].v[j];
          }
        }
        if constexpr (sizeof(OT) == 2)
          *reinterpret_cast<uint2*>(cs + i32 * CP + c / 2) = uint2{pack2bf(o[0], o[1]), pack2bf(o[2], o[3])};
        else *reinterpret_cast<f32x4*>(cs + i32 * CP + c) = o;
      }
    }
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    constexpr int PER = 16 / sizeof(OT);  // columns of a 16-byte store
    constexpr int LPR = WCOLS / PER;      // lanes a row
#pragma unroll
    for (int u = 0; u < 32 * LPR / 64; ++u) {
      const int r = u * (64 / LPR) + lane / LPR, c = lane % LPR * PER;
      const u32x4 o = *reinterpret_cast<const u32x4*>(cs + r * CP + c * (int)sizeof(OT) / 4);
      if (r0 + r < at.mlen && c0 + c < g.N)
        *reinterpret_cast<u32x4*>(out + (at.mbase + r0 + r) * g.N + c0 + c) = o;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The number of row tiles of expert e: all (KIND 0), those of more than 64 rows (1) or a shorter one behind them (2).
template <int BM, int KIND>
__device__ __forceinline__ int i8_row_tiles(const I8Args& g, int e) {
  if (e >= g.E) return 0;
  const int64_t r = max(seg(g, e + 1) - seg(g, e), (int64_t)0);
  const int all = (int)((r + BM - 1) / BM), tall = (int)((r + BM - 65) / BM);
  return KIND == 0 ? all : KIND == 1 ? tall : all - tall;
}
template <int BM, int KIND>
__device__ __forceinline__ int i8_total(const I8Args& g, int lane) {
  int sum = 0;
  for (int e0 = 0; e0 < g.E; e0 += 64) sum += i8_row_tiles<BM, KIND>(g, e0 + lane);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  return __builtin_amdgcn_readfirstlane(sum) * g.Tn;
}
// Tile number L (below the total) of that kind: experts one after the other, within an expert groups of up to 8 row tiles with the
// columns walked inside a group, so that the tiles that run at once share few operand panels.
template <int BM, int KIND>
__device__ __forceinline__ I8Place i8_place(const I8Args& g, int L, int cw, int lane) {
  int e = 0, before = 0, cnt = 0;  // row tiles of the experts before e, and of e
  for (int e0 = 0;; e0 += 64) {
    if (e0 >= g.E) return I8Place{};  // (only where offsets decrease and the total has overflowed: no rows)
    const int c = i8_row_tiles<BM, KIND>(g, e0 + lane);
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
  I8Place p;
  p.e = __builtin_amdgcn_readfirstlane(e);
  cnt = __builtin_amdgcn_readfirstlane(cnt);
  const int local = L - __builtin_amdgcn_readfirstlane(before) * g.Tn;
  constexpr int GM = 8;
  const int grp = local / (GM * g.Tn), rest = local - grp * GM * g.Tn, gm = min(cnt - grp * GM, GM);
  const int nt = rest / gm;
  int mt = grp * GM + rest - nt * gm;
  const int64_t lo = seg(g, p.e), hi = seg(g, p.e + 1);
  if (KIND == 2) mt = i8_row_tiles<BM, 1>(g, p.e);
  p.mbase = lo + (int64_t)mt * BM;
  p.mlen = (int)min(hi - p.mbase, (int64_t)BM);
  p.n0 = nt * cw;
  p.k0 = 0;
  p.klen = g.K;
  p.part = 0;
  return p;
}

// Tiles of up to BM rows by BN weight rows, each as tall as its rows need.  One dimension of blocks, sized for the most tiles any
// routing can produce; the tiles that there are lie in 8 contiguous ranges, one an XCD (blockIdx mod 8).
//   256 x 256: many rows.  g.tails: the short tiles of experts' last rows come behind all others, so that they fill the last round.
//   192 x 128, 64 x 256: few enough that the weights' stream bounds the product; two blocks a CU, for more of it on its way.
//     DEEP: one block a CU with more slices on their way, where there are no more tiles than CUs, or 49 to 160 rows and long sums.
//     TURN: an expert's tiles start their reductions at different eighths where all of its rows are in one row of tiles: in step,
//     tiles whose weight rows lie a power of two apart ask the same few memory channels.  (Tiles that share weights stay in step:
//     14336 x 4096, 512 rows 48 | 68 us.)
template <bool GU, typename OT, int BM, int BN, bool DEEP, bool TURN>
__global__ __launch_bounds__(256, BM == 256 || DEEP ? 1 : 2) void k_i8_tile(I8Args g) {
  constexpr int SMEM = BM == 256 ? std::max(3 * i8_stage<1, 4, 2>(), 2 * i8_stage<2, 4, 4>())
                       : DEEP ? 6 * i8_stage<2, 1, 2>() : BM == 192 ? 2 * i8_stage<2, 3, 2>() : 2 * i8_stage<1, 2, 2>();
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];
  const int lane = threadIdx.x & 63;
  constexpr int CW = GU ? BN / 2 : BN;
  const int xcd = (int)(blockIdx.x & 7), slot = (int)(blockIdx.x >> 3);
  I8Place at;
  if (BM == 256 && g.tails) {
    const int n1 = i8_total<BM, 1>(g, lane), n2 = i8_total<BM, 2>(g, lane), c1 = (n1 + 7) >> 3, c2 = (n2 + 7) >> 3;
    if (slot < c1) {
      const int L = xcd * c1 + slot;
      if (L >= n1) return;
      at = i8_place<BM, 1>(g, L, CW, lane);
    } else {
      const int L = xcd * c2 + slot - c1;
      if (slot - c1 >= c2 || L >= n2) return;
      at = i8_place<BM, 2>(g, L, CW, lane);
    }
  } else {
    const int n = i8_total<BM, 0>(g, lane) * g.parts, chunk = (n + 7) >> 3, L = xcd * chunk + slot;
    if (slot >= chunk || L >= n) return;
    at = i8_place<BM, 0>(g, L / g.parts, CW, lane);
    if constexpr (std::is_same_v<OT, int>) {
      const int nk = (g.K + 127) / 128;
      at.part = L % g.parts;
      at.k0 = nk * at.part / g.parts * 128;
      at.klen = min(nk * (at.part + 1) / g.parts * 128, g.K) - at.k0;
    }
  }
  if (at.mlen <= 0) return;
  at.turn = TURN && seg(g, at.e + 1) - seg(g, at.e) <= BM ? slot & 7 : 0;
  if constexpr (BM == 256) {
    if (at.mlen > 192) i8_tile<GU, OT, 2, 4, 4, 2, BM != 256, TURN>(g, at, smem);
    else if (at.mlen > 128) i8_tile<GU, OT, 2, 3, 4, 2, BM != 256, TURN>(g, at, smem);
    else if (at.mlen > 64) i8_tile<GU, OT, 1, 4, 2, 3, BM != 256, TURN>(g, at, smem);
    else i8_tile<GU, OT, 1, 2, 2, 3, BM != 256, TURN>(g, at, smem);
  } else if constexpr (BM == 192) {
    if (at.mlen > 128) i8_tile<GU, OT, 2, 3, 2, DEEP ? 3 : 2, BM != 256, TURN>(g, at, smem);
    else if (at.mlen > 64) i8_tile<GU, OT, 2, 2, 2, DEEP ? 4 : 2, BM != 256, TURN>(g, at, smem);
    else i8_tile<GU, OT, 2, 1, 2, DEEP ? 6 : 3, BM != 256, TURN>(g, at, smem);
  } else {
    i8_tile<GU, OT, 1, 2, 2, 2, BM != 256, TURN>(g, at, smem);
  }
}

template <bool GU, typename OT, int BM, int BN, bool DEEP = false, bool TURN = false>
int launch_tile(hipStream_t s, I8Args a, int parts) {
  constexpr const char* name = BM == 64    ? (GU ? "k_i8_tile64_gu" : "k_i8_tile64")
                               : BM == 256 ? (GU ? "k_i8_tile256_gu" : "k_i8_tile256")
                               : TURN      ? (GU ? "k_i8_tile192_turn_gu" : "k_i8_tile192_turn")
                               : DEEP      ? (GU ? "k_i8_tile192_deep_gu" : "k_i8_tile192_deep")
                                           : (GU ? "k_i8_tile192_gu" : "k_i8_tile192");
  static_assert(BM == 192 || !std::is_same_v<OT, int>, "no product splits the reduction of other tiles");
  a.Tn = cdiv(a.N, GU ? BN / 2 : BN);
  a.tails = parts == 1 && a.R >= 512 * (int64_t)a.E;
  a.parts = parts;
  // the most tiles that any routing can produce, and what rounding two ranges up may add
  const int64_t tiles = (a.offsets ? a.R / BM + std::min<int64_t>(a.E, a.R) : cdiv(a.R, BM)) * a.Tn * parts;
  MOE_LAUNCH(name, (k_i8_tile<GU, OT, BM, BN, DEEP, TURN>), dim3((unsigned)((tiles + 7) / 8 * 8 + 8)), dim3(256), 0, s, a);
  return check_launch(name);
}

// y of a product whose reduction was split: the parts' sums added (whole numbers: in any order) and scaled.  A block a row.
template <typename OT>
__global__ __launch_bounds__(256) void k_i8_join(I8Args g, const int* __restrict__ part) {
  const int64_t row = blockIdx.x;
  int e = 0;
  if (g.offsets != nullptr) {  // the row's expert: those whose rows all come before it
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < g.E; e0 += 64) {
      const int n = __popcll(__ballot(e0 + lane < g.E && seg(g, min(e0 + lane, g.E - 1) + 1) <= row));
      e += n;
      if (n < 64) break;
    }
    e = __builtin_amdgcn_readfirstlane(e);
    if (e >= g.E || row < seg(g, e)) return;
  }
  const float sx = g.sa[source_row(g, row)];
  const float* const sb = g.sb + (int64_t)e * g.N;
  for (int c = threadIdx.x * 4; c < g.N; c += 1024) {
    i32x4 v = {0, 0, 0, 0};
    for (int p = 0; p < g.parts; ++p) v += *reinterpret_cast<const i32x4*>(part + ((int64_t)p * g.R + row) * g.N + c);
    const Scale4 sc = *reinterpret_cast<const Scale4*>(sb + c);
    f32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (float)v[j] * sx * sc.v[j];
    OT* const y = static_cast<OT*>(g.C) + row * g.N + c;
    if constexpr (sizeof(OT) == 4) *reinterpret_cast<f32x4*>(y) = o;
    else *reinterpret_cast<uint2*>(y) = uint2{pack2bf(o[0], o[1]), pack2bf(o[2], o[3])};
  }
}

// The form of a product, by its sizes alone (the host does not know the rows of each expert).  r: rows an expert that can have
// any; tiles: of 192 x 128.  Measured (us; E, H, F for both products of the experts, K x N for one):
//   small | 192 x 128    few tiles: E 8, H 4096, F 14336, one token: gate and up (448 tiles) 47 | 40, down (64) 24 | 53.  E 128,
//                        H 2048, F 768, 8, 16 rows (96 and 128, 192 and 256 tiles): 21 | 24, 27 | 25.  4096 x 4096, 16 rows (32)
//                        7 | 13; 4096 x 14336 (112) 15 | 14
//   small | 192 x 128    little work: 4096 x 4096, 32, 64 rows 10 | 13, 14 | 13; 2048 x 2048, 128, 256 rows 8 | 11, 13 | 14; E 8,
//                        1024 x 512, r 64, 128: 5.8 | 7.4, 8.8 | 8.6; E 8, 528 x 3088, r 16, 32: 6.7 | 6.8, 9 | 7
//   small | 192 | 64     E 8, H 4096, F 14336, r 1, 4, 16: 191 | 182 | 267, 241 | 216 | 284, 282 | 222 | 290.  E 128, H 2048, F 768,
//                        r 2, 4, 8, 32: 110 | 108 | 107, 122 | 119 | 112, 126 | 122 | 114, 191 | 133 | 125; routed with a Zipf(1.1)
//                        bias, r 4, 8, 16, 32: 65 | 60 | 55, 100 | 87 | 76, 126 | 95 | 101, 178 | 117 | 117.  E 64, H 2048, F 1408,
//                        r 6, 24: 110 | 99 | 102, 153 | 106 | 108.  E 32, 1024 x 1024, r 32: 11 | 8 | 11
//   192 | 64             small experts, both products with r 2, 8, 16, 24: E 64, H 2048, F 1024: 69 | 62, 82 | 70, 83 | 72, 86 | 74;
//                        E 96, 1024, 2048: 106 | 96, 119 | 108, 123 | 113, 130 | 120; E 128, 1024, 1024: 79 | 69, 86 | 76, 88 | 78,
//                        92 | 82; E 160, 1536, 768: 108 | 96, 118 | 106, 123 | 111, 128 | 115; E 256, 2048, 512: 158 | 132, 171 | 148,
//                        177 | 154, 182 | 160; E 512, 1024, 256: 140 | 97, 155 | 107, 162 | 113, 166 | 118; E 128, 4096, 512: 163 |
//                        156, 178 | 176, 184 | 182, 187 | 185.  Routed with a Zipf(1.1) bias, r 2, 8, 24: E 128, 1024, 1024: 59 | 57,
//                        85 | 71, 105 | 101; E 256, 2048, 512: 94 | 78, 156 | 133, 199 | 181; E 160, 1536, 768: 78 | 83, 112 | 100,
//                        135 | 139.  Behind with columns that fill no whole tile (E 72, 2048, 1008: 85 | 83, 103 | 116, 105 | 118,
//                        108 | 120) and with fewer weights than the rule asks for (E 64, 1408, 1408: 69 | 72, 75 | 77, 78 | 78, 82 | 81)
//   192 | deep | 256     E 8, H 4096, F 14336, r 16: 222 | 237 | 279; 32: 239 | 254 | 296; 64: 319 | 287 | 316; 128: 374 | 354 |
//                        411; 256: 520 | 606 | 547; 512: 887 | 924 | 904; 1024: 1601 | 1785 | 1554.  E 128, H 2048, F 768 (16 and
//                        6 slices), r 128: 205 | 244 | 210.  4096 x 14336, 96 to 256 rows 25 | 18 | 26 to 30 | 25 | 45, 512: 40 |
//                        47 | 48, 1024: 71 | 79 | 60; 4096 x 4096, 2048 rows 43 | 50 | 50
//   deep | turn          E 8, H 4096, F 14336, r 50, 64, 96, 128, 150: 270 | 274, 293 | 291, 331 | 327, 363 | 355, 385 | 376.  E 32, H
//                        2048, F 4096: 176 | 163, 188 | 172, 213 | 203, 234 | 227, 251 | 240.  4096 x 28672, 64 rows 26 | 22
//   parts 1 | 2 | 4      14336 x 4096, 64 rows: 35 | 26 | 21; 256: 58 | 39 | 36; 512: 58 | 45 | 54; 4096 x 4096, 64: 13 | 14 | 15
enum { kSmall, kTile64, kTile192, kTile192Deep, kTile192Turn, kTile256 };
struct I8Form {
  int kind;
  int parts;  // blocks that a tile's reduction is split over
};
I8Form i8_form(int64_t R, int64_t K, int64_t N, int64_t E, bool gu) {
  const int64_t live = std::min(E, R), r = R / live, nk = (K + 127) / 128, cols = gu ? 2 * N : N;
  const int64_t tiles = (r + 191) / 192 * live * ((cols + 127) / 128);
  if (r <= 16 && tiles < 192) return {kSmall, 1};
  if (live * N * K <= (int64_t)1 << 26 && R * K * N <= (int64_t)1 << (live == 1 ? 30 : 28) && (nk < 64 || r <= 16))
    return {kSmall, 1};
  if (r > 512 && (r + 255) / 256 * live * ((cols + 255) / 256) >= 192) return {kTile256, 1};
  if (N * K <= (int64_t)1 << 21 && live * N * K >= (int64_t)1 << 27 && r <= 24) return {kTile64, 1};
  const int parts = !gu && tiles <= 128 && nk >= 64 ? (int)std::min<int64_t>(4, 256 / tiles) : 1;
  const bool deep = r > 48 && (tiles * parts <= 256 || (r <= 160 && nk >= 32));
  return {!deep ? kTile192 : r <= 192 ? kTile192Turn : kTile192Deep, parts};
}

// A product's tiles; a split reduction's int32 sums (OT int) are made by the 192 x 128 forms alone, i8_form's only ones with parts.
template <bool GU, typename OT>
int launch_form(hipStream_t s, const I8Args& a, const I8Form& f) {
  switch (f.kind) {
    case kTile192: return launch_tile<GU, OT, 192, 128>(s, a, f.parts);
    case kTile192Deep: return launch_tile<GU, OT, 192, 128, true>(s, a, f.parts);
    case kTile192Turn: return launch_tile<GU, OT, 192, 128, true, true>(s, a, f.parts);
  }
  if constexpr (!std::is_same_v<OT, int>) {
    if (f.kind == kTile64) return launch_tile<GU, OT, 64, 256>(s, a, f.parts);
    if (f.kind == kTile256) return launch_tile<GU, OT, 256, 256>(s, a, f.parts);
  }
  return fail_arg("int8 product: no tiles for form %d in %d parts", f.kind, f.parts);
}

template <bool GU, typename OT>
int product(hipStream_t s, const I8Args& a, void* ws) {
  const I8Form f = i8_form(a.R, a.K, a.N, a.E, GU);
  if (f.kind == kSmall) return launch_small<GU, OT>(s, a);
  if constexpr (!GU) {
    if (f.parts > 1) {
      I8Args p = a;
      p.C = ws;
      if (int rc = launch_form<false, int>(s, p, f)) return rc;
      p = a;
      p.parts = f.parts;
      MOE_LAUNCH("k_i8_join", k_i8_join<OT>, dim3((unsigned)a.R), dim3(256), 0, s, p, static_cast<const int*>(ws));
      return check_launch("k_i8_join");
    }
  }
  return launch_form<GU, OT>(s, a, f);
}

// Bytes of the parts' sums.
size_t i8_part_bytes(int64_t R, int64_t K, int64_t N, int64_t E) {
  const I8Form f = i8_form(R, K, N, E, false);
  return f.parts > 1 ? (size_t)f.parts * R * N * 4 : 0;
}

bool al16_i8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

// Sizes that the kernels' 32-bit quantities hold: sums (127 * 127 K), row offsets inside an expert's matrix, block counts.
constexpr int64_t kI8MaxK = 131056;
bool i8_sizes(int64_t R, int64_t K, int64_t N, int64_t E) {
  return R >= 0 && R <= INT32_MAX / 2 && K >= 16 && K % 16 == 0 && K <= kI8MaxK && N >= 8 && N % 8 == 0 && E >= 1 && E <= 1024 &&
         N * K < ((int64_t)1 << 32) - 4096 && (E + R / kI8Pass + 1) * ((N + 15) / 16) < INT32_MAX;
}
}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_matmul_int8_workspace(int64_t R, int64_t K, int64_t N, int64_t E) {
  if (R <= 0 || !i8_sizes(R, K, N, E)) return 0;
  return i8_part_bytes(R, K, N, E);
}

extern "C" int moe_matmul_int8(const void* xq, const float* sx, const void* wq, const float* sw, const int32_t* offsets,
                               int64_t R, int64_t K, int64_t N, int64_t E, void* y, int y_dtype, void* workspace,
                               size_t ws_bytes, void* stream) {
  if (!i8_sizes(R, K, N, E) || (y_dtype != MOE_BF16 && y_dtype != MOE_F32) || (!offsets && E != 1))
    return fail_arg("moe_matmul_int8: bad arguments R=%lld K=%lld N=%lld E=%lld (need K %% 16 == 0, K <= %lld, N %% 8 == 0, "
                    "N K < 2^32, E <= 1024, bf16 or fp32 y; E == 1 without offsets)", (long long)R, (long long)K, (long long)N,
                    (long long)E, (long long)kI8MaxK);
  if (R == 0) return 0;
  if (!xq || !sx || !wq || !sw || !y || !al16_i8(xq) || !al16_i8(wq) || !al16_i8(y))
    return fail_arg("moe_matmul_int8: null or misaligned pointer");
  const size_t need = moe_matmul_int8_workspace(R, K, N, E);
  if (need > 0 && (!workspace || !al16_i8(workspace) || ws_bytes < need))
    return set_error("moe_matmul_int8: workspace %zu < %zu bytes, or misaligned", ws_bytes, need), MOE_EWORKSPACE;
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
  return y_dtype == MOE_BF16 ? product<false, uint16_t>(s, a, workspace)
                             : product<false, float>(s, a, workspace);
}

// act (bf16), then act in int8 and its scales; the down projection's partial sums lie where act was
extern "C" size_t moe_swiglu_fwd_int8_workspace(int64_t R, int64_t H, int64_t F, int64_t E) {
  if (R <= 0 || !i8_sizes(R, H, F, E) || !i8_sizes(R, F, H, E)) return 0;
  return up256(std::max((size_t)R * F * 2, i8_part_bytes(R, F, H, E))) + up256((size_t)R * F) + up256((size_t)R * 4);
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
  if (row_slot && T * H >= ((int64_t)1 << 32) - 4096)
    return fail_arg("moe_swiglu_fwd_int8: T H must be below 2^32 with row_slot, got T=%lld H=%lld", (long long)T, (long long)H);
  if (!xq || !sx || !wg_q || !sg || !wu_q || !su || !wd_q || !sd || !offsets || !y || !al16_i8(xq) || !al16_i8(wg_q) ||
      !al16_i8(wu_q) || !al16_i8(wd_q) || !al16_i8(y) || !al16_i8(workspace))
    return fail_arg("moe_swiglu_fwd_int8: null or misaligned pointer");
  const size_t need = moe_swiglu_fwd_int8_workspace(R, H, F, E);
  if (!workspace || ws_bytes < need)
    return set_error("moe_swiglu_fwd_int8: workspace %zu < %zu bytes", ws_bytes, need), MOE_EWORKSPACE;
  uint8_t* const act = static_cast<uint8_t*>(workspace);
  uint8_t* const aq = act + up256(std::max((size_t)R * F * 2, i8_part_bytes(R, F, H, E)));
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
  if (int rc = product<true, uint16_t>(s, a, nullptr)) return rc;
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
  return product<false, uint16_t>(s, b, act);
}

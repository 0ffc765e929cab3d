// Load balance of the router's choices within each sequence, over valid tokens only: the loss, the z-loss, the per-expert
// counts and their gradient with respect to the logits.
//
// Sequence s holds the tokens [off[s], off[s + 1]); n_s of them are valid (mask).  With p = softmax(logits) and c_se the
// choices of expert e by the valid tokens of s,
//   f_se = E c_se / (K n_s),   P_se = mean over valid t of p[t, e],   L_s = sum_e f_se P_se,
//   balance = coef / S+ * sum_s L_s   (S+ sequences have a valid token),   z = zcoef / n * sum over valid t of lse_t^2,
//   d balance / dl[t, j] = coef / (S+ n_s) p[t, j] (f_sj - sum_e p[t, e] f_se),   dz / dl[t, j] = 2 zcoef / n lse_t p[t, j].
//
// Both directions are one read of the logits (and one write of the gradient), N E 4 bytes: bound by memory for large
// batches, by launches and chains of dependent loads for small ones.  A block owns a run of consecutive tokens.  LPT lanes
// share a token, each with four neighbouring experts (one 16-byte load); a lane group's U tokens are loaded and their
// softmax formed while the block finds the sequences that meet its run, and then it walks them.  A sequence's probabilities
// are summed in registers and over the block's waves, its counts by LDS atomics of integers, and go to a row of their own:
// run c and sequence s meet in row c + s, which is distinct for every pair that meets (along a walk one of the two grows by
// one), and a sequence's rows are consecutive.  Its rows are then added in order (64 bits), so every result is the same from
// run to run: by one block that also forms the losses where there are few rows, else by a block a sequence and a third launch.
// Small batches are one block's altogether (k_balance_one).
//
// Measured, forward | sums | losses | backward, us: 65536 tokens, E 64, K 6, 16 sequences 10.7 | 7.1 | 4.4 | 13.1; 32768 tokens,
// E 128, K 8, 700 sequences 15.0 | 4.9 | 4.4 | 13.8 (16.8 MB read a forward, 33.6 MB moved a backward: 1.6 and 2.6 TB/s; what is
// left is launches and each kernel's chain of loads).  A ticket whose last block forms the losses, in place of the third
// launch: sums 10.3 us, nothing won.
#include <algorithm>

#include "common.h"

namespace moe {
namespace {

constexpr int kMaxBalanceE = 256;
constexpr int kBalanceNT = 512;  // threads of a block of the two kernels over tokens
constexpr int kFewSeqs = 64;     // sequences, and rows of sums, that one block adds up
constexpr int kFewRows = 128;
constexpr int kOneSeqs = 16;     // sequences, experts and tokens a lane group of a batch that one block finishes
constexpr int kOneE = 64;
constexpr int kOneU = 4;

struct BalanceArgs {
  const float* logits;    // [N][E]
  const int64_t* idx;     // [N][K] (forward)
  const int64_t* off;     // [S + 1]; null: one sequence of all tokens
  const uint8_t* mask;    // [N] nonzero: valid; null: all are
  int64_t N, S;
  int E, K;
  float* part_p;          // [rows][E]
  int* part_c;            // [rows][E]
  int* part_n;            // [rows]
  float* part_z;          // [runs]
  // backward
  const int64_t* counts;  // [S][E]
  const int64_t* tokens;  // [S + 2]
  const float* grad_b;
  const float* grad_z;
  float bcoef, zcoef;
  float* dlogits;
};

template <int LPT>
__device__ __forceinline__ float team_max(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
template <int LPT>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

__device__ __forceinline__ int64_t seq_off(const BalanceArgs& a, int64_t s) {
  return a.off ? a.off[s] : (s == 0 ? 0 : a.N);
}

// The first sequence that ends past token t (S if none does): 64 ends a step.
__device__ __forceinline__ int64_t first_seq(const BalanceArgs& a, int64_t t, int lane) {
  int64_t lo = 0, n = a.S;  // among sequences [lo, lo + n)
  while (n > 0) {
    const int64_t w = (n + 63) / 64;  // ends at lo + w - 1, lo + 2 w - 1, ...
    const int64_t i = min((lane + 1) * w, n) - 1;
    const unsigned long long past = __ballot(seq_off(a, lo + i + 1) > t);
    if (!past) return lo + n;
    if (w == 1) return lo + __builtin_ctzll(past);
    const int64_t l = __builtin_ctzll(past);
    const int64_t end = min((l + 1) * w, n);
    lo += l * w;
    n = end - l * w;
  }
  return lo;
}

// The four logits of this lane of one token; -inf past E.
template <bool VEC>
__device__ __forceinline__ f32x4 load_logits(const BalanceArgs& a, int64_t t, int e0) {
  const float* const p = a.logits + t * a.E + e0;
  f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if constexpr (VEC) {
    if (e0 < a.E) v = *reinterpret_cast<const f32x4*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e0 + j < a.E) v[j] = p[j];
  }
  return v;
}

// softmax of the token whose logits these lanes hold: p in their place, logsumexp returned.
template <int LPT>
__device__ __forceinline__ float softmax_token(f32x4& p) {
  const float m = team_max<LPT>(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])));
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = expf(p[j] - m);
  const float s = team_sum<LPT>((p[0] + p[1]) + (p[2] + p[3]));
  const float inv = 1.f / s;
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] *= inv;
  return m + logf(s);
}

// The bounds of up to 63 sequences from s0 on, one a lane (the last one's end in the next lane).
struct SeqWindow {
  int64_t s0, bound;
};
__device__ __forceinline__ SeqWindow seq_window(const BalanceArgs& a, int64_t s0, int lane) {
  return SeqWindow{s0, s0 < a.S ? seq_off(a, min(s0 + lane, a.S)) : a.N};
}
// The window that the walk of a run starting at c0 begins with.
__device__ __forceinline__ SeqWindow first_window(const BalanceArgs& a, int64_t c0, int lane) {
  return seq_window(a, a.S <= 63 ? 0 : first_seq(a, c0, lane), lane);
}

// Walks the sequences that meet tokens [c0, c1): visit(s, lo, hi) for each.
template <class V>
__device__ __forceinline__ void walk(const BalanceArgs& a, SeqWindow w, int64_t c0, int64_t c1, int lane, V visit) {
  int64_t pos = c0;
  while (w.s0 < a.S && pos < c1) {
    const int n = (int)min((int64_t)63, a.S - w.s0);
    // of these, from the first that ends past the tokens walked so far
    const unsigned long long past = __ballot(w.bound > pos) >> 1;
    for (int i = past ? __builtin_ctzll(past) : 63; i < n && pos < c1; ++i) {
      const int64_t b = __shfl(w.bound, i), e = __shfl(w.bound, i + 1);
      const int64_t lo = max(b, pos), hi = min(e, c1);
      if (lo >= c1) return;  // starts grow: none after it meets the run
      if (lo < hi) {
        visit(w.s0 + i, lo, hi);
        pos = hi;
      }
    }
    w = seq_window(a, w.s0 + 63, lane);
  }
}

// A block's run is U tokens for each of its lane groups.
template <int LPT, int U>
constexpr int run_tokens() {
  return U * (kBalanceNT / LPT);
}

template <int LPT, int U, bool VEC>
__global__ __launch_bounds__(kBalanceNT) void k_balance_fwd(BalanceArgs a) {
  constexpr int TEAMS = kBalanceNT / LPT, NW = kBalanceNT / 64, EW = LPT * 4;
  __shared__ f32x4 s_p[2][NW][LPT];
  __shared__ int s_c[2][EW];
  __shared__ int s_n[2][NW];
  __shared__ float s_z[NW];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, sub = lane % LPT, team = tid / LPT;
  const int64_t c = blockIdx.x;
  const int64_t c0 = c * run_tokens<LPT, U>(), c1 = min(a.N, c0 + run_tokens<LPT, U>());
  const int E = a.E, K = a.K;
  f32x4 p[U];
  int64_t id[U];  // the first of the lane's share of its tokens' choices
  bool ok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = min(c0 + u * TEAMS + team, c1 - 1);
    p[u] = load_logits<VEC>(a, t, sub * 4);
    id[u] = sub < K ? a.idx[t * K + sub] : -1;
    ok[u] = a.mask == nullptr || a.mask[t] != 0;
  }
  const SeqWindow w0 = first_window(a, c0, lane);
  for (int i = tid; i < 2 * EW; i += kBalanceNT) s_c[i / EW][i % EW] = 0;
  float lse[U];
#pragma unroll
  for (int u = 0; u < U; ++u) lse[u] = softmax_token<LPT>(p[u]);
  __syncthreads();
  float z = 0.f;
  int b = 0;
  walk(
      a, w0, c0, c1, lane, [&](int64_t s, int64_t lo, int64_t hi) {
        f32x4 P = {0.f, 0.f, 0.f, 0.f};
        int n = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t t = c0 + u * TEAMS + team;
          if (ok[u] && t >= lo && t < hi) {
            P += p[u];
            z += lse[u] * lse[u];
            ++n;
            if (id[u] >= 0 && id[u] < E) atomicAdd(&s_c[b][id[u]], 1);
            for (int k = sub + LPT; k < K; k += LPT) {
              const int64_t i = a.idx[t * K + k];
              if (i >= 0 && i < E) atomicAdd(&s_c[b][i], 1);
            }
          }
        }
#pragma unroll
        for (int o = LPT; o < 64; o <<= 1) {  // over the wave's lane groups
          n += __shfl_xor(n, o);
#pragma unroll
          for (int j = 0; j < 4; ++j) P[j] += __shfl_xor(P[j], o);
        }
        if (lane < LPT) s_p[b][wv][sub] = P;
        if (lane == 0) s_n[b][wv] = n;
        __syncthreads();
        const int64_t row = c + s;
        if (tid < E) {
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < NW; ++w) v += reinterpret_cast<const float*>(s_p[b][w])[tid];
          a.part_p[row * E + tid] = v;
          a.part_c[row * E + tid] = s_c[b][tid];
          s_c[b][tid] = 0;  // used again two sequences on, behind the next one's barrier
        }
        if (tid == kBalanceNT - 1) {
          int v = 0;
#pragma unroll
          for (int w = 0; w < NW; ++w) v += s_n[b][w];
          a.part_n[row] = v;
        }
        b ^= 1;
      });
#pragma unroll
  for (int o = LPT; o < 64; o <<= 1) z += __shfl_xor(z, o);
  if (lane == 0) s_z[wv] = z;
  __syncthreads();
  if (tid == 0) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += s_z[w];
    a.part_z[c] = v;
  }
}

// Gradient: each token finds its own sequence among the windows of bounds (in LDS), so the counts of a lane group's U tokens
// are in flight together whatever sequences they are of.
template <int LPT, int U, bool VEC>
__global__ __launch_bounds__(kBalanceNT) void k_balance_bwd(BalanceArgs a) {
  constexpr int TEAMS = kBalanceNT / LPT;
  __shared__ int64_t s_b[64];
  const int lane = threadIdx.x & 63, sub = lane % LPT, team = threadIdx.x / LPT;
  const int64_t c0 = (int64_t)blockIdx.x * run_tokens<LPT, U>(), c1 = min(a.N, c0 + run_tokens<LPT, U>());
  const int E = a.E, e0 = sub * 4;
  f32x4 p[U];
  bool ok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = min(c0 + u * TEAMS + team, c1 - 1);
    p[u] = load_logits<VEC>(a, t, e0);
    ok[u] = a.mask == nullptr || a.mask[t] != 0;
  }
  const float gb = a.bcoef * (a.grad_b ? a.grad_b[0] : 1.f), gz = a.zcoef * (a.grad_z ? a.grad_z[0] : 1.f);
  const float total = (float)max(a.tokens[a.S], (int64_t)1), used = (float)max(a.tokens[a.S + 1], (int64_t)1);
  SeqWindow w = first_window(a, c0, lane);
  const float cz = gz * 2.f / total, cs = (float)E / (float)a.K;
  int64_t seq[U];
#pragma unroll
  for (int u = 0; u < U; ++u) seq[u] = -1;
  for (;;) {  // windows until one ends past the run
    if (threadIdx.x < 64) s_b[threadIdx.x] = w.bound;
    __syncthreads();
    const int n = (int)min((int64_t)63, a.S - w.s0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = min(c0 + u * TEAMS + team, c1 - 1);
      int lo = 0, len = n;  // the first of the window's sequences that ends past t
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        const int half = len >> 1;
        const bool on = len > 0 && s_b[lo + half + 1] <= t;
        lo = on ? lo + half + 1 : lo;
        len = len > 0 ? (on ? len - half - 1 : half) : 0;
      }
      if (seq[u] < 0 && lo < n && s_b[lo] <= t) seq[u] = w.s0 + lo;
    }
    const bool more = w.s0 + n < a.S && s_b[n] < c1;
    if (!more) break;
    w = seq_window(a, w.s0 + n, lane);
    __syncthreads();
  }
  uint32_t cnt[U][4], n[U];  // all counts are below 2^31: their low halves
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t s = max(seq[u], (int64_t)0);
    n[u] = reinterpret_cast<const uint32_t*>(a.tokens + s)[0];
    const uint32_t* const c = reinterpret_cast<const uint32_t*>(a.counts + s * E + e0);
    if constexpr (VEC) {  // a lane past E (fewer experts than lanes) has no counts
      const bool in = e0 < E;
      const u32x4 lo = *reinterpret_cast<const u32x4*>(in ? c : reinterpret_cast<const uint32_t*>(a.counts));
      const u32x4 hi = *reinterpret_cast<const u32x4*>((in ? c : reinterpret_cast<const uint32_t*>(a.counts)) + 4);
      cnt[u][0] = in ? lo[0] : 0u, cnt[u][1] = in ? lo[2] : 0u, cnt[u][2] = in ? hi[0] : 0u, cnt[u][3] = in ? hi[2] : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) cnt[u][j] = e0 + j < E ? c[2 * j] : 0u;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = c0 + u * TEAMS + team;
    const float lse = softmax_token<LPT>(p[u]);
    const float in = 1.f / (float)max(n[u], 1u), cb = gb / used * in, fs = cs * in;
    f32x4 d;
    float pf = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      d[j] = (float)cnt[u][j] * fs;
      pf += p[u][j] * d[j];
    }
    pf = team_sum<LPT>(pf);
    const bool live = ok[u] && seq[u] >= 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = live ? p[u][j] * (cb * (d[j] - pf) + cz * lse) : 0.f;
    if (t < c1) {
      float* const o = a.dlogits + t * E + e0;
      if constexpr (VEC) {
        if (e0 < E) *reinterpret_cast<f32x4*>(o) = d;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e0 + j < E) o[j] = d[j];
      }
    }
  }
}

struct BalanceSumArgs {
  const int64_t* off;
  const float* part_p;
  const int* part_c;
  const int* part_n;
  const float* part_z;
  int64_t N, S, runs;
  int E, K, run;
  float bcoef, zcoef;
  int64_t* counts;        // [S][E]
  int64_t* tokens;        // [S + 2]
  float* mean_p;          // [S][E]
  double* seq_loss;       // [S]
  float* balance;
  float* z;
};

template <typename T>
__device__ __forceinline__ T wave_sum_of(T v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// One sequence's rows, added by W waves of a block (a power of two; wave w of them).  Lanes lie side by side on a row's
// experts, 64 at a time, and with fewer experts on several rows.  Every wave of the block calls it, with live false where
// it has no sequence.  EJ: 64-wide pieces of a row.  sm: a row for each of the block's waves.  Returns the sequence's loss and
// valid tokens to wave 0's lanes.
template <int EJ>
__device__ __forceinline__ double sum_sequence(const BalanceSumArgs& a, int64_t s, bool live, int W, int w, int lane,
                                               double* sm_p, int64_t* sm_c, int64_t* sm_n, int64_t& n) {
  const int E = a.E;
  int64_t r0 = 0, r1 = 0;
  if (live) {
    const int64_t b = min(max(a.off ? a.off[s] : (int64_t)0, (int64_t)0), a.N);
    const int64_t h = min(max(a.off ? a.off[s + 1] : a.N, (int64_t)0), a.N);
    r0 = b / a.run + s;
    r1 = h > b ? (h - 1) / a.run + s + 1 : r0;
  }
  int EP = 1;
  while (EP < E && EP < 64) EP *= 2;
  const int el = lane & (EP - 1), rl = lane / EP, rows = 64 / EP;
  double p[EJ];
  int64_t c[EJ];
#pragma unroll
  for (int j = 0; j < EJ; ++j) p[j] = 0., c[j] = 0;
  for (int64_t r = r0 + w * rows + rl; r < r1; r += 4 * W * rows) {
    float pv[4][EJ];
    int cv[4][EJ];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t ri = r + i * W * rows;
#pragma unroll
      for (int j = 0; j < EJ; ++j) {
        const int e = el + 64 * j;
        const bool in = ri < r1 && e < E;
        pv[i][j] = in ? a.part_p[ri * E + e] : 0.f;
        cv[i][j] = in ? a.part_c[ri * E + e] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < EJ; ++j) {
        p[j] += (double)pv[i][j];
        c[j] += cv[i][j];
      }
  }
  n = 0;
  for (int64_t r = r0 + w * 64 + lane; r < r1; r += W * 64) n += a.part_n[r];
  n = wave_sum_of(n);
#pragma unroll
  for (int j = 0; j < EJ; ++j)
    for (int o = EP; o < 64; o <<= 1) {
      p[j] += __shfl_xor(p[j], o);
      c[j] += __shfl_xor(c[j], o);
    }
  if (W > 1) {
#pragma unroll
    for (int j = 0; j < EJ; ++j) {
      sm_p[w * (64 * EJ) + lane + 64 * j] = p[j];
      sm_c[w * (64 * EJ) + lane + 64 * j] = c[j];
    }
    if (lane == 0) sm_n[w] = n;
    __syncthreads();
    if (w == 0) {
      for (int x = 1; x < W; ++x) {
#pragma unroll
        for (int j = 0; j < EJ; ++j) {
          p[j] += sm_p[x * (64 * EJ) + lane + 64 * j];
          c[j] += sm_c[x * (64 * EJ) + lane + 64 * j];
        }
        n += sm_n[x];
      }
    }
    __syncthreads();
  }
  double l = 0.;
  if (live && w == 0) {
    const double inv = n > 0 ? 1. / (double)n : 0.;
#pragma unroll
    for (int j = 0; j < EJ; ++j) {
      const int e = el + 64 * j;
      if (rl == 0 && e < E) {
        const double m = p[j] * inv;
        a.counts[s * E + e] = c[j];
        a.mean_p[s * E + e] = (float)m;
        l += (double)E * (double)c[j] * inv / (double)a.K * m;
      }
    }
    l = wave_sum_of(l);
    if (lane == 0) a.tokens[s] = n;
  }
  return l;
}

// A small batch, whole, by one block: its probabilities and choices go to LDS, a wave takes every eighth sequence, and the
// losses follow behind a barrier.  1000 tokens of 8 experts in 8 sequences: 9.5 us, where runs and their sums took 6.5 and 8 in
// two launches; the calls' own cost on the host is most of what is left of both directions' 19 us.
template <int LPT, bool VEC>
__global__ __launch_bounds__(kBalanceNT) void k_balance_one(BalanceArgs a, BalanceSumArgs o) {
  constexpr int TEAMS = kBalanceNT / LPT, NW = kBalanceNT / 64, EW = LPT * 4, TOK = kOneU * TEAMS;
  static_assert(EW <= 64);
  __shared__ __attribute__((aligned(16))) float s_p[TOK * EW];  // 32 KB
  __shared__ uint8_t s_id[TOK * (EW < 32 ? EW : 32)];           // K <= min(E, 32)
  __shared__ float s_l[TOK];                                    // squared logsumexp, negative where the token is masked
  __shared__ int s_c[NW][EW];
  __shared__ double s_loss[kOneSeqs], s_z[kOneSeqs];
  __shared__ int s_n[kOneSeqs];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, sub = lane % LPT, team = tid / LPT;
  const int E = a.E, K = a.K, N = (int)a.N, S = (int)a.S;
  f32x4 p[kOneU];
  bool ok[kOneU];
#pragma unroll
  for (int u = 0; u < kOneU; ++u) {
    const int64_t t = min(u * TEAMS + team, N - 1);
    p[u] = load_logits<VEC>(a, t, sub * 4);
    ok[u] = a.mask == nullptr || a.mask[t] != 0;
  }
  const int64_t bound = min(max(seq_off(a, min(lane, S)), (int64_t)0), a.N);
  for (int i = tid; i < N * K; i += kBalanceNT) {
    const int64_t v = a.idx[i];
    s_id[i] = (uint8_t)(v >= 0 && v < E ? v : 255);
  }
#pragma unroll
  for (int u = 0; u < kOneU; ++u) {
    const int t = u * TEAMS + team;
    const float lse = softmax_token<LPT>(p[u]);
    if (t < N) {
      *reinterpret_cast<f32x4*>(s_p + t * EW + sub * 4) = p[u];
      if (sub == 0) s_l[t] = ok[u] ? lse * lse : -1.f;
    }
  }
  __syncthreads();
  const int el = lane % EW, rl = lane / EW;
  for (int s = wv; s < S; s += NW) {
    const int lo = (int)__shfl(bound, s), hi = (int)__shfl(bound, s + 1);
    if (lane < EW) s_c[wv][lane] = 0;
    __asm__ volatile("" ::: "memory");
    double P = 0., z = 0.;
    int n = 0;
    for (int t = lo + rl; t < hi; t += 64 / EW) P += !(s_l[t] < 0.f) ? (double)s_p[t * EW + el] : 0.;
    for (int t = lo + lane; t < hi; t += 64) {
      const float l = s_l[t];
      if (!(l < 0.f)) {
        z += (double)l;
        ++n;
        for (int k = 0; k < K; ++k) {
          const int e = s_id[t * K + k];
          if (e < E) atomicAdd(&s_c[wv][e], 1);
        }
      }
    }
#pragma unroll
    for (int x = EW; x < 64; x <<= 1) P += __shfl_xor(P, x);
    n = wave_sum_of(n);
    z = wave_sum_of(z);
    __asm__ volatile("" ::: "memory");
    const double inv = n > 0 ? 1. / (double)n : 0.;
    double l = 0.;
    if (lane < E) {
      const int c = s_c[wv][lane];
      o.counts[s * E + lane] = c;
      o.mean_p[s * E + lane] = (float)(P * inv);
      l = (double)E * (double)c * inv / (double)K * (P * inv);
    }
    l = wave_sum_of(l);
    if (lane == 0) {
      o.tokens[s] = n;
      s_loss[s] = l;
      s_z[s] = z;
      s_n[s] = n;
    }
  }
  __syncthreads();
  if (tid == 0) {
    double sum = 0., z = 0.;
    int all = 0, used = 0;
    for (int s = 0; s < S; ++s) {
      sum += s_loss[s];
      z += s_z[s];
      all += s_n[s];
      used += s_n[s] > 0;
    }
    o.tokens[S] = all;
    o.tokens[S + 1] = used;
    *o.balance = (float)((double)o.bcoef * sum / fmax((double)used, 1.));
    *o.z = (float)((double)o.zcoef * z / fmax((double)all, 1.));
  }
}

// This thread's share of the runs' z sums.
__device__ __forceinline__ double z_share(const BalanceSumArgs& a) {
  double zs = 0.;
  for (int64_t i = threadIdx.x; i < a.runs; i += blockDim.x) zs += (double)a.part_z[i];
  return zs;
}

// The losses from the sequences' losses and the threads' shares of the z sums, by a whole block.
template <typename F, typename G>
__device__ __forceinline__ void total_losses(const BalanceSumArgs& a, double zs, F loss_of, G tokens_of, double* red) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wv = tid >> 6;
  double sum = 0., all = 0., used = 0.;  // whole numbers below 2^53 are exact
  for (int64_t i = tid; i < a.S; i += nt) {
    sum += loss_of(i);
    const int64_t m = tokens_of(i);
    all += (double)m;
    used += m > 0 ? 1. : 0.;
  }
  double v[4] = {wave_sum_of(sum), wave_sum_of(zs), wave_sum_of(all), wave_sum_of(used)};
  __syncthreads();
  if (lane < 4) red[wv * 4 + lane] = lane == 0 ? v[0] : lane == 1 ? v[1] : lane == 2 ? v[2] : v[3];
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < (nt >> 6); ++w)
      for (int i = 0; i < 4; ++i) v[i] += red[w * 4 + i];
    a.tokens[a.S] = (int64_t)v[2];
    a.tokens[a.S + 1] = (int64_t)v[3];
    *a.balance = (float)((double)a.bcoef * v[0] / fmax(v[3], 1.));
    *a.z = (float)((double)a.zcoef * v[1] / fmax(v[2], 1.));
  }
}

// Up to kFewSeqs sequences: one block of 16 waves, W of them a sequence.
template <int EJ>
__global__ __launch_bounds__(1024) void k_balance_sum_few(BalanceSumArgs a, int W) {
  __shared__ double s_p[16 * 64 * EJ];
  __shared__ int64_t s_c[16 * 64 * EJ];
  __shared__ int64_t s_n[16];
  __shared__ double s_loss[kFewSeqs];
  __shared__ int64_t s_tok[kFewSeqs];
  __shared__ double red[64];
  const double zs = z_share(a);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, grp = wv / W, groups = 16 / W;
  for (int64_t s0 = 0; s0 < a.S; s0 += groups) {
    const int64_t s = s0 + grp;
    int64_t n;
    const double l = sum_sequence<EJ>(a, s, s < a.S, W, wv & (W - 1), lane, s_p + grp * W * 64 * EJ,
                                      s_c + grp * W * 64 * EJ, s_n + grp * W, n);
    if (s < a.S && (wv & (W - 1)) == 0 && lane == 0) {
      s_loss[s] = l;
      s_tok[s] = n;
    }
  }
  __syncthreads();
  total_losses(
      a, zs, [&](int64_t i) { return s_loss[i]; }, [&](int64_t i) { return s_tok[i]; }, red);
}

template <int EJ>
__global__ __launch_bounds__(1024) void k_balance_sum(BalanceSumArgs a) {
  __shared__ double s_p[16 * 64 * EJ];
  __shared__ int64_t s_c[16 * 64 * EJ];
  __shared__ int64_t s_n[16];
  int64_t n;
  const double l = sum_sequence<EJ>(a, blockIdx.x, true, blockDim.x >> 6, threadIdx.x >> 6, threadIdx.x & 63, s_p, s_c, s_n, n);
  if (threadIdx.x == 0) a.seq_loss[blockIdx.x] = l;
}

__global__ __launch_bounds__(1024) void k_balance_total(BalanceSumArgs a) {
  __shared__ double red[64];
  total_losses(
      a, z_share(a), [&](int64_t i) { return a.seq_loss[i]; }, [&](int64_t i) { return a.tokens[i]; }, red);
}

// Lane groups of a token and tokens of a group.  A group's U tokens are in flight together and a block's run is 128 or 256
// tokens (64 past 128 experts); batches that give fewer than 256 such runs take one token a group, for more blocks.
struct BalanceForm {
  int lpt, u, run;
};
BalanceForm balance_form(int64_t N, int64_t E, bool fwd) {
  BalanceForm f;
  f.lpt = 2;
  while (f.lpt * 4 < E) f.lpt *= 2;
  f.u = f.lpt <= 2 ? 1 : f.lpt <= 4 ? 2 : f.lpt <= 16 ? 4 : 8;
  if (N < (int64_t)256 * f.u * (kBalanceNT / f.lpt)) f.u = 1;
  if (!fwd) f.u = std::min(f.u, 2);
  f.run = f.u * (kBalanceNT / f.lpt);
  return f;
}

// A small batch is one block's (k_balance_one).  A wave has every eighth sequence and takes 64 / EW of its tokens a step (EW: 4
// lpt), so with one or two sequences the other waves wait for it: up to 48 steps on average, which is all that the host knows.
// A call in a graph of 20, us, one block | runs and their sums: E 8, one sequence of 256 tokens 7.6 | 10.5, 512 (64 steps) 11.6 | 10.7,
// 1024 19.2 | 11.3; two, 768 tokens (48 steps) 10.0 | 11.3, 1024 12.2 | 11.3; four, 1024 9.0 | 11.5; eight 7.5 | 12.5; sixteen
// 8.7 | 14.2.  At the same steps E 16, 32 and 64 are within 1 us of these in the first column and 2 in the second.  (One of
// several sequences that has nearly all the tokens costs what one sequence does.)
bool balance_in_one(int64_t N, int64_t E, int64_t S, int lpt) {
  return S <= kOneSeqs && E <= kOneE && N <= kOneU * (kBalanceNT / lpt) && N * lpt <= 768 * S;
}

size_t al256b(size_t v) { return (v + 255) & ~(size_t)255; }
struct BalanceWs {
  int64_t runs, rows;
  size_t off_loss, off_p, off_c, off_n, off_z, total;
};
BalanceWs balance_ws(int64_t N, int64_t E, int64_t S) {
  BalanceWs w;
  const int run = balance_form(N, E, true).run;
  w.runs = (N + run - 1) / run;
  w.rows = w.runs + S;
  w.off_loss = 0;
  w.off_p = w.off_loss + al256b((size_t)S * 8);
  w.off_c = w.off_p + al256b((size_t)w.rows * E * 4);
  w.off_n = w.off_c + al256b((size_t)w.rows * E * 4);
  w.off_z = w.off_n + al256b((size_t)w.rows * 4);
  w.total = w.off_z + al256b((size_t)w.runs * 4);
  return w;
}

int balance_check(const char* what, int64_t N, int64_t E, int64_t K, int64_t S) {
  const int64_t lim = INT32_MAX;
  if (N < 1 || N > lim / 32 || E < 1 || E > kMaxBalanceE || K < 1 || K > 32 || K > E || S < 1 || S > lim - 1)
    return fail_arg("%s: bad shape N=%lld E=%lld K=%lld S=%lld (need N, S >= 1, N < 2^26, E <= %d, K <= min(E, 32))", what, (long long)N,
                    (long long)E, (long long)K, (long long)S, kMaxBalanceE);
  return 0;
}

// VEC: every lane's four logits are one aligned 16-byte word.
#define MOE_BALANCE_FWD(VEC)                                                                                  \
  do {                                                                                                        \
    const dim3 grid((unsigned)runs), block(kBalanceNT);                                                       \
    switch (f.lpt * 16 + f.u) {                                                                               \
      case 2 * 16 + 1: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<2, 1, VEC>), grid, block, 0, s, a); break;  \
      case 4 * 16 + 1: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<4, 1, VEC>), grid, block, 0, s, a); break;  \
      case 4 * 16 + 2: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<4, 2, VEC>), grid, block, 0, s, a); break;  \
      case 8 * 16 + 1: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<8, 1, VEC>), grid, block, 0, s, a); break;  \
      case 8 * 16 + 4: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<8, 4, VEC>), grid, block, 0, s, a); break;  \
      case 16 * 16 + 1: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<16, 1, VEC>), grid, block, 0, s, a); break;\
      case 16 * 16 + 4: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<16, 4, VEC>), grid, block, 0, s, a); break;\
      case 32 * 16 + 1: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<32, 1, VEC>), grid, block, 0, s, a); break;\
      case 32 * 16 + 8: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<32, 8, VEC>), grid, block, 0, s, a); break;\
      case 64 * 16 + 1: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<64, 1, VEC>), grid, block, 0, s, a); break;\
      case 64 * 16 + 8: MOE_LAUNCH("k_balance_fwd", (k_balance_fwd<64, 8, VEC>), grid, block, 0, s, a); break;\
    }                                                                                                         \
  } while (0)
#define MOE_BALANCE_ONE(VEC)                                                                                  \
  do {                                                                                                        \
    const dim3 grid(1), block(kBalanceNT);                                                                    \
    switch (f.lpt) {                                                                                          \
      case 2: MOE_LAUNCH("k_balance_one", (k_balance_one<2, VEC>), grid, block, 0, s, a, b); break;           \
      case 4: MOE_LAUNCH("k_balance_one", (k_balance_one<4, VEC>), grid, block, 0, s, a, b); break;           \
      case 8: MOE_LAUNCH("k_balance_one", (k_balance_one<8, VEC>), grid, block, 0, s, a, b); break;           \
      case 16: MOE_LAUNCH("k_balance_one", (k_balance_one<16, VEC>), grid, block, 0, s, a, b); break;         \
    }                                                                                                         \
  } while (0)
#define MOE_BALANCE_BWD(VEC)                                                                                  \
  do {                                                                                                        \
    const dim3 grid((unsigned)runs), block(kBalanceNT);                                                       \
    switch (f.lpt * 16 + f.u) {                                                                               \
      case 2 * 16 + 1: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<2, 1, VEC>), grid, block, 0, s, a); break;  \
      case 4 * 16 + 1: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<4, 1, VEC>), grid, block, 0, s, a); break;  \
      case 4 * 16 + 2: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<4, 2, VEC>), grid, block, 0, s, a); break;  \
      case 8 * 16 + 1: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<8, 1, VEC>), grid, block, 0, s, a); break;  \
      case 8 * 16 + 2: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<8, 2, VEC>), grid, block, 0, s, a); break;  \
      case 16 * 16 + 1: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<16, 1, VEC>), grid, block, 0, s, a); break;\
      case 16 * 16 + 2: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<16, 2, VEC>), grid, block, 0, s, a); break;\
      case 32 * 16 + 1: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<32, 1, VEC>), grid, block, 0, s, a); break;\
      case 32 * 16 + 2: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<32, 2, VEC>), grid, block, 0, s, a); break;\
      case 64 * 16 + 1: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<64, 1, VEC>), grid, block, 0, s, a); break;\
      case 64 * 16 + 2: MOE_LAUNCH("k_balance_bwd", (k_balance_bwd<64, 2, VEC>), grid, block, 0, s, a); break;\
    }                                                                                                         \
  } while (0)

bool al16b(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_balance_fwd_workspace(int64_t N, int64_t E, int64_t S) {
  if (N < 1 || E < 1 || S < 1) return 0;
  return balance_ws(N, E, S).total;
}

extern "C" int moe_balance_fwd(const float* logits, const int64_t* idx, const int64_t* seq_offsets, const uint8_t* token_mask,
                               int64_t N, int64_t E, int64_t K, int64_t S, float balance_coef, float z_coef, float* balance,
                               float* z, int64_t* counts, int64_t* tokens, float* mean_prob, void* workspace,
                               size_t ws_bytes, void* stream) {
  if (int rc = balance_check("moe_balance_fwd", N, E, K, S)) return rc;
  if (!logits || !idx || !balance || !z || !counts || !tokens || !mean_prob || (!seq_offsets && S != 1))
    return fail_arg("moe_balance_fwd: null pointer argument");
  const BalanceWs w = balance_ws(N, E, S);
  if (ws_bytes < w.total || !workspace)
    return set_error("moe_balance_fwd: workspace %zu < %zu bytes", ws_bytes, w.total), MOE_EWORKSPACE;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const int64_t runs = w.runs;
  BalanceArgs a{};
  a.logits = logits;
  a.idx = idx;
  a.off = seq_offsets;
  a.mask = token_mask;
  a.N = N;
  a.S = S;
  a.E = (int)E;
  a.K = (int)K;
  const BalanceForm f = balance_form(N, E, true);
  a.part_p = reinterpret_cast<float*>(ws + w.off_p);
  a.part_c = reinterpret_cast<int*>(ws + w.off_c);
  a.part_n = reinterpret_cast<int*>(ws + w.off_n);
  a.part_z = reinterpret_cast<float*>(ws + w.off_z);
  BalanceSumArgs b{};
  b.off = seq_offsets;
  b.part_p = a.part_p;
  b.part_c = a.part_c;
  b.part_n = a.part_n;
  b.part_z = a.part_z;
  b.N = N;
  b.S = S;
  b.runs = runs;
  b.E = (int)E;
  b.K = (int)K;
  b.run = f.run;
  b.bcoef = balance_coef;
  b.zcoef = z_coef;
  b.counts = counts;
  b.tokens = tokens;
  b.mean_p = mean_prob;
  b.seq_loss = reinterpret_cast<double*>(ws + w.off_loss);
  b.balance = balance;
  b.z = z;
  const bool vec = E % 4 == 0 && al16b(logits);
  if (balance_in_one(N, E, S, f.lpt)) {
    if (vec) MOE_BALANCE_ONE(true);
    else MOE_BALANCE_ONE(false);
    return check_launch("moe_balance_fwd");
  }
  if (vec) MOE_BALANCE_FWD(true);
  else MOE_BALANCE_FWD(false);
  if (int rc = check_launch("k_balance_fwd")) return rc;
#define MOE_BALANCE_SUM(KERNEL, name, grid, block, ...)                               \
  do {                                                                                \
    if (E <= 64) MOE_LAUNCH(name, KERNEL<1>, grid, block, 0, s, __VA_ARGS__);         \
    else if (E <= 128) MOE_LAUNCH(name, KERNEL<2>, grid, block, 0, s, __VA_ARGS__);   \
    else MOE_LAUNCH(name, KERNEL<4>, grid, block, 0, s, __VA_ARGS__);                 \
  } while (0)
  if (S <= kFewSeqs && w.rows <= kFewRows) {
    int W = 16;
    while (W > 1 && W * S > 16) W /= 2;
    MOE_BALANCE_SUM(k_balance_sum_few, "k_balance_sum_few", dim3(1), dim3(1024), b, W);
    return check_launch("moe_balance_fwd");
  }
  // a sequence's rows by 16 waves where sequences are long on average, by 4 where they are many
  MOE_BALANCE_SUM(k_balance_sum, "k_balance_sum", dim3((unsigned)S), dim3(runs / S >= 16 ? 1024 : 256), b);
  MOE_LAUNCH("k_balance_total", k_balance_total, dim3(1), dim3(1024), 0, s, b);
  return check_launch("moe_balance_fwd");
}

extern "C" int moe_balance_bwd(const float* logits, const int64_t* counts, const int64_t* tokens, const int64_t* seq_offsets,
                               const uint8_t* token_mask, const float* grad_balance, const float* grad_z, int64_t N, int64_t E,
                               int64_t K, int64_t S, float balance_coef, float z_coef, float* dlogits, void* stream) {
  if (int rc = balance_check("moe_balance_bwd", N, E, K, S)) return rc;
  if (!logits || !counts || !tokens || !dlogits || (!seq_offsets && S != 1))
    return fail_arg("moe_balance_bwd: null pointer argument");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  BalanceArgs a{};
  a.logits = logits;
  a.off = seq_offsets;
  a.mask = token_mask;
  a.N = N;
  a.S = S;
  a.E = (int)E;
  a.K = (int)K;
  const BalanceForm f = balance_form(N, E, false);
  a.counts = counts;
  a.tokens = tokens;
  a.grad_b = grad_balance;
  a.grad_z = grad_z;
  a.bcoef = balance_coef;
  a.zcoef = z_coef;
  a.dlogits = dlogits;
  const int64_t runs = (N + f.run - 1) / f.run;
  if (E % 4 == 0 && al16b(logits) && al16b(counts) && al16b(dlogits)) MOE_BALANCE_BWD(true);
  else MOE_BALANCE_BWD(false);
  return check_launch("moe_balance_bwd");
}

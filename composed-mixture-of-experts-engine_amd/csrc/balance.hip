// Load balance of the router's choices within each sequence, over valid tokens only: the loss, the z-loss, the per-expert
// counts and their gradient with respect to the logits.
//
// Sequence s holds the tokens [off[s], off[s + 1]); n_s of them are valid (mask).  With p = softmax(logits) and c_se the
// choices of expert e by the valid tokens of s,
//   f_se = E c_se / (K n_s),   P_se = mean over valid t of p[t, e],   L_s = sum_e f_se P_se,
//   balance = coef / S+ * sum_s L_s   (S+ sequences have a valid token),   z = zcoef / n * sum over valid t of lse_t^2,
//   d balance / dl[t, j] = coef / (S+ n_s) p[t, j] (f_sj - sum_e p[t, e] f_se),   dz / dl[t, j] = 2 zcoef / n lse_t p[t, j].
//
// Both directions are one read of the logits (and one write of the gradient): N E 4 bytes, bound by memory for large
// batches and by two launches for small ones.  A wave owns a run of consecutive tokens and walks the sequences that meet
// it; LPT lanes share a token, each with every LPT-th expert.  A sequence's sums stay in registers until the wave leaves
// it, and go to a row of their own: run c and sequence s meet in row c + s, which is distinct for every pair that meets
// (along a walk one of the two grows by one), and a sequence's rows are consecutive.  k_balance_sum then adds each
// sequence's rows in order (64 bits), so every result is the same from run to run; its last block adds the sequences.
#include <algorithm>

#include "common.h"

namespace moe {
namespace {

constexpr int kMaxBalanceE = 256;

struct BalanceArgs {
  const float* logits;    // [N][E]
  const int64_t* idx;     // [N][K] (forward)
  const int64_t* off;     // [S + 1]; null: one sequence of all tokens
  const uint8_t* mask;    // [N] nonzero: valid; null: all are
  int64_t N, S;
  int E, K, run;          // run: tokens of a wave
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

// softmax of the token whose logits these lanes hold: p and logsumexp.
template <int LPT, int EPL>
__device__ __forceinline__ float softmax_token(float (&p)[EPL]) {
  float m = p[0];
#pragma unroll
  for (int j = 1; j < EPL; ++j) m = fmaxf(m, p[j]);
  m = team_max<LPT>(m);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    p[j] = expf(p[j] - m);
    s += p[j];
  }
  s = team_sum<LPT>(s);
  const float inv = 1.f / s;
#pragma unroll
  for (int j = 0; j < EPL; ++j) p[j] *= inv;
  return m + logf(s);
}

// Walks the sequences that meet tokens [c0, c1): visit(s, lo, hi) for each, gap(lo, hi) for the tokens of none.
template <class V, class G>
__device__ __forceinline__ void walk(const BalanceArgs& a, int64_t c0, int64_t c1, int lane, V visit, G gap) {
  int64_t s0 = first_seq(a, c0, lane), pos = c0;
  for (; s0 < a.S && pos < c1; s0 += 63) {
    // the bounds of up to 63 sequences, one a lane
    const int64_t mine = seq_off(a, min(s0 + lane, a.S));
    const int n = (int)min((int64_t)63, a.S - s0);
    // the first of them that starts past the run (starts grow)
    for (int i = 0; i < n && pos < c1; ++i) {
      const int64_t b = __shfl(mine, i), e = __shfl(mine, i + 1);
      const int64_t lo = max(b, pos), hi = min(e, c1);
      if (lo >= c1) {
        s0 = a.S;
        break;
      }
      if (lo < hi) {
        if (pos < lo) gap(pos, lo);
        visit(s0 + i, lo, hi);
        pos = hi;
      }
    }
  }
  if (pos < c1) gap(pos, c1);
}

template <int LPT, int EPL>
__global__ __launch_bounds__(256) void k_balance_fwd(BalanceArgs a) {
  constexpr int TPW = 64 / LPT;
  const int lane = threadIdx.x & 63, sub = lane % LPT, team = lane / LPT;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t c0 = c * a.run, c1 = min(a.N, c0 + a.run);
  if (c0 >= c1) return;
  const int E = a.E, K = a.K;
  float z = 0.f;
  walk(
      a, c0, c1, lane,
      [&](int64_t s, int64_t lo, int64_t hi) {
        float P[EPL];
        int C[EPL], n = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) P[j] = 0.f, C[j] = 0;
        for (int64_t t0 = lo; t0 < hi; t0 += TPW) {
          const int64_t t = t0 + team;
          const bool ok = t < hi && (a.mask == nullptr || a.mask[min(t, hi - 1)] != 0);
          const int64_t tr = min(t, hi - 1);
          float p[EPL];
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            const int e = sub + LPT * j;
            p[j] = e < E ? a.logits[tr * E + e] : -INFINITY;
          }
          const float lse = softmax_token<LPT, EPL>(p);
#pragma unroll
          for (int j = 0; j < EPL; ++j) P[j] += ok ? p[j] : 0.f;
          z += ok ? lse * lse : 0.f;
          n += ok;
          for (int k = 0; k < K; ++k) {
            const int64_t id = a.idx[tr * K + k];
#pragma unroll
            for (int j = 0; j < EPL; ++j) C[j] += ok && id == sub + LPT * j;
          }
        }
        // sums over the wave's teams
#pragma unroll
        for (int o = LPT; o < 64; o <<= 1) {
          n += __shfl_xor(n, o);
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            P[j] += __shfl_xor(P[j], o);
            C[j] += __shfl_xor(C[j], o);
          }
        }
        const int64_t row = c + s;
        if (team == 0) {
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            const int e = sub + LPT * j;
            if (e < E) {
              a.part_p[row * E + e] = P[j];
              a.part_c[row * E + e] = C[j];
            }
          }
        }
        if (lane == 0) a.part_n[row] = n;
      },
      [](int64_t, int64_t) {});
#pragma unroll
  for (int o = LPT; o < 64; o <<= 1) z += __shfl_xor(z, o);
  if (lane == 0) a.part_z[c] = z;
}

template <int LPT, int EPL>
__global__ __launch_bounds__(256) void k_balance_bwd(BalanceArgs a) {
  constexpr int TPW = 64 / LPT;
  const int lane = threadIdx.x & 63, sub = lane % LPT, team = lane / LPT;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t c0 = c * a.run, c1 = min(a.N, c0 + a.run);
  if (c0 >= c1) return;
  const int E = a.E;
  const float gb = a.bcoef * (a.grad_b ? a.grad_b[0] : 1.f), gz = a.zcoef * (a.grad_z ? a.grad_z[0] : 1.f);
  const float total = (float)max(a.tokens[a.S], (int64_t)1), used = (float)max(a.tokens[a.S + 1], (int64_t)1);
  const float cz = gz * 2.f / total;
  auto zeros = [&](int64_t lo, int64_t hi) {
    for (int64_t i = lo * E + lane; i < hi * E; i += 64) a.dlogits[i] = 0.f;
  };
  walk(
      a, c0, c1, lane,
      [&](int64_t s, int64_t lo, int64_t hi) {
        const float n = (float)max(a.tokens[s], (int64_t)1);
        const float cb = gb / (used * n), fs = (float)E / ((float)a.K * n);
        float f[EPL];
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const int e = sub + LPT * j;
          f[j] = e < E ? (float)a.counts[s * E + e] * fs : 0.f;
        }
        for (int64_t t0 = lo; t0 < hi; t0 += TPW) {
          const int64_t t = t0 + team, tr = min(t, hi - 1);
          const bool ok = a.mask == nullptr || a.mask[tr] != 0;
          float p[EPL];
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            const int e = sub + LPT * j;
            p[j] = e < E ? a.logits[tr * E + e] : -INFINITY;
          }
          const float lse = softmax_token<LPT, EPL>(p);
          float pf = 0.f;
#pragma unroll
          for (int j = 0; j < EPL; ++j) pf += p[j] * f[j];
          pf = team_sum<LPT>(pf);
          if (t < hi) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
              const int e = sub + LPT * j;
              const float d = p[j] * (cb * (f[j] - pf) + cz * lse);
              if (e < E) a.dlogits[t * E + e] = ok ? d : 0.f;
            }
          }
        }
      },
      zeros);
}

struct BalanceSumArgs {
  const int64_t* off;
  const float* part_p;
  const int* part_c;
  const int* part_n;
  const float* part_z;
  int64_t N, S, runs;
  int E, K, run, EP;      // EP: lanes of a row of experts, a power of two
  float bcoef, zcoef;
  int64_t* counts;        // [S][E]
  int64_t* tokens;        // [S + 2]
  float* mean_p;          // [S][E]
  double* seq_loss;       // [S]
  float* balance;
  float* z;
  unsigned* ticket;
};

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  const int wv = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[wv] = v;
  __syncthreads();
  T t = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) t += red[i];
  return t;
}

// One block a sequence: EP threads side by side on a row of experts, the block's other threads on further rows.
__global__ __launch_bounds__(1024) void k_balance_sum(BalanceSumArgs a) {
  __shared__ double s_p[1024];
  __shared__ int64_t s_c[1024];
  __shared__ double s_red[16];
  __shared__ int64_t s_redi[16];
  __shared__ bool s_last;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int64_t s = blockIdx.x;
  const int e = tid & (a.EP - 1), rg = tid / a.EP, nrg = nt / a.EP;
  const int64_t b = min(max(a.off ? a.off[s] : (int64_t)0, (int64_t)0), a.N);
  const int64_t h = min(max(a.off ? a.off[s + 1] : a.N, (int64_t)0), a.N);
  const int64_t r0 = b / a.run + s, r1 = h > b ? (h - 1) / a.run + s + 1 : r0;
  double p = 0.;
  int64_t c = 0, n = 0;
  if (e < a.E)
    for (int64_t r = r0 + rg; r < r1; r += nrg) {
      p += (double)a.part_p[r * a.E + e];
      c += a.part_c[r * a.E + e];
    }
  for (int64_t r = r0 + tid; r < r1; r += nt) n += a.part_n[r];
  n = block_sum(n, s_redi);
  s_p[tid] = p;
  s_c[tid] = c;
  __syncthreads();
  double l = 0.;
  if (tid < a.E) {
    for (int g = 1; g < nrg; ++g) {
      p += s_p[g * a.EP + tid];
      c += s_c[g * a.EP + tid];
    }
    const double inv = n > 0 ? 1. / (double)n : 0.;
    p *= inv;
    a.counts[s * a.E + tid] = c;
    a.mean_p[s * a.E + tid] = (float)p;
    l = (double)a.E * (double)c * inv / (double)a.K * p;
  }
  l = block_sum(l, s_red);
  if (tid == 0) {
    a.tokens[s] = n;
    a.seq_loss[s] = l;
    __threadfence();
    s_last = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0., zs = 0.;
  int64_t all = 0, used = 0;
  for (int64_t i = tid; i < a.S; i += nt) {
    sum += __hip_atomic_load(a.seq_loss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int64_t m = __hip_atomic_load(a.tokens + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    all += m;
    used += m > 0;
  }
  for (int64_t i = tid; i < a.runs; i += nt) zs += (double)a.part_z[i];
  sum = block_sum(sum, s_red);
  zs = block_sum(zs, s_red);
  all = block_sum(all, s_redi);
  used = block_sum(used, s_redi);
  if (tid == 0) {
    a.tokens[a.S] = all;
    a.tokens[a.S + 1] = used;
    *a.balance = (float)((double)a.bcoef * sum / (double)max(used, (int64_t)1));
    *a.z = (float)((double)a.zcoef * zs / (double)max(all, (int64_t)1));
    *a.ticket = 0u;
  }
}

// Tokens of a wave: enough waves for every SIMD to hold a few (16 tokens each below 65536 tokens), and at most 4096 of them.
int run_of(int64_t N) { return (int)std::max<int64_t>(16, ((N + 4095) / 4096 + 15) / 16 * 16); }

size_t al256b(size_t v) { return (v + 255) & ~(size_t)255; }
struct BalanceWs {
  int64_t runs, rows;
  size_t off_loss, off_p, off_c, off_n, off_z, total;
};
BalanceWs balance_ws(int64_t N, int64_t E, int64_t S) {
  BalanceWs w;
  w.runs = (N + run_of(N) - 1) / run_of(N);
  w.rows = w.runs + S;
  w.off_loss = 256;  // the ticket's line first
  w.off_p = w.off_loss + al256b((size_t)S * 8);
  w.off_c = w.off_p + al256b((size_t)w.rows * E * 4);
  w.off_n = w.off_c + al256b((size_t)w.rows * E * 4);
  w.off_z = w.off_n + al256b((size_t)w.rows * 4);
  w.total = w.off_z + al256b((size_t)w.runs * 4);
  return w;
}

int balance_check(const char* what, int64_t N, int64_t E, int64_t K, int64_t S) {
  const int64_t lim = INT32_MAX;
  if (N < 1 || N > lim || E < 1 || E > kMaxBalanceE || K < 1 || K > 32 || K > E || S < 1 || S > lim - 1)
    return fail_arg("%s: bad shape N=%lld E=%lld K=%lld S=%lld (need N, S >= 1, E <= %d, K <= min(E, 32))", what, (long long)N,
                    (long long)E, (long long)K, (long long)S, kMaxBalanceE);
  return 0;
}

#define MOE_BALANCE(KERNEL, name)                                                                                       \
  do {                                                                                                                  \
    const dim3 grid((unsigned)cdiv(runs, 4));                                                                           \
    if (E <= 8) MOE_LAUNCH(name, (KERNEL<8, 1>), grid, dim3(256), 0, s, a);                                             \
    else if (E <= 16) MOE_LAUNCH(name, (KERNEL<16, 1>), grid, dim3(256), 0, s, a);                                      \
    else if (E <= 32) MOE_LAUNCH(name, (KERNEL<16, 2>), grid, dim3(256), 0, s, a);                                      \
    else if (E <= 64) MOE_LAUNCH(name, (KERNEL<16, 4>), grid, dim3(256), 0, s, a);                                      \
    else if (E <= 128) MOE_LAUNCH(name, (KERNEL<16, 8>), grid, dim3(256), 0, s, a);                                     \
    else MOE_LAUNCH(name, (KERNEL<32, 8>), grid, dim3(256), 0, s, a);                                                   \
  } while (0)

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
  a.run = run_of(N);
  a.part_p = reinterpret_cast<float*>(ws + w.off_p);
  a.part_c = reinterpret_cast<int*>(ws + w.off_c);
  a.part_n = reinterpret_cast<int*>(ws + w.off_n);
  a.part_z = reinterpret_cast<float*>(ws + w.off_z);
  MOE_BALANCE(k_balance_fwd, "k_balance_fwd");
  if (int rc = check_launch("k_balance_fwd")) return rc;
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
  b.run = a.run;
  b.EP = 1;
  while (b.EP < E) b.EP *= 2;
  b.bcoef = balance_coef;
  b.zcoef = z_coef;
  b.counts = counts;
  b.tokens = tokens;
  b.mean_p = mean_prob;
  b.seq_loss = reinterpret_cast<double*>(ws + w.off_loss);
  b.balance = balance;
  b.z = z;
  b.ticket = reinterpret_cast<unsigned*>(ws);
  MOE_LAUNCH("k_balance_sum", k_balance_sum, dim3((unsigned)S), dim3(256), 0, s, b);
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
  a.run = run_of(N);
  a.counts = counts;
  a.tokens = tokens;
  a.grad_b = grad_balance;
  a.grad_z = grad_z;
  a.bcoef = balance_coef;
  a.zcoef = z_coef;
  a.dlogits = dlogits;
  const int64_t runs = (N + a.run - 1) / a.run;
  MOE_BALANCE(k_balance_bwd, "k_balance_bwd");
  return check_launch("moe_balance_bwd");
}

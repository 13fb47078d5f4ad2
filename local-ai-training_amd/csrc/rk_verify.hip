// Verification of drafted tokens against the target's probabilities, from given random numbers
// (gfx950): which nodes of a tree of drafts stand, and the token that follows the last one that
// does. The reference draws one token at a time, on the CPU (generate.py:180-197).
//
//   p_n, q_n = softmax of the target's and the drafter's logits at node n over the temperature,
//              without what lies below the k-th largest logit (equal ones stay)
//   from the root on, the children c of node n in their order, of token x:
//     c stands if u_c q(x) < p(x), and the walk goes on from it;
//     otherwise p <- max(p - q, 0) over its sum, and the next child is tried (p stays where that
//     sum is up to kNothing: only drafts that q does not hold come there, and it is rounding)
//   where no child stands: the first token whose cumulated p passes u_0 times its sum
// so that the tokens are distributed as the target's own. Without the drafter's logits q is 1 at
// the drafted token. At temperature 0 a child stands if its token is the target's first largest.
//
// Tokens are whole numbers, which no rounding may turn: of the V borders of a cumulated sum each
// would be off by the sum's error, and a drawn number falls between a border and its shadow with
// that probability. So probabilities and their sums are 64-bit numbers, with an exponential of
// their own (exp2_64) of a relative error of a few 2^-53.
#include "rk_common.h"
#include "rk_tree.h"

#include <math.h>

namespace rk {

constexpr int kStatThreads = 512;
constexpr int kWalkThreads = 1024;
constexpr int kSegments = 2048;  // of a row, whose sums a draw scans
constexpr int kExpSteps = 32;
constexpr double kNothing = 0x1p-40;

struct RowStat {
  double inv;   // 1 / the sum of the exponentials; NaN where the row is no distribution
  float most;   // the largest logit: p(v) = exp2((v - most) c) inv
  float floor;  // the k-th largest logit, or -inf
  int best;     // the first largest logit's index (temperature 0)
};

struct Verify {
  const void* logits;  // [B][N][V], strides lb, ln
  const void* drafts;  // the same of the drafter, or null
  int64_t lb, ln, db, dn, B, N, V;
  bool vec, dvec;      // rows can be read as vectors of four
  const int64_t* tokens;    // [B][N]
  const float* uniforms;    // [B][N]
  const int32_t* parents;   // [trees][N]
  int64_t tree_step;
  const int64_t* lengths;   // [B] or null
  double c;                 // log2(e) / temperature; 0: greedy
  int64_t top_k;            // 0: all
  RowStat* stats;           // [2][B][N]
  int64_t *path, *counts, *next;
};

// 2^y for y <= 0 (a little above it in rounding): y = n / 32 + r / ln 2, 2^(n / 32) from a table of
// 32, e^r by its series up to r^5 / 120 (|r| <= ln 2 / 64: the next term is below 2^-48.7 of the
// result, 2.2e-15). NaN gives 0: rows that hold one are noticed by their statistics.
__device__ __forceinline__ double exp2_64(double y, const double* table) {
  y = y >= -1100.0 ? y : -1100.0;
  const double n = __builtin_rint(y * kExpSteps);
  const int i = static_cast<int>(n);
  const double r = __builtin_fma(n, -1.0 / kExpSteps, y) * 0.69314718055994530942;
  double p = __builtin_fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_ldexp(table[i & (kExpSteps - 1)] * p, i >> 5);
}

// 2^((x - most) c): the difference first, which is exact (or far below the result's last bit).
__device__ __forceinline__ double scaled_exp(float x, float most, double c, const double* table) {
  return exp2_64((static_cast<double>(x) - static_cast<double>(most)) * c, table);
}

__device__ __forceinline__ void exp_table(double* table, int tid) {
  if (tid < kExpSteps) table[tid] = exp2(tid / static_cast<double>(kExpSteps));
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off /= 2) v = v + __shfl_xor(v, off);
  return v;
}

// Four logits from index i on, -inf past the row's end.
template <int DT>
__device__ __forceinline__ void load4(const void* row, int64_t i, int64_t V, bool vec,
                                      float (&x)[4]) {
  if (vec && i + 4 <= V) {
    if constexpr (DT == RK_F32) {
      load_vec16<RK_F32>(row, i, x);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + i);
      x[0] = __uint_as_float(w.x << 16);
      x[1] = __uint_as_float(w.x & 0xffff0000u);
      x[2] = __uint_as_float(w.y << 16);
      x[3] = __uint_as_float(w.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = i + e < V ? load_elem<DT>(row, i + e) : -INFINITY;
  }
}

// Whole numbers in the order of the floats; -0 is 0, NaN above all.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x == x ? k : 0xffffffffu;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The bin of hist in which the `want`-th largest lies (1: the largest), and how many lie above it.
// By the first wavefront; BINS is a multiple of 64.
template <int BINS>
__device__ __forceinline__ void find_bin(const int* hist, int want, int lane, int& bin,
                                         int& above) {
  constexpr int PER = BINS / 64;
  // lane l holds the bins from the top: BINS - 1 - PER l downwards
  int own = 0;
  for (int i = 0; i < PER; ++i) own += hist[BINS - 1 - (PER * lane + (i + lane) % PER)];
  int sum = own;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int v = __shfl_up(sum, off);
    if (lane >= off) sum += v;
  }
  const uint64_t enough = __ballot(sum >= want);
  const int at = enough ? static_cast<int>(__builtin_ctzll(enough)) : 63;
  int over = __shfl(sum - own, at);
  int i = 0;
  for (; i < PER - 1; ++i) {
    const int h = hist[BINS - 1 - (PER * at + i)];
    if (over + h >= want) break;
    over += h;
  }
  bin = BINS - 1 - (PER * at + i);
  above = over;
}

// grid (B * N, 1 or 2: target, drafter), 512 threads: a row's statistics.
template <int DT>
__global__ __launch_bounds__(kStatThreads) void verify_stats_kernel(Verify a) {
  constexpr int WAVES = kStatThreads / 64;
  __shared__ double table[kExpSteps];
  __shared__ int hist[2048];
  __shared__ uint64_t best[WAVES];
  __shared__ double sums[WAVES];
  __shared__ int box[2];
  const uint32_t un = static_cast<uint32_t>(a.N), ub = blockIdx.x / un;
  const int64_t b = ub, n = blockIdx.x - ub * un, V = a.V;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t len = a.lengths ? a.lengths[b] : a.N;
  len = len < a.N ? len : a.N;
  const int32_t* const parents = a.parents + b * a.tree_step;
  if (n >= len || parents[n] == kTreeOff) return;
  const bool drafter = blockIdx.y != 0;
  if (drafter) {  // only where the node has a child
    bool child = false;
    for (int64_t i = n + 1 + tid; i < len; i += kStatThreads) child |= parents[i] == n;
    if (!__syncthreads_or(child)) return;
  }
  const char* const base = static_cast<const char*>(drafter ? a.drafts : a.logits);
  const void* const row =
      base + (drafter ? b * a.db + n * a.dn : b * a.lb + n * a.ln) * (DT == RK_F32 ? 4 : 2);
  const bool vec = drafter ? a.dvec : a.vec;
  RowStat* const out = a.stats + (drafter ? a.B * a.N : 0) + b * a.N + n;
  constexpr int STEP = 4 * kStatThreads;

  if (a.c == 0.0) {  // the first largest
    uint64_t top = 0;
    for (int64_t i = 4 * tid; i < V; i += STEP) {
      float x[4];
      load4<DT>(row, i, V, vec, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t k = static_cast<uint64_t>(order_key(x[e])) << 32 |
                           (0xffffffffu - static_cast<uint32_t>(i + e));
        if (i + e < V) top = k > top ? k : top;
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off /= 2) {
      const uint64_t o = __shfl_xor(static_cast<unsigned long long>(top), off);
      top = o > top ? o : top;
    }
    if (lane == 0) best[wave] = top;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < WAVES; ++w) top = best[w] > top ? best[w] : top;
      out->best = static_cast<int>(0xffffffffu - static_cast<uint32_t>(top));
    }
    return;
  }

  exp_table(table, tid);
  float floor = -INFINITY;
  if (a.top_k > 0 && a.top_k < V) {
    // the k-th largest by its bits, 11 at a time from the top (a bf16 logit has 16)
    uint32_t prefix = 0;
    int want = static_cast<int>(a.top_k);
    constexpr int SHIFTS[3] = {21, 10, 0};
    constexpr int PASSES = DT == RK_F32 ? 3 : 2;
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int shift = SHIFTS[pass], high = pass == 0 ? 32 : SHIFTS[pass - 1];
      for (int i = tid; i < 2048; i += kStatThreads) hist[i] = 0;
      __syncthreads();
      for (int64_t i = 4 * tid; i < V; i += STEP) {
        float x[4];
        load4<DT>(row, i, V, vec, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = order_key(x[e]);
          if (i + e < V && (high == 32 || k >> (high & 31) == prefix))
            atomicAdd(&hist[(k >> shift) & 2047], 1);
        }
      }
      __syncthreads();
      if (wave == 0) {
        int bin, above;
        find_bin<2048>(hist, want, lane, bin, above);
        if (lane == 0) {
          box[0] = bin;
          box[1] = above;
        }
      }
      __syncthreads();
      const int bits = high - shift;
      prefix = prefix << bits | static_cast<uint32_t>(box[0] & ((1 << bits) - 1));
      want -= box[1];
    }
    floor = key_value(prefix << SHIFTS[PASSES - 1]);
  }
  __syncthreads();
  // a running maximum and sum of a thread's logits, then of the threads
  float m = -INFINITY;
  double s = 0.0;
  bool bad = false;
  for (int64_t i = 4 * tid; i < V; i += STEP) {
    float x[4];
    load4<DT>(row, i, V, vec, x);
    const float t = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    bad |= x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3];
    if (!(t >= floor)) continue;
    if (t > m) {
      if (m != -INFINITY) s = s * scaled_exp(m, t, a.c, table);
      m = t;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double v = scaled_exp(x[e], ref, a.c, table);
      s = s + (x[e] >= floor ? v : 0.0);
    }
  }
  bad |= m == INFINITY;
  float most = wave_max(m);
  if (lane == 0) sums[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) most = fmaxf(most, static_cast<float>(sums[w]));
  s = m == -INFINITY ? 0.0 : s * scaled_exp(m, most, a.c, table);
  s = wave_sum_f64(s);
  bad = __syncthreads_or(bad);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.0;
    for (int w = 0; w < WAVES; ++w) s = s + sums[w];
    out->most = most == -INFINITY ? 0.0f : most;
    out->inv = bad || !(s > 0.0) ? __longlong_as_double(0x7ff8000000000000ll) : 1.0 / s;
    out->floor = floor;
  }
}

// grid (B), 1024 threads: the walk and the draw. Every thread walks by itself, over what LDS holds
// of the nodes; the passes over a row (a residual's sum, a draw) are the workgroup's.
template <int DT, bool DRAFTS>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(Verify a) {
  constexpr int WAVES = kWalkThreads / 64;
  __shared__ double table[kExpSteps], seg[kSegments], P[kTreeNodes], Q[kTreeNodes],
      scale[kTreeNodes];
  __shared__ float U[kTreeNodes];
  __shared__ int par[kTreeNodes], tok[kTreeNodes], rejected[kTreeNodes], way[kTreeNodes];
  const int64_t b = blockIdx.x, V = a.V;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t len = a.lengths ? a.lengths[b] : a.N;
  const int n = static_cast<int>(len < a.N ? len : a.N);
  const int32_t* const parents = a.parents + b * a.tree_step;
  const RowStat* const stats = a.stats + b * a.N;
  const RowStat* const dstats = stats + a.B * a.N;
  const bool greedy = a.c == 0.0;
  if (n <= 0 || parents[0] != -1) {
    for (int64_t i = tid; i < a.N; i += kWalkThreads) a.path[b * a.N + i] = -1;
    if (tid == 0) {
      a.counts[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  const auto row_of = [&](int node, bool drafter) -> const void* {
    const char* const base = static_cast<const char*>(drafter ? a.drafts : a.logits);
    return base + (drafter ? b * a.db + node * a.dn : b * a.lb + node * a.ln) *
                      (DT == RK_F32 ? 4 : 2);
  };
  const auto chance = [&](float v, const RowStat& st) {
    const double e = scaled_exp(v, st.most, a.c, table);
    return v >= st.floor ? e * st.inv : 0.0 * st.inv;
  };
  exp_table(table, tid);
  __syncthreads();
  if (tid < n) {
    const int p = parents[tid];
    const int64_t x = a.tokens[b * a.N + tid];
    const bool ok = x >= 0 && x < V;
    par[tid] = p;
    tok[tid] = ok ? static_cast<int>(x) : -1;
    way[tid] = 0;
    U[tid] = greedy ? 0.0f : a.uniforms[b * a.N + tid];
    P[tid] = Q[tid] = 0.0;
    if (!greedy && p >= 0 && p < tid && ok) {
      P[tid] = chance(load_elem<DT>(row_of(p, false), x), stats[p]);
      Q[tid] = 1.0;
      if constexpr (DRAFTS) Q[tid] = chance(load_elem<DT>(row_of(p, true), x), dstats[p]);
    }
  }
  __syncthreads();

  const int64_t per = (V + 256 * kSegments - 1) / (256 * kSegments);  // 256s of a segment
  const int segments = static_cast<int>((V + 256 * per - 1) / (256 * per));
  int cur = 0, k = 0, count = 1;
  // what k rejected children of `cur` leave of p at four tokens from i on, the last one not
  // normalized
  const auto left4 = [&](const RowStat& st, const RowStat& ds, int64_t i, double (&r)[4]) {
    float x[4];
    load4<DT>(row_of(cur, false), i, V, a.vec, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = chance(x[e], st);
    if constexpr (DRAFTS) {
      if (k > 0) {
        float y[4];
        load4<DT>(row_of(cur, true), i, V, a.dvec, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double q = chance(y[e], ds);
          double t = r[e];
          for (int j = 0; j < k; ++j) {
            t = t - q;
            t = (t < 0.0 ? 0.0 : t) * (j + 1 < k ? scale[j] : 1.0);
          }
          r[e] = t;
        }
      }
    } else {
      for (int j = 0; j < k; ++j) {
        const int64_t x0 = tok[rejected[j]] - i;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = x0 == e ? 0.0 : r[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = i + e < V ? r[e] : 0.0;
  };
  // the segments' sums of that, and their sum
  const auto pass = [&]() {
    const RowStat st = stats[cur], ds = DRAFTS && k > 0 ? dstats[cur] : st;
    __syncthreads();
    for (int s = wave; s < segments; s += WAVES) {
      double sum = 0.0;
      for (int64_t u = 0; u < per; ++u) {
        const int64_t i = (s * per + u) * 256 + 4 * lane;
        double r[4];
        left4(st, ds, i, r);
        sum = sum + ((r[0] + r[1]) + (r[2] + r[3]));
      }
      sum = wave_sum_f64(sum);
      if (lane == 0) seg[s] = sum;
    }
    __syncthreads();
    double total = 0.0;
    for (int s = lane; s < segments; s += 64) total = total + seg[s];
    return wave_sum_f64(total);
  };

  bool pending = false;  // the last rejected child's residual has no sum yet
  double rest = 1.0;     // without a drafter: what the rejected tokens left
  int pick = greedy ? stats[0].best : 0;
  for (int i = 1; i < n; ++i) {
    if (par[i] != cur) continue;
    bool stands;
    if (greedy) {
      stands = tok[i] == pick;
    } else if constexpr (DRAFTS) {
      if (pending) {
        const double z = pass();
        if (z <= kNothing) {
          --k;
        } else {
          if (tid == 0) scale[k - 1] = 1.0 / z;
          __syncthreads();
        }
        pending = false;
      }
      double t = P[i];
      for (int j = 0; j < k; ++j) {
        t = t - Q[i];
        t = (t < 0.0 ? 0.0 : t) * scale[j];
      }
      stands = U[i] * Q[i] < t;
    } else {
      double t = P[i];
      for (int j = 0; j < k; ++j) t = tok[rejected[j]] == tok[i] ? 0.0 : t;
      stands = U[i] * rest < t;
      if (!stands && rest - t <= kNothing * rest) continue;
      if (!stands) rest = rest - t;
    }
    if (stands) {
      cur = i;
      k = 0;
      rest = 1.0;
      pending = false;
      if (tid == 0) way[count] = i;
      ++count;
      if (greedy) pick = stats[cur].best;
    } else if (!greedy) {
      __syncthreads();
      if (tid == 0) rejected[k] = i;
      __syncthreads();
      ++k;
      pending = true;
    }
  }
  __syncthreads();
  for (int64_t i = tid; i < a.N; i += kWalkThreads) a.path[b * a.N + i] = i < count ? way[i] : -1;
  if (tid == 0) a.counts[b] = count;
  if (greedy) {
    if (tid == 0) a.next[b] = pick;
    return;
  }
  double total = pass();
  if (DRAFTS && k > 0 && total <= kNothing) {
    --k;
    total = pass();
  }
  if (wave != 0) return;
  if (!(total > 0.0)) {
    if (lane == 0) a.next[b] = -1;
    return;
  }
  // the segment, then the token in it
  const int each = (segments + 63) / 64;
  double own = 0.0;
  for (int s = each * lane; s < each * (lane + 1) && s < segments; ++s) own = own + seg[s];
  double sum = own;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const double v = __shfl_up(sum, off);
    if (lane >= off) sum = sum + v;
  }
  double bound = U[0] * __shfl(sum, 63);
  // (where rounding lets no sum pass the bound: the last token of any weight)
  const uint64_t over = __ballot(sum > bound), some = __ballot(own > 0.0);
  const int at = over ? static_cast<int>(__builtin_ctzll(over))
                      : 63 - static_cast<int>(__builtin_clzll(some | 1));
  double before = __shfl(sum, at > 0 ? at - 1 : 0);
  if (at == 0) before = 0.0;
  int s = each * at;
  bool found = false;
  for (int u = each * at; u < each * (at + 1) && u < segments && !found; ++u) {
    if (seg[u] > 0.0) s = u;
    found = before + seg[u] > bound;
    if (!found) before = before + seg[u];
  }
  if (!found) bound = INFINITY;
  const RowStat st = stats[cur], ds = DRAFTS && k > 0 ? dstats[cur] : st;
  int64_t token = -1, last = -1;
  for (int64_t u = 0; u < per && token < 0; ++u) {
    const int64_t i = (s * per + u) * 256 + 4 * lane;
    double r[4];
    left4(st, ds, i, r);
    const double mine = (r[0] + r[1]) + (r[2] + r[3]);
    double upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const double v = __shfl_up(upto, off);
      if (lane >= off) upto = upto + v;
    }
    // the first of this lane's tokens that passes the bound, and the last of any weight
    double cum = before + (upto - mine);
    int hit = 4, weighty = -1;
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const double c = e == 0   ? cum + r[0]
                       : e == 1 ? cum + (r[0] + r[1])
                       : e == 2 ? cum + (r[0] + r[1] + r[2])
                                : before + upto;
      if (c > bound && r[e] > 0.0) hit = e;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r[e] > 0.0) weighty = e;
    const uint64_t hits = __ballot(hit < 4), weights = __ballot(weighty >= 0);
    if (hits) {
      const int from = static_cast<int>(__builtin_ctzll(hits));
      token = __shfl(i + hit, from);
    }
    if (weights) last = __shfl(i + weighty, 63 - static_cast<int>(__builtin_clzll(weights)));
    before = before + __shfl(upto, 63);
  }
  if (lane == 0) a.next[b] = token >= 0 ? token : last;
}

}  // namespace rk

using namespace rk;

extern "C" int64_t rk_verify_drafts_work(const rk_verify_drafts_args* args) {
  if (!args || args->B <= 0 || args->N <= 0) return 0;
  return 2 * args->B * args->N * static_cast<int64_t>(sizeof(RowStat));
}

extern "C" int rk_verify_drafts(const rk_verify_drafts_args* args, void* work,
                                int64_t work_bytes, void* stream) {
  clear_error();
  if (!args) return fail(RK_ERR_ARG, "null arguments");
  const rk_verify_drafts_args& p = *args;
  if (p.B < 0 || p.N < 0 || p.V < 0 || p.top_k < 0) return fail(RK_ERR_ARG, "negative size");
  if (p.N > kTreeNodes) return fail(RK_ERR_UNSUPPORTED, "a tree has at most %d nodes", kTreeNodes);
  if (p.dtype != RK_F32 && p.dtype != RK_BF16)
    return fail(RK_ERR_ARG, "logits are float32 or bfloat16");
  if (p.trees != 1 && p.trees != p.B) return fail(RK_ERR_ARG, "one tree, or one per sequence");
  if (!(p.temperature >= 0.0) || !(p.temperature < INFINITY))
    return fail(RK_ERR_ARG, "temperature must be finite and not negative");
  if (p.temperature > 0.0 && !(p.temperature >= 1e-6))
    return fail(RK_ERR_UNSUPPORTED, "a temperature below 1e-6 (0: greedy)");
  if (p.B == 0 || p.N == 0) return RK_OK;
  if (p.V == 0) return fail(RK_ERR_ARG, "an empty vocabulary");
  const bool greedy = p.temperature == 0.0;
  if (!p.logits || !p.tokens || !p.parents || !p.path || !p.counts || !p.next ||
      (!greedy && !p.uniforms))
    return fail(RK_ERR_ARG, "null pointer");
  const int64_t size = dtype_size(p.dtype);
  const int64_t strides[] = {p.lb, p.ln, p.db, p.dn};
  for (int64_t st : strides)
    if (st < 0) return fail(RK_ERR_ARG, "negative stride");
  if (p.V >= (int64_t{1} << 31) - (int64_t{1} << 20) || p.B * p.N >= (int64_t{1} << 23))
    return fail(RK_ERR_UNSUPPORTED, "too many logits for one launch");
  if (!work || !aligned16(work) || work_bytes < rk_verify_drafts_work(args))
    return fail(RK_ERR_ARG, "verification workspace too small");
  const auto vec = [&](const void* at, int64_t sb, int64_t sn) {
    return reinterpret_cast<uintptr_t>(at) % (4 * size) == 0 && sb % 4 == 0 && sn % 4 == 0;
  };
  const bool drafts = p.drafts && !greedy;
  const Verify a{p.logits, drafts ? p.drafts : nullptr, p.lb, p.ln, p.db, p.dn, p.B, p.N, p.V,
                 vec(p.logits, p.lb, p.ln), vec(p.drafts, p.db, p.dn), p.tokens, p.uniforms,
                 p.parents, p.trees > 1 ? p.N : 0, p.lengths,
                 greedy ? 0.0 : 1.4426950408889634074 / p.temperature, p.top_k,
                 static_cast<RowStat*>(work), p.path, p.counts, p.next};
  hipStream_t st = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(p.B * p.N), drafts ? 2 : 1);
  if (p.dtype == RK_F32) {
    verify_stats_kernel<RK_F32><<<grid, kStatThreads, 0, st>>>(a);
    if (drafts) verify_walk_kernel<RK_F32, true><<<p.B, kWalkThreads, 0, st>>>(a);
    else verify_walk_kernel<RK_F32, false><<<p.B, kWalkThreads, 0, st>>>(a);
  } else {
    verify_stats_kernel<RK_BF16><<<grid, kStatThreads, 0, st>>>(a);
    if (drafts) verify_walk_kernel<RK_BF16, true><<<p.B, kWalkThreads, 0, st>>>(a);
    else verify_walk_kernel<RK_BF16, false><<<p.B, kWalkThreads, 0, st>>>(a);
  }
  return launch_status("verify_drafts");
}

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
// their own (scaled_exp) of a relative error of 2.3e-15, some 2^-48.6: kNothing is 400 times that.
#include "rk_common.h"
#include "rk_tree.h"

#include <float.h>
#include <math.h>

#include <type_traits>

namespace rk {

constexpr int kPassThreads = 256;
constexpr int kSegments = 2048;    // of a row at most, whose sums a draw scans
constexpr int kCandidates = 2048;  // of a row, among which the k-th largest is sought
constexpr int kExpSteps = 32;
constexpr double kNothing = 0x1p-40;

struct RowStat {
  double inv;   // 1 / the sum of the exponentials; NaN where the row is no distribution (of a part of
                // a row: the sum itself)
  float most;   // the largest logit: p(v) = exp2((v - most) c) inv
  float floor;  // logits below it have no probability
  int best;     // the first largest logit's index (temperature 0)
};

// Where a sequence's walk stands between two launches.
struct WalkState {
  double scale[kTreeNodes], P[kTreeNodes], Q[kTreeNodes], seg[kSegments], rest;
  float top[kSegments];
  int rejected[kTreeNodes], way[kTreeNodes];
  RowStat stat[2];  // of the row of `cur`: the target's, the drafter's
  int cur, k, count, i, pending;
  int bare;     // the row of `cur` has no statistics
  int request;  // a pass over it is wanted (0: the walk has ended)
};

struct Verify {
  const void* logits;  // [B][N][V], strides lb, ln
  const void* drafts;  // the same of the drafter, or null
  int64_t lb, ln, db, dn, B, N, V;
  const int64_t* tokens;    // [B][N]
  const float* uniforms;    // [B][N]
  const int32_t* parents;   // [trees][N]
  int64_t tree_step;
  const int64_t* lengths;   // [B] or null
  double c;                 // log2(e) / temperature; 0: greedy
  int64_t top_k;            // 0: all
  RowStat* stats;           // [2][B][N], by the first launch of the walk from
  RowStat* parts_of;        // [2][B][N][parts], the statistics of the rows' parts
  int64_t parts, part;      // part: logits of each
  WalkState* states;        // [B], or null: one launch walks to the end
  int64_t *path, *counts, *next;
};

// 2^((x - from) c), c32 = 32 c, for (x - from) c in -1000 .. 1000 (the caller sees to that). In 32nds:
// 32 (x - from) c = n + f, |f| <= 1/2, n in the low word of the sum with 1.5 2^52; 2^(n / 32) from a
// table of 32, whose reads meet no bank twice; e^(f ln 2 / 32) by its series to the fifth power (what it
// leaves out is at most 2.3e-15 of the result; without the fifth, 1.3e-12, more than kNothing). The difference comes first: it is exact, or rounded
// far below the result's last bit, where the products' difference is not.
__device__ __forceinline__ double scaled_exp(float x, double from, double c32, const double* table) {
  constexpr double kMagic = 6755399441055744.0;
  constexpr double a1 = 0.69314718055994530942 / kExpSteps;
  constexpr double a2 = a1 * a1 / 2.0, a3 = a2 * a1 / 3.0, a4 = a3 * a1 / 4.0;
  constexpr double a5 = a4 * a1 / 5.0;
  const double d = static_cast<double>(x) - from;
  const double t = __builtin_fma(d, c32, kMagic);
  const int n = static_cast<int>(__builtin_bit_cast(uint64_t, t));
  const double f = __builtin_fma(d, c32, kMagic - t);
  double p = __builtin_fma(f, a5, a4);
  p = __builtin_fma(p, f, a3);
  p = __builtin_fma(p, f, a2);
  p = __builtin_fma(p, f, a1);
  p = __builtin_fma(p, f, 1.0);
  p = p * table[n & (kExpSteps - 1)];
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t high = static_cast<uint32_t>(bits >> 32) +
                        (static_cast<uint32_t>(n & ~(kExpSteps - 1)) << 15);
  return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 |
                                        static_cast<uint32_t>(bits));
}
// The least logit that scaled_exp takes below `most`, rounded upwards.
__device__ __forceinline__ float exp_floor(float most, double c) {
  const float f = static_cast<float>(static_cast<double>(most) - 1000.0 / c);
  const bool low = (static_cast<double>(most) - static_cast<double>(f)) * c > 1000.0;
  return !(f >= -FLT_MAX) ? -FLT_MAX : low ? nextafterf(f, INFINITY) : f;
}

__device__ __forceinline__ void exp_table(double* table, int tid) {
  if (tid < kExpSteps) table[tid] = exp2(tid / static_cast<double>(kExpSteps));
}

// v + v[lane ^ 32], ^ 16, .. ^ 1, each half of the bits moved as in wave_butterfly.
__device__ __forceinline__ double wave_sum_f64(double v) {
  const auto join = [](uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
  };
  const auto low = [](double x) { return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, x)); };
  const auto high = [](double x) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, x) >> 32);
  };
  {
    const auto l = __builtin_amdgcn_permlane32_swap(low(v), low(v), false, false);
    const auto h = __builtin_amdgcn_permlane32_swap(high(v), high(v), false, false);
    v = join(l[0], h[0]) + join(l[1], h[1]);
  }
  {
    const auto l = __builtin_amdgcn_permlane16_swap(low(v), low(v), false, false);
    const auto h = __builtin_amdgcn_permlane16_swap(high(v), high(v), false, false);
    v = join(l[0], h[0]) + join(l[1], h[1]);
  }
  v = v + join(dpp_u32<0x128>(low(v)), dpp_u32<0x128>(high(v)));
  v = v + join(dpp_u32<0x141>(dpp_u32<0x1b>(low(v))), dpp_u32<0x141>(dpp_u32<0x1b>(high(v))));
  v = v + join(dpp_u32<0x4e>(low(v)), dpp_u32<0x4e>(high(v)));
  v = v + join(dpp_u32<0xb1>(low(v)), dpp_u32<0xb1>(high(v)));
  return v;
}

// A 16-byte piece of logits from index i on, -inf past the row's end. Rows lie at any multiple of
// their element (an odd vocabulary), which 16-byte loads of global memory allow.
template <int DT>
__device__ __forceinline__ void load_piece(const void* row, int64_t i, int64_t V,
                                           float (&x)[Vec<DT>::N]) {
  using E = typename Vec<DT>::Elem;
  const E* const at = static_cast<const E*>(row) + i;
  if (i + Vec<DT>::N <= V) {
    uint4 w;
    __builtin_memcpy(&w, at, 16);
    widen_vec16<DT>(w, x);
  } else {
#pragma unroll
    for (int e = 0; e < Vec<DT>::N; ++e) x[e] = i + e < V ? load_elem<DT>(row, i + e) : -INFINITY;
  }
}

// f(x, i) for a thread's 16-byte pieces x of a row, at logits first, first + step, .., UNROLL loads in
// flight. Pieces past the row's end are -inf.
template <int DT, int UNROLL, class F>
__device__ __forceinline__ void each_piece(const void* row, int64_t first, int64_t step, int64_t V,
                                           const F& f) {
  constexpr int VN = Vec<DT>::N;
  const auto* const base = static_cast<const typename Vec<DT>::Elem*>(row);
  const int64_t whole = V / VN * VN;
#pragma unroll 1
  for (int64_t i = first; i < whole; i += UNROLL * step) {
    uint4 w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      __builtin_memcpy(&w[u], base + (i + u * step < whole ? i + u * step : i), 16);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float x[VN];
      widen_vec16<DT>(w[u], x);
      if (i + u * step >= whole) {
#pragma unroll
        for (int e = 0; e < VN; ++e) x[e] = -INFINITY;
      }
      f(x, i + u * step < whole ? i + u * step : V);
    }
  }
  if (whole < V && whole % step == first) {
    float x[VN];
    load_piece<DT>(row, whole, V, x);
    f(x, whole);
  }
}

template <int DT>
__device__ __forceinline__ const void* row_at(const Verify& a, bool drafter, int64_t b, int64_t n) {
  const char* const base = static_cast<const char*>(drafter ? a.drafts : a.logits);
  return base + (drafter ? b * a.db + n * a.dn : b * a.lb + n * a.ln) * (DT == RK_F32 ? 4 : 2);
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

constexpr int kBins = 2048;

__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int u = __shfl_up(v, off);
    if (lane >= off) v += u;
  }
  return v;
}
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const double u = __shfl_up(v, off);
    if (lane >= off) v = v + u;
  }
  return v;
}

// The bin of hist in which the `want`-th largest lies (1: the largest; the last bin with any if
// there are fewer), and how many lie above it. By one wavefront.
__device__ __forceinline__ void find_bin(const int* hist, int want, int lane, int& bin,
                                         int& above) {
  constexpr int PER = kBins / 64;
  // lane l takes the bins kBins - 1 - PER l downwards, then each of one lane's bins has a lane
  int own = 0;
#pragma unroll 8
  for (int i = 0; i < PER; ++i) own += hist[kBins - 1 - (PER * lane + (i + lane) % PER)];
  const int sum = wave_scan(own, lane);
  const uint64_t enough = __ballot(sum >= want);
  const int at = enough ? static_cast<int>(__builtin_ctzll(enough)) : 63;
  const int over = __shfl(sum - own, at);
  const int one = lane < PER ? hist[kBins - 1 - (PER * at + lane)] : 0;
  const int part = wave_scan(one, lane);
  const uint64_t hit = __ballot(lane < PER && over + part >= want);
  const int u = hit ? static_cast<int>(__builtin_ctzll(hit)) : PER - 1;
  bin = kBins - 1 - (PER * at + u);
  above = over + __shfl(part - one, u);
}

// Without the k-th largest to find, a row whose node has no child is only drawn from, for which the
// pass over it is enough.
__device__ __forceinline__ bool all_rows(const Verify& a) { return a.top_k > 0 && a.top_k < a.V; }

enum { kGreedy, kTopK, kAll };  // what a row's statistics are for

// grid (B * N * parts, 1 or 2: target, drafter): a row's statistics, or a part's. A row's parts are
// neighbours: all rows' first parts one after the other, a power of two of bytes apart, took 101 us
// where this took 65, 70 with the exponential's fifth power (512 rows of 131072 bf16 logits that are
// looked at: 134 MB and 67 million 64-bit exponentials, whose instructions take 47 us to issue). Top-k rows: 25 us for 32 MB, the bins and the candidates' ranks.
template <int DT, int kStatThreads, int MODE>
__global__ __launch_bounds__(kStatThreads) void verify_stats_kernel(Verify a) {
  constexpr int WAVES = kStatThreads / 64, VN = Vec<DT>::N, STEP = VN * kStatThreads;
  __shared__ double table[kExpSteps];
  __shared__ int hist[MODE == kTopK ? kBins : 1];
  __shared__ __attribute__((aligned(16))) uint32_t list[MODE == kTopK ? kCandidates : 1];
  __shared__ uint64_t best[WAVES];
  __shared__ double sums[WAVES], ranked[kStatThreads];
  __shared__ int box[3];
  const uint32_t un = static_cast<uint32_t>(a.N), up = static_cast<uint32_t>(a.parts);
  const uint32_t at = blockIdx.x / up, p = blockIdx.x - at * up, ub = at / un;
  const int64_t b = ub, n = at - ub * un, skip = p * a.part;
  const int64_t V = a.V - skip < a.part ? a.V - skip : a.part;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool drafter = blockIdx.y != 0;
  const void* const row = static_cast<const typename Vec<DT>::Elem*>(row_at<DT>(a, drafter, b, n)) +
                          skip;
  float ref = load_elem<DT>(row, 0);
  int64_t len = a.lengths ? a.lengths[b] : a.N;
  len = len < a.N ? len : a.N;
  const int32_t* const parents = a.parents + b * a.tree_step;
  if (n >= len || parents[n] == kTreeOff) return;
  if (drafter || MODE == kAll) {  // only where the node has a child
    bool child = false;
    for (int64_t i = n + 1 + tid; i < len; i += kStatThreads) child |= parents[i] == n;
    if (!__syncthreads_or(child)) return;
  }
  RowStat* const out =
      a.parts_of + ((drafter ? a.B * a.N : 0) + b * a.N + n) * a.parts + p;

  if constexpr (MODE == kGreedy) {  // the first largest
    uint64_t top = 0;
    each_piece<DT, 4>(row, VN * tid, STEP, V, [&](const float (&x)[VN], int64_t i) {
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const uint64_t k = static_cast<uint64_t>(order_key(x[e])) << 32 |
                           (0xffffffffu - static_cast<uint32_t>(i + e));
        if (i + e < V) top = k > top ? k : top;
      }
    });
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
  const double c32 = a.c * kExpSteps;
  float m = -INFINITY;  // of this thread's logits
  bool bad = false;
  const auto note = [&](const float (&x)[VN]) {
#pragma unroll
    for (int e = 0; e < VN; e += 2) {
      m = fmaxf(m, fmaxf(x[e], x[e + 1]));
      bad |= __builtin_isunordered(x[e], x[e + 1]);
    }
  };
  const auto block_max = [&](float v) {
    v = wave_max(v);
    __syncthreads();
    if (lane == 0) sums[wave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v = fmaxf(v, static_cast<float>(sums[w]));
    return v;
  };
  const auto block_sum = [&](double v) {
    v = wave_sum_f64(v);
    __syncthreads();
    if (lane == 0) sums[wave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < WAVES; ++w) v = v + sums[w];
    return v;
  };
  float most, floor;
  double s = 0.0;
  if constexpr (MODE == kTopK) {
    each_piece<DT, 4>(row, VN * tid, STEP, V, [&](const float (&x)[VN], int64_t) { note(x); });
    most = block_max(m);
    const float least = -block_max(m > -INFINITY ? -m : -INFINITY);  // of the threads' largest
    const auto clear = [&] {
      __syncthreads();
      for (int i = tid; i < kBins; i += kStatThreads) hist[i] = 0;
      if (tid == 0) box[2] = 0;
      __syncthreads();
    };
    int want = static_cast<int>(a.top_k);
    const auto find = [&] {
      __syncthreads();
      if (wave == 0) {
        int bin, above;
        find_bin(hist, want, lane, bin, above);
        if (lane == 0) {
          box[0] = bin;
          box[1] = above;
        }
      }
      __syncthreads();
    };
    // The k-th largest of the threads' largest bounds the row's from below. Bins of equal width between
    // the largest and the least of them say where it lies; what lies below its bin need not be looked
    // at again. (A difference and a product of floats keep the order.)
    const float width = (kBins - 1) / (most - least);
    float bound = INFINITY;  // in bins below the largest
    clear();
    if (want <= kStatThreads && width < FLT_MAX && width > 0.0f) {
      const float at = (most - m) * width;
      atomicAdd(&hist[kBins - 1 - (at < kBins - 1 ? static_cast<int>(at) : kBins - 1)], 1);
      find();
      // (the last bin holds threads without a logit too)
      if (box[0] > 0) bound = static_cast<float>(kBins - box[0]);
    }
    // the candidates, in any order
    each_piece<DT, 16 / VN>(row, VN * tid, STEP, V, [&](const float (&x)[VN], int64_t i) {
      float t = x[0];
#pragma unroll
      for (int e = 1; e < VN; ++e) t = fmaxf(t, x[e]);
      if (bound != INFINITY && !__any((most - t) * width < bound)) return;
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const bool mine = i + e < V && (bound == INFINITY || (most - x[e]) * width < bound);
        const uint64_t some = __ballot(mine);
        if (some) {  // one addition for a wavefront's
          const int before = __builtin_popcountll(some & ((1ull << lane) - 1));
          int at = 0;
          if (mine && before == 0) at = atomicAdd(&box[2], __builtin_popcountll(some));
          at = __shfl(at, static_cast<int>(__builtin_ctzll(some))) + before;
          if (mine && at < kCandidates) list[at] = order_key(x[e]);
        }
      }
    });
    __syncthreads();
    const int found = box[2];
    if (found <= kStatThreads) {
      // each one's rank; the exponentials of those that stay by their ranks (equal ones are equal),
      // so that their sum has an order
      const uint32_t key = tid < found ? list[tid] : 0;
      int above = 0, same = 0;
      for (int u = 0; u < found; u += 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(list + u);
        const uint32_t k4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          above += u + e < found && k4[e] > key;
          same += u + e < tid && k4[e] == key;
        }
      }
      if (tid == 0) box[0] = 0;
      __syncthreads();
      const bool stays = tid < found && above < want;
      const float x = key_value(key);
      if (stays) {
        ranked[above + same] =
            x >= exp_floor(most, a.c) ? scaled_exp(x, most, c32, table) : 0.0;
        atomicMax(&box[0], above + same + 1);
        if (above + same == want - 1) box[1] = static_cast<int>(key);
      }
      __syncthreads();
      floor = fmaxf(key_value(static_cast<uint32_t>(box[1])), exp_floor(most, a.c));
      s = tid < box[0] ? ranked[tid] : 0.0;
    } else {
      // its bits, 11 at a time from the top (a bf16 logit has 16), among them or over the row again
      uint32_t prefix = 0;
      constexpr int SHIFTS[3] = {21, 10, 0};
      constexpr int PASSES = DT == RK_F32 ? 3 : 2;
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        const int shift = SHIFTS[pass], high = pass == 0 ? 32 : SHIFTS[pass - 1];
        const auto count = [&](uint32_t k) {
          if (high == 32 || k >> (high & 31) == prefix) atomicAdd(&hist[(k >> shift) & 2047], 1);
        };
        clear();
        if (found <= kCandidates) {
          for (int i = tid; i < found; i += kStatThreads) count(list[i]);
        } else {
          each_piece<DT, 2>(row, VN * tid, STEP, V, [&](const float (&x)[VN], int64_t i) {
#pragma unroll
            for (int e = 0; e < VN; ++e)
              if (i + e < V) count(order_key(x[e]));
          });
        }
        find();
        const int bits = high - shift;
        prefix = prefix << bits | static_cast<uint32_t>(box[0] & ((1 << bits) - 1));
        want -= box[1];
      }
      floor = fmaxf(key_value(prefix << SHIFTS[PASSES - 1]), exp_floor(most, a.c));
      const double ref = most;
      each_piece<DT, 2>(row, VN * tid, STEP, V, [&](const float (&x)[VN], int64_t) {
#pragma unroll
        for (int e = 0; e < VN; ++e)
          if (x[e] >= floor) s = s + scaled_exp(x[e], ref, c32, table);
      });
    }
    s = block_sum(s);
  } else {
    // One pass, relative to the row's first logit: 64-bit exponentials leave room for others that
    // lie up to 2^900 above it. Where that is not enough, another one relative to the largest.
    // (Logits 2^1000 below the reference are taken as that, which no sum shows.)
    __syncthreads();
    ref = fabsf(ref) <= FLT_MAX ? ref : 0.0f;
    double apart = 0.0;
#pragma unroll 1
    for (bool again = true; again;) {
      const float low = exp_floor(ref, a.c);
      const double from = ref;
      s = 0.0;
      each_piece<DT, 16 / VN>(row, VN * tid, STEP, V, [&](const float (&x)[VN], int64_t) {
        double v[VN];
        note(x);
#pragma unroll
        for (int e = 0; e < VN; ++e)
          v[e] = scaled_exp(__builtin_amdgcn_fmed3f(x[e], low, INFINITY), from, c32, table);
#pragma unroll
        for (int w = VN / 2; w > 0; w /= 2)
#pragma unroll
          for (int e = 0; e < w; ++e) v[e] = v[e] + v[e + w];
        s = s + v[0];
      });
      most = block_max(m);
      apart = (static_cast<double>(ref) - static_cast<double>(most)) * a.c;
      again = !(fabs(apart) <= 900.0) && ref != most && fabsf(most) <= FLT_MAX;
      if (again) ref = most;
    }
    if (!(fabsf(most) <= FLT_MAX)) ref = most, s = 0.0;  // no distribution
    floor = exp_floor(most, a.c);
    s = block_sum(s);
    if (ref != most) s = apart > 0.0 ? s / scaled_exp(most, ref, c32, table)
                                     : s * scaled_exp(ref, most, c32, table);
  }
  bad = __syncthreads_or(bad || most == INFINITY);
  if (tid == 0) {
    out->most = most;
    out->inv = bad ? __longlong_as_double(0x7ff8000000000000ll) : s;
    out->floor = floor;
  }
}

// A row's statistics from its parts'.
__device__ __forceinline__ RowStat whole_row(const RowStat* parts, int64_t n, double c,
                                             const double* table) {
  RowStat st = parts[0];
  double s = st.inv;
  if (n > 1) {
    for (int64_t p = 1; p < n; ++p) st.most = fmaxf(st.most, parts[p].most);
    st.floor = exp_floor(st.most, c);
    s = 0.0;
    for (int64_t p = 0; p < n; ++p) {
      const double t = scaled_exp(parts[p].most, st.most, c * kExpSteps, table);
      s = s + parts[p].inv * (parts[p].most >= st.floor ? t : 0.0);
    }
  }
  st.inv = s > 0.0 ? 1.0 / s : __longlong_as_double(0x7ff8000000000000ll);
  return st;
}

__device__ __forceinline__ double chance(float v, const RowStat& st, double c32,
                                         const double* table) {
  const double e = scaled_exp(v, st.most, c32, table);
  return (v >= st.floor ? e : 0.0) * st.inv;
}

// What k rejected children of a node leave of its distribution, at four tokens, the last one not
// normalized: the children's tokens (no drafter) or the earlier residuals' 1 / sums.
template <int DT, bool DRAFTS>
struct Residual {
  const void *row, *drow;
  RowStat st, ds;
  int64_t V;
  double c32;
  int k;
  bool few;  // k-th largest logits
  const double *scale, *table;
  const int* rejected;

  __device__ __forceinline__ Residual(const Verify& a, int64_t b, int cur, int k, const RowStat& st,
                                      const RowStat& ds, const double* scale, const int* rejected,
                                      const double* table)
      : row(row_at<DT>(a, false, b, cur)), drow(DRAFTS ? row_at<DT>(a, true, b, cur) : nullptr),
        st(st), ds(ds), V(a.V), c32(a.c * kExpSteps), k(k), few(all_rows(a)), scale(scale),
        table(table), rejected(rejected) {}

  __device__ __forceinline__ void load(const void* from, int64_t i, float (&x)[4]) const {
    const auto* const at = static_cast<const typename Vec<DT>::Elem*>(from) + i;
    if (i + 4 <= V) {
      if constexpr (DT == RK_F32) {
        __builtin_memcpy(x, at, 16);
      } else {
        uint2 w;
        __builtin_memcpy(&w, at, 8);
        x[0] = __uint_as_float(w.x << 16);
        x[1] = __uint_as_float(w.x & 0xffff0000u);
        x[2] = __uint_as_float(w.y << 16);
        x[3] = __uint_as_float(w.y & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = i + e < V ? load_elem<DT>(from, i + e) : -INFINITY;
    }
  }

  __device__ __forceinline__ void at(int64_t i, double (&r)[4]) const {
    float x[4], y[4];
    load(row, i, x);
    if (DRAFTS && k > 0) load(drow, i, y);
    const auto token = [&](int e) {
      double t = i + e < V ? chance(x[e], st, c32, table) : 0.0;
      if constexpr (DRAFTS) {
        if (k > 0) {
          const double q = chance(y[e], ds, c32, table);
#pragma unroll 1
          for (int j = 0; j < k; ++j) {
            t = t - q;
            t = (t < 0.0 ? 0.0 : t) * (j + 1 < k ? scale[j] : 1.0);
          }
        }
      }
      r[e] = t;
    };
    if (few) {
      // nothing is left of what p does not hold, most of a row below its k-th largest logit: a
      // wavefront's 64 tokens at a time (a walk of some passes over 8192 tokens 17 -> 15 us)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = 0.0;
        if (__any(x[e] >= st.floor) || st.inv != st.inv) token(e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) token(e);
    }
    if constexpr (!DRAFTS) {
      for (int j = 0; j < k; ++j) {
        const int64_t gone = rejected[j] - i;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = gone == e ? 0.0 : r[e];
      }
    }
  }

  // The sum over segment s, of `per` times four tokens a lane. A row without statistics (`bare`)
  // is taken relative to the segment's largest logit, which comes too.
  __device__ __forceinline__ double segment(int64_t s, int64_t per, int lane, bool bare, double c,
                                            float& top) {
    bool bad = false;
    if (bare) {
      float m = -INFINITY;
      for (int64_t u = 0; u < per; ++u) {
        float x[4];
        load(row, (s * per + u) * 256 + 4 * lane, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m = fmaxf(m, x[e]);
          bad |= x[e] != x[e];
        }
      }
      top = wave_max(m);
      bad = __any(bad) || top == INFINITY;
      st = RowStat{1.0, top, exp_floor(top, c), 0};
    }
    double sum = 0.0;
#pragma unroll 1
    for (int64_t u = 0; u < per; ++u) {
      double r[4];
      at((s * per + u) * 256 + 4 * lane, r);
      sum = sum + ((r[0] + r[1]) + (r[2] + r[3]));
    }
    sum = wave_sum_f64(sum);
    return bad ? __longlong_as_double(0x7ff8000000000000ll) : sum;
  }
};

// A row in at most kSegments segments of `per` times 256 tokens.
struct Segments {
  int64_t per;
  int count;
  __device__ __forceinline__ explicit Segments(int64_t V) {
    const int64_t wide = 256;
    per = (V + wide * kSegments - 1) / (wide * kSegments);
    count = static_cast<int>((V + wide * per - 1) / (wide * per));
  }
};

// The walk and the draw of sequence b, by one workgroup. Every thread walks by itself, over what LDS
// holds of the nodes. Where it needs a pass over a row (a residual's sum, a draw), the workgroup makes
// it (LAST), or the walk stops for verify_pass_kernel and goes on in the next launch.
template <int DT, bool DRAFTS, bool LAST>
__device__ __forceinline__ void walk(const Verify& a, int64_t b, bool begin) {
  __shared__ double seg[kSegments], P[kTreeNodes], Q[kTreeNodes], scale[kTreeNodes];
  __shared__ float U[kTreeNodes], top[kSegments];
  __shared__ int par[kTreeNodes], tok[kTreeNodes], rejected[kTreeNodes], way[kTreeNodes];
  __shared__ RowStat stat[DRAFTS ? 2 : 1][kTreeNodes];
  __shared__ double table[kExpSteps];
  const int64_t V = a.V;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = blockDim.x;
  WalkState* const state = a.states ? a.states + b : nullptr;
  const Segments rows(V);
  const bool greedy = a.c == 0.0;
  const double c32 = a.c * kExpSteps;
  // every load that depends on no other first (workgroups have at least kTreeNodes threads)
  const bool wanted = begin || state->request;
  const int64_t len = a.lengths ? a.lengths[b] : a.N;
  const int32_t* const parents = a.parents + b * a.tree_step;
  const int root = parents[0];
  int up = -1;
  int64_t token_id = -1;
  float u = 0.0f;
  if (tid < a.N) {
    up = parents[tid];
    token_id = a.tokens[b * a.N + tid];
    u = greedy ? 0.0f : a.uniforms[b * a.N + tid];
  }
  int cur = 0, k = 0, count = 1, i = 1;
  bool pending = false;  // the last rejected child's residual has no sum yet
  bool served = false;   // the pass that the walk stopped for is there
  bool bare = false;     // the row of `cur` has no statistics
  float most = 0.0f;     // its largest logit then
  // without a drafter: what the rejected tokens left, off by some 2^-48 (a rejected token leaves 2^-24 of
  // it at least, the step of the numbers below 1)
  double rest = 1.0;
  RowStat own{}, other{};  // of the row of `cur` where the walk began again
  int own_of = -1;
  if (!begin) {
    own = state->stat[0], other = state->stat[1];
    cur = state->cur, k = state->k, count = state->count, i = state->i;
    pending = state->pending, rest = state->rest, bare = state->bare;
    served = true;
    own_of = cur;
    if (tid < kTreeNodes) {
      way[tid] = state->way[tid];
      scale[tid] = state->scale[tid];
      rejected[tid] = state->rejected[tid];
      P[tid] = state->P[tid];
      Q[tid] = state->Q[tid];
    }
    for (int s = tid; s < rows.count; s += threads) {
      seg[s] = state->seg[s];
      top[s] = state->top[s];
    }
  }
  if (!wanted) return;
  exp_table(table, tid);
  const int n = static_cast<int>(len < a.N ? len : a.N);
  if (n <= 0 || root != -1) {
    for (int64_t t = tid; t < a.N; t += threads) a.path[b * a.N + t] = -1;
    if (tid == 0) {
      a.counts[b] = 0;
      a.next[b] = -1;
      if (state) state->request = 0;
    }
    return;
  }
  const bool known = token_id >= 0 && token_id < V;
  if (tid < n) {
    par[tid] = up;
    tok[tid] = known ? static_cast<int>(token_id) : -1;
    U[tid] = u;
  }
  if (begin) {
    const bool tested = tid < n && !greedy && up >= 0 && up < tid && known;
    float lp = 0.0f, lq = 0.0f;
    if (tested) {
      lp = load_elem<DT>(row_at<DT>(a, false, b, up), token_id);
      if constexpr (DRAFTS) lq = load_elem<DT>(row_at<DT>(a, true, b, up), token_id);
    }
    __syncthreads();
    // (the statistics of rows that were not wanted hold anything)
    for (int t = tid; t < (DRAFTS ? 2 : 1) * n; t += threads) {
      const int side = t < n ? 0 : 1, node = t < n ? t : t - n;
      const int64_t row = side * a.B * a.N + b * a.N + node;
      stat[side][node] = whole_row(a.parts_of + row * a.parts, a.parts, a.c, table);
      a.stats[row] = stat[side][node];
    }
    __syncthreads();
    if (tid < n) {
      way[tid] = 0;
      P[tid] = tested ? chance(lp, stat[0][up], c32, table) : 0.0;
      Q[tid] = !tested ? 0.0 : DRAFTS ? chance(lq, stat[1][up], c32, table) : 1.0;
    }
  }
  __syncthreads();

  // the statistics of the row of `cur`
  const auto row_stats = [&] {
    if (own_of == cur) return;
    if (begin) {
      own = stat[0][cur];
      if constexpr (DRAFTS) other = stat[1][cur];
    } else {
      own = a.stats[b * a.N + cur];
      if constexpr (DRAFTS) other = a.stats[(a.B + b) * a.N + cur];
    }
    own_of = cur;
  };
  // the segments' sums of what is left at `cur`, and their sum; false where the walk has to stop
  const auto sums = [&](double& total) {
    if (!LAST && !served) {
      row_stats();
      __syncthreads();  // what thread 0 wrote
      for (int t = tid; t < n; t += threads) {
        state->way[t] = way[t];
        state->scale[t] = scale[t];
        state->rejected[t] = rejected[t];
        state->P[t] = P[t];
        state->Q[t] = Q[t];
      }
      if (tid == 0) {
        state->cur = cur, state->k = k, state->count = count, state->i = i;
        state->pending = pending, state->rest = rest;
        state->stat[0] = own, state->stat[1] = other;
        state->bare = bare;
        state->request = 1;
      }
      return false;
    }
    __syncthreads();
    if constexpr (LAST) {
      if (!served) {
        row_stats();
        Residual<DT, DRAFTS> left(a, b, cur, k, own, other, scale, rejected, table);
#pragma unroll 1
        for (int s = wave; s < rows.count; s += threads / 64) {
          float t = 0.0f;
          const double sum = left.segment(s, rows.per, lane, bare, a.c, t);
          if (lane == 0) {
            seg[s] = sum;
            top[s] = t;
          }
        }
      }
    }
    served = false;
    __syncthreads();
    if (bare) {  // relative to the largest of all
      most = -INFINITY;
      for (int s = lane; s < rows.count; s += 64) most = fmaxf(most, top[s]);
      most = wave_max(most);
      const float low = exp_floor(most, a.c);
      __syncthreads();
      for (int s = tid; s < rows.count; s += threads) {
        const double t = top[s] >= low ? scaled_exp(top[s], most, c32, table) : 0.0;
        seg[s] = seg[s] * t;
      }
      __syncthreads();
    }
    total = 0.0;
    for (int s = lane; s < rows.count; s += 64) total = total + seg[s];
    total = wave_sum_f64(total);
    return true;
  };

  // the first child of `cur` from node `from` on, or n (a child of a node that stands comes behind it)
  int mine[kTreeNodes / 64];
#pragma unroll
  for (int w = 0; w < kTreeNodes / 64; ++w) mine[w] = 64 * w + lane < n ? par[64 * w + lane] : -1;
  const auto child = [&](int from) {
    int at = n;
#pragma unroll
    for (int w = kTreeNodes / 64 - 1; w >= 0; --w) {
      uint64_t some = __ballot(mine[w] == cur);
      const int skip = from - 64 * w;
      some = skip <= 0 ? some : skip < 64 ? some & (~0ull << skip) : 0;
      at = some ? 64 * w + static_cast<int>(__builtin_ctzll(some)) : at;
    }
    return at;
  };
  int pick = greedy ? stat[0][0].best : 0;
  double total = 0.0;
  for (i = child(i);;) {
    while (i < n && !(DRAFTS && pending)) {
      bool stands;
      if (tok[i] < 0) {  // no token: a child that is not there
        i = child(i + 1);
        continue;
      }
      if (greedy) {
        stands = tok[i] == pick;
      } else if constexpr (DRAFTS) {
        double t = P[i];
        for (int j = 0; j < k; ++j) {
          t = t - Q[i];
          t = (t < 0.0 ? 0.0 : t) * scale[j];
        }
        stands = U[i] * Q[i] < t;
      } else {
        double t = P[i];
        for (int j = 0; j < k; ++j) t = rejected[j] == tok[i] ? 0.0 : t;
        stands = U[i] * rest < t;
        if (!stands && rest - t <= kNothing * rest) {
          i = child(i + 1);
          continue;
        }
        if (!stands) rest = rest - t;
      }
      if (stands) {
        cur = i;
        k = 0;
        rest = 1.0;
        if (tid == 0) way[count] = i;
        ++count;
        if (greedy) pick = stat[0][cur].best;
      } else if (!greedy) {
        __syncthreads();
        if (tid == 0) rejected[k] = tok[i];
        __syncthreads();
        ++k;
        pending = true;
      }
      i = child(i + 1);
    }
    if (greedy) break;
    // the sum of what the rejected children leave, for the next child or the draw
    bare = i == n && !all_rows(a) && child(cur + 1) == n;
    if (!sums(total)) return;
    pending = false;
    if (DRAFTS && k > 0 && total <= kNothing) {
      --k;
      // (what was left before has its sum already, but a draw wants it over the segments)
      if (i < n) continue;
      if (!sums(total)) return;
    }
    if (i == n) break;
    if (tid == 0) scale[k - 1] = 1.0 / total;
    __syncthreads();
  }
  __syncthreads();
  for (int64_t t = tid; t < a.N; t += threads) a.path[b * a.N + t] = t < count ? way[t] : -1;
  if (tid == 0) {
    a.counts[b] = count;
    if (state) state->request = 0;
  }
  if (wave != 0) return;
  if (greedy || !(total > 0.0)) {
    if (lane == 0) a.next[b] = greedy ? pick : -1;
    return;
  }
  // the segment, then the token in it
  const int each = (rows.count + 63) / 64;
  double share = 0.0;
  for (int s = each * lane; s < each * (lane + 1) && s < rows.count; ++s) share = share + seg[s];
  const double sum = wave_scan(share, lane);
  double bound = U[0] * __shfl(sum, 63);
  // (where rounding lets no sum pass the bound: the last token of any weight)
  const uint64_t over = __ballot(sum > bound), some = __ballot(share > 0.0);
  const int at = over ? static_cast<int>(__builtin_ctzll(over))
                      : 63 - static_cast<int>(__builtin_clzll(some | 1));
  double before = __shfl(sum, at > 0 ? at - 1 : 0);
  if (at == 0) before = 0.0;
  int s = each * at;
  bool found = false;
  for (int u = each * at; u < each * (at + 1) && u < rows.count && !found; ++u) {
    if (seg[u] > 0.0) s = u;
    found = before + seg[u] > bound;
    if (!found) before = before + seg[u];
  }
  if (!found) bound = INFINITY;
  row_stats();
  Residual<DT, DRAFTS> left(a, b, cur, k, own, other, scale, rejected, table);
  if (bare) left.st = RowStat{1.0, most, exp_floor(most, a.c), 0};
  int64_t token = -1, weighty = -1;
#pragma unroll 1
  for (int64_t u = 0; u < rows.per && token < 0; ++u) {
    const int64_t first = (s * rows.per + u) * 256 + 4 * lane;
    double r[4];
    left.at(first, r);
    const double mine = (r[0] + r[1]) + (r[2] + r[3]);
    const double upto = wave_scan(mine, lane);
    // the first of this lane's tokens that passes the bound, and the last of any weight
    double cum = before + (upto - mine);
    int hit = 4, heavy = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cum = e < 3 ? cum + r[e] : before + upto;
      if (r[e] > 0.0) {
        heavy = e;
        if (cum > bound && hit == 4) hit = e;
      }
    }
    const uint64_t hits = __ballot(hit < 4), weights = __ballot(heavy >= 0);
    if (hits) token = __shfl(first + hit, static_cast<int>(__builtin_ctzll(hits)));
    if (weights) weighty = __shfl(first + heavy, 63 - static_cast<int>(__builtin_clzll(weights)));
    before = before + __shfl(upto, 63);
  }
  if (lane == 0) a.next[b] = token >= 0 ? token : weighty;
}

// grid (B): a walk from its begin, or what the rounds left of it. Latencies of dependent reads bound it:
// 15 us with its own passes over 8192 tokens (26 nodes), 7 a launch between passes of the device's.
template <int DT, bool DRAFTS, bool LAST>
__global__ __launch_bounds__(LAST ? 1024 : kTreeNodes) void verify_walk_kernel(Verify a,
                                                                                bool begin) {
  walk<DT, DRAFTS, LAST>(a, blockIdx.x, begin);
}

// grid (B * parts of a row), 256 threads: the segments' sums that a sequence's walk asked for. (The
// workgroup that ends last going on with the walk itself, behind a fence and a counter, made it
// 22 to 57 us instead of 9 and a launch of the walk of 6: each workgroup's fence writes a cache back.)
template <int DT, bool DRAFTS>
__global__ __launch_bounds__(kPassThreads) void verify_pass_kernel(Verify a, int parts) {
  __shared__ double table[kExpSteps];
  const int64_t b = blockIdx.x / static_cast<uint32_t>(parts);
  const int part = static_cast<int>(blockIdx.x - static_cast<uint32_t>(b * parts));
  WalkState& w = a.states[b];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool wanted = w.request, bare = w.bare;
  Residual<DT, DRAFTS> left(a, b, w.cur, w.k, w.stat[0], w.stat[1], w.scale, w.rejected, table);
  if (!wanted) return;
  exp_table(table, tid);
  __syncthreads();
  const Segments rows(a.V);
  const int step = parts * (kPassThreads / 64);
  for (int s = part * (kPassThreads / 64) + (tid >> 6); s < rows.count; s += step) {
    float t = 0.0f;
    const double sum = left.segment(s, rows.per, lane, bare, a.c, t);
    if (lane == 0) {
      w.seg[s] = sum;
      w.top[s] = t;
    }
  }
}

// Passes over rows of up to kOwnPass tokens, or twice as many of which few have a probability (top_k),
// are the walk's own workgroup's (4 to 5 us at 8192, 25 at 32003 with a drafter, where the device's with
// the launches it takes is 20; a call with top_k and a drafter, 16 sequences of 13 nodes: 42 us at 32000
// tokens where the device's passes make it 47, 58 and 55 at 50000). Over larger ones the device shares
// them, so many of a sequence's one after the other. A chain's walk needs one pass, a tree's one more for each
// rejected child but its last, so up to the number of nodes but the root; the rule does not look at the
// nodes. A round that no sequence needs takes 4 us, so a chain or a single draft over a large vocabulary
// beside a drafter waits 28 us for seven (a sequence of 13 nodes, top_k: 36 us at 50000 tokens, 62 at
// 100000); one too few, of 131072 tokens, up to 60. (16 trees of 64 nodes with four children each, eight
// sets of drafts: 141 to 267 us with six rounds, 160 on the average; with eight 148 to 176, 156, and 151
// to 180, 159, in another run; with eleven 160 to 188, 167.)
constexpr int64_t kOwnPass = 16384;
static int verify_rounds(const rk_verify_drafts_args& p) {
  const bool few = p.top_k > 0 && p.top_k < p.V;
  if (p.temperature == 0.0 || p.V <= (few ? 2 : 1) * kOwnPass) return 0;
  return !p.drafts ? 1 : p.V <= 4 * kOwnPass ? 2 : 8;
}

// Rows of a launch: fewer than 2^22. (Each factor by itself first: a product may not fit 64 bits.)
static bool too_many(const rk_verify_drafts_args& p) {
  constexpr int64_t kRows = int64_t{1} << 22;
  return p.B >= kRows || p.B * p.N >= kRows || p.V >= (int64_t{1} << 31) - (int64_t{1} << 20);
}

// Logits of a part of a row: a multiple of 4096 (what 256 threads have in flight), 8192 at least, up
// to eight parts a row and some thousand workgroups. (With one of 256 threads a row, 512 rows of
// 131072 had two wavefronts a SIMD: 106 us, in four parts 62.)
static int64_t stat_part(const rk_verify_drafts_args& p) {
  if (p.temperature == 0.0 || (p.top_k > 0 && p.top_k < p.V)) return p.V;
  const int64_t want = 4096 / (p.B * p.N), parts = want < 1 ? 1 : want < 8 ? want : 8;
  const int64_t part = ((p.V + parts - 1) / parts + 4095) / 4096 * 4096;
  return part < 8192 ? 8192 : part;
}
static int64_t stat_parts(const rk_verify_drafts_args& p) {
  const int64_t part = stat_part(p);
  return (p.V + part - 1) / part;
}
// Workspace of the statistics: whole rows, then their parts.
static int64_t stat_bytes(const rk_verify_drafts_args& p) {
  return (2 * p.B * p.N * (1 + stat_parts(p)) * static_cast<int64_t>(sizeof(RowStat)) + 15) / 16 *
         16;
}

template <int DT, bool DRAFTS>
static void launch_walk(const Verify& a, int rounds, hipStream_t st) {
  const unsigned B = static_cast<unsigned>(a.B);
  const int64_t most = 65536 / a.B < 1 ? 1 : 65536 / a.B < 64 ? 65536 / a.B : 64;
  const int64_t parts = (a.V + 2047) / 2048 < most ? (a.V + 2047) / 2048 : most;
  const unsigned grid = B * static_cast<unsigned>(parts);
  for (int r = 0; r < rounds; ++r) {
    verify_walk_kernel<DT, DRAFTS, false><<<B, kTreeNodes, 0, st>>>(a, r == 0);
    verify_pass_kernel<DT, DRAFTS><<<grid, kPassThreads, 0, st>>>(a, static_cast<int>(parts));
  }
  verify_walk_kernel<DT, DRAFTS, true><<<B, 1024, 0, st>>>(a, rounds == 0);
}

}  // namespace rk

using namespace rk;

extern "C" int64_t rk_verify_drafts_work(const rk_verify_drafts_args* args) {
  if (!args || args->B <= 0 || args->N <= 0 || args->V <= 0 || args->N > kTreeNodes ||
      too_many(*args))
    return 0;
  return stat_bytes(*args) +
         (verify_rounds(*args) ? args->B * static_cast<int64_t>(sizeof(WalkState)) : 0);
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
  const int64_t strides[] = {p.lb, p.ln, p.db, p.dn};
  for (int64_t st : strides)
    if (st < 0) return fail(RK_ERR_ARG, "negative stride");
  if (too_many(p))
    return fail(RK_ERR_UNSUPPORTED, "too many logits for one launch");
  if (!work || !aligned16(work) || work_bytes < rk_verify_drafts_work(args))
    return fail(RK_ERR_ARG, "verification workspace too small");
  const bool drafts = p.drafts && !greedy;
  const int rounds = verify_rounds(p);
  RowStat* const stats = static_cast<RowStat*>(work);
  const int64_t parts = stat_parts(p);
  const Verify a{p.logits, drafts ? p.drafts : nullptr, p.lb, p.ln, p.db, p.dn, p.B, p.N, p.V,
                 p.tokens, p.uniforms, p.parents, p.trees > 1 ? p.N : 0, p.lengths,
                 greedy ? 0.0 : 1.4426950408889634074 / p.temperature, p.top_k, stats,
                 stats + 2 * p.B * p.N, parts, stat_part(p),
                 rounds ? reinterpret_cast<WalkState*>(static_cast<char*>(work) + stat_bytes(p))
                        : nullptr,
                 p.path, p.counts, p.next};
  hipStream_t st = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(p.B * p.N * parts), drafts ? 2 : 1);
  const int mode = greedy ? kGreedy : p.top_k > 0 && p.top_k < p.V ? kTopK : kAll;
  const auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    // whole rows by 512 threads, parts by 256
    if (mode == kGreedy) verify_stats_kernel<DT, 512, kGreedy><<<grid, 512, 0, st>>>(a);
    else if (mode == kTopK) verify_stats_kernel<DT, 512, kTopK><<<grid, 512, 0, st>>>(a);
    else if (parts > 1) verify_stats_kernel<DT, 256, kAll><<<grid, 256, 0, st>>>(a);
    else verify_stats_kernel<DT, 512, kAll><<<grid, 512, 0, st>>>(a);
    if (drafts) launch_walk<DT, true>(a, rounds, st);
    else launch_walk<DT, false>(a, rounds, st);
  };
  if (p.dtype == RK_F32) run(std::integral_constant<int, RK_F32>{});
  else run(std::integral_constant<int, RK_BF16>{});
  return launch_status("verify_drafts");
}

// Pieces shared by the forward and backward of attention with modified scores (rk_scored.hip,
// rk_scored_bwd.hip): the arguments, the score's modification and the mask's intervals.
//
// A score in base-2 units, from the dot product x = q . k and the distance |i - j|:
//   plain   t = x scale log2(e)
//   capped  t = cap log2(e) tanh(x scale / cap) = C - 2 C r,  r = 1 / (exp2(x c) + 1),
//           C = cap log2(e),  c = 2 log2(e) scale / cap;   1 - tanh^2 = 4 r (1 - r)
//   biased  t - slope log2(e) |i - j|
// exp2 and the reciprocal are the hardware's (1 ulp): the capped score is off by at most a few
// 2^-24 of the cap, 2e-5 of a probability at cap 50 against the 2^-9 of its rounding to bf16. Caps
// lie in 1e-3 .. 1e3 (2e-4 there).
//
// A mask is two intervals per position (rk_attention_mask): the keys [key_lo, key_hi) that a
// query sees and the queries [query_lo, query_hi) that see a key. A position that sees nothing
// has empty ones. Both kernels test the intervals of the rows they own, one per lane.
#pragma once

#include "rk_attention.h"

namespace rk {

struct ScoredArgs {
  rk_scored_attention_args p;
  uint32_t BH, H, G;  // query heads of all, of a sequence, per key head
  int64_t S32;      // padding words per row
  int64_t Sp;       // S rounded up to 128 (row statistics)
  float dot_scale;  // plain: scale log2(e); capped: 2 log2(e) scale / cap
  float cap2;       // cap log2(e)
  // near_capped: scale log2(e), the largest |x|, the coefficients by C^-2, C^-4, .., 1 / C
  float near_scale, near_limit, near[4], inv_cap2;
};

constexpr float kLog2e = 1.4426950408889634f;

// The capped score in base-2 units by an odd polynomial, y + y z (c1 + c2 z + c3 z^2 + c4 z^3) with
// y = x scale log2(e), z = y^2: tanh(u) / u fitted by least squares at Chebyshev nodes of
// |u| <= 1/2, off by 2e-8 there. The exponential form is off by 2^-24 of the cap whatever the
// score, which the slopes' gradient, a float32 sum over all pairs, shows: 3e-6 of its norm at
// caps of 50 to 100, against 2e-7 to 5e-7 with the polynomial there and in the forward. Other results are
// bf16 and keep the exponential: with a branch between the two forms those kernels were slower,
// the forward by a fifth.
__device__ __forceinline__ float near_capped(const ScoredArgs& a, float x, float& slack) {
  const float y = x * a.near_scale, z = y * y;
  float q = __builtin_fmaf(a.near[3], z, a.near[2]);
  q = __builtin_fmaf(q, z, a.near[1]);
  q = __builtin_fmaf(q, z, a.near[0]);
  const float t = __builtin_fmaf(y, z * q, y), th = t * a.inv_cap2;
  slack = __builtin_fmaf(-th, th, 1.0f);
  return t;
}

struct Span {
  int lo, hi;  // what this lane's row sees; rows without any see everything and are discarded
  bool valid;
};

// The interval of row `row` (0 .. S - 1, or past it) of batch b; `kind` 0: keys of a query,
// 2: queries of a key. Without a mask: causal.
__device__ __forceinline__ Span row_span(const rk_scored_attention_args& p, int kind, int64_t b,
                                         int row) {
  const int S = static_cast<int>(p.S);
  Span s{0, 0, row < S};
  if (s.valid) {
    if (p.bounds) {
      const int32_t* at = p.bounds + (kind * p.mask_batch + (p.mask_batch > 1 ? b : 0)) * p.S + row;
      s.lo = at[0] > 0 ? at[0] : 0;
      s.hi = at[p.mask_batch * p.S];
      s.hi = s.hi < S ? s.hi : S;
    } else {
      s.lo = kind == 0 ? 0 : row;
      s.hi = kind == 0 ? row + 1 : S;
    }
    s.valid = s.hi > s.lo;
  }
  return s;
}

__device__ __forceinline__ int wave_min_int(int v) {
  return wave_butterfly(v, [](int a, int b) { return a < b ? a : b; });
}
__device__ __forceinline__ int wave_max_int(int v) {
  return wave_butterfly(v, [](int a, int b) { return a > b ? a : b; });
}

// What a wavefront's rows see: anything lies in [lo, hi), everything in [all_lo, all_hi).
struct WaveSpan {
  int lo, hi, all_lo, all_hi;
  __device__ __forceinline__ explicit WaveSpan(Span& s) {
    lo = __builtin_amdgcn_readfirstlane(wave_min_int(s.valid ? s.lo : 0x7fffffff));
    hi = __builtin_amdgcn_readfirstlane(wave_max_int(s.valid ? s.hi : 0));
    all_lo = __builtin_amdgcn_readfirstlane(wave_max_int(s.valid ? s.lo : 0));
    all_hi = __builtin_amdgcn_readfirstlane(wave_min_int(s.valid ? s.hi : 0x7fffffff));
    if (!s.valid) {
      s.lo = 0;
      s.hi = 0x7fffffff;
    }
  }
  __device__ __forceinline__ bool none(int r0, int rows) const {
    return r0 >= hi || r0 + rows <= lo;
  }
  __device__ __forceinline__ bool all(int r0, int rows) const {
    return r0 >= all_lo && r0 + rows <= all_hi;
  }
};

// The workgroup's range over its four wavefronts' (box: 8 ints of LDS).
__device__ __forceinline__ void block_range(const WaveSpan& w, int wave, int lane, int* box,
                                            int& lo, int& hi) {
  if (lane == 0) {
    box[wave] = w.lo;
    box[4 + wave] = w.hi;
  }
  __syncthreads();
  lo = box[0];
  hi = box[4];
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    lo = box[i] < lo ? box[i] : lo;
    hi = box[4 + i] > hi ? box[4 + i] : hi;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
}

// Padding bits of rows row0 .. row0 + R - 1 (row0 a multiple of 32) of batch b.
template <int R>
__device__ __forceinline__ uint64_t padding_bits(const ScoredArgs& a, int64_t b, int row0) {
  if (!a.p.padding) return 0;
  const uint32_t* at = a.p.padding + (a.p.mask_batch > 1 ? b : 0) * a.S32;
  const int w = row0 / 32;
  uint64_t bits = at[w];
  if constexpr (R == 64) {
    if (w + 1 < a.S32) bits |= static_cast<uint64_t>(at[w + 1]) << 32;
  }
  return bits;
}

// Zeros the padding rows of a staged tile: their values, which may be anything, meet
// probabilities of zero. Every thread of the workgroup calls it, between two barriers.
template <int D, int R>
__device__ __forceinline__ void clear_rows(uint8_t* tile, uint64_t bits, int tid) {
  constexpr int SEGS = D / 8;
  for (int i = tid; i < R * SEGS; i += 256)
    if (bits >> (i / SEGS) & 1)
      *reinterpret_cast<uint4*>(tile + 16 * i) = make_uint4(0, 0, 0, 0);
}

// What rounding 4 numbers to the bf16 pairs lo, hi left, a byte each in 256ths of the bf16 step
// (to the nearest, so to 2^-16 of the number, and exact where nothing was left: a token that sees
// only itself gets no gradient from o's own rounding): the second byte of the bit patterns'
// difference, which lies in -2^15 .. 2^15 (the upper end, a tie, taken as the largest byte).
__device__ __forceinline__ uint32_t bf16_rest4(const float (&x)[4], uint32_t lo, uint32_t hi) {
  const uint32_t r[4] = {lo << 16, lo & 0xffff0000u, hi << 16, hi & 0xffff0000u};
  uint32_t d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int diff = static_cast<int>(__float_as_uint(x[e]) - r[e]) + 128;
    d[e] = static_cast<uint32_t>(diff < 0x7fff ? diff : 0x7fff);
  }
  const uint32_t p01 = __builtin_amdgcn_perm(d[1], d[0], 0x0c0c0501u);
  const uint32_t p23 = __builtin_amdgcn_perm(d[3], d[2], 0x0c0c0501u);
  return __builtin_amdgcn_perm(p23, p01, 0x05040100u);
}

// Where the rests of a head's 32 rows from row0 on lie: words [D / 8][64], word r of lane l + 32 h
// (features 8 r + 4 h .. + 3 of row l) at 64 r + 32 h + l. In rows as o has them the forward's
// 4-byte stores and the backward's 8-byte loads, each to a row of its own, cost 5 us each at
// B 8, H 16, S 1024, D 128.
template <int D>
__device__ __forceinline__ uint32_t* rest_words(const ScoredArgs& a, int64_t bh, int row0) {
  return reinterpret_cast<uint32_t*>(a.p.rest + (bh * a.Sp + row0) * D);
}

// The float32 number, to half of its rest's step.
__device__ __forceinline__ float with_rest(uint32_t bf16_high, int rest) {
  return __uint_as_float(bf16_high + static_cast<uint32_t>(rest * 256));
}

int check_scored(const rk_scored_attention_args& p, bool backward);
ScoredArgs scored_args(const rk_scored_attention_args& p);

}  // namespace rk

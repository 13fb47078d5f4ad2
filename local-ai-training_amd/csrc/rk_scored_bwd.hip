// The backward of attention with modified scores (rk_scored.hip; gfx950): from bf16 q, k, v, o,
// the gradient g of o and the forward's log-sum-exp,
//   p_ij = exp(s_ij - lse_i) where i sees j, else 0,     delta_i = g_i . o_i,
//   d_ij = p_ij (g_i . v_j - delta_i)                    (gradient of the modified score)
//   ds_ij = d_ij (1 - tanh^2)                            (of the plain one; no cap: d_ij)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij g_i,
//   dslope_h = -sum_ij d_ij |i - j|.
// Products of bf16 operands summed in float32; p and ds enter the second products rounded to
// bf16 (half a step); scores, exponentials, delta are float32, o with what its rounding left
// (`rest`): with the bf16 o alone, dq and dk of concentrated rows were off by 2.7e-3 to 3.2e-3 of
// their norm instead of 2.4e-3 (the rounding of ds and of the results). Two launches, as
// at rk_attention_bwd.hip: the queries' (dq, and delta for the second) and the keys' (dk, dv; the
// query heads that share a key head are summed by the one wavefront that owns the key, in order),
// every output summed in a fixed order, so results repeat.
//
// The slopes' gradient takes three sums per query, of p dp, p |i - j| and p dp |i - j| with
// dp = g . v - delta: with the first in place of what rounding o to bf16 left of it,
// sum_j d_ij |i - j| = sum p dp |i - j| - (sum p dp)(sum p |i - j|). A third launch adds the
// queries in 64 bits.
//
// B 8, H 16, S 1024, D 128: causal 85 + 115 us (rk_attention_backward 75 + 90 for the same 120
// GFLOP), in documents of 400 on average 59 + 69, capped as well 67 + 88; B 4, S 1001 with a
// learned bias 54 + 62; B 32, H 8, S 512, D 64 in documents of 150 29.6 + 29.5 us. Per step a
// wavefront of the keys' launch waits 58% of its cycles (barriers, LDS operands, dependent
// products), its vector instructions fill 18 of the 88 us and its MFMAs 12.5. Three stages of
// tiles for the queries changed nothing, 64 staged rows at D 128 and both products ahead of a
// p formed in two halves were slower.
#include "rk_scored.h"

namespace rk {

struct ScoredBwdArgs {
  ScoredArgs f;
  float inv_scale;  // 1 / scale
  float* rows;      // [B H][2][Sp]: log-sum-exp term and -delta (zeros where a row is none)
  float* slope_rows;  // [B H][Sp], or null
  // the query heads of a key head in `parts` workgroups each: their float32 dk, dv [parts][2]
  // [B Hkv][S][D], added by a launch of their own (1: written as they are)
  int64_t parts;
  float* part_rows;
};

constexpr int kBwdRows = 32;  // staged rows per step
constexpr int64_t kBwdBlocks = 1024;  // workgroups wanted of the second launch (head_parts)

// p and the factor of the score's gradient from the accumulated dot product. `term`: plain,
// already in the accumulator (-lse / scale); otherwise lse log2(e), subtracted here.
template <bool CAP, bool BIAS>
__device__ __forceinline__ float score_p(const ScoredArgs& a, float x, float term, float slope2,
                                         float dist, float& slack) {
  if constexpr (CAP) {
    const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * a.dot_scale) + 1.0f);
    slack = 4.0f * r * (1.0f - r);
    float t = __builtin_fmaf(-2.0f * a.cap2, r, a.cap2 - term);
    if constexpr (BIAS) t = __builtin_fmaf(-slope2, fabsf(dist), t);
    return __builtin_amdgcn_exp2f(t);
  } else {
    slack = 1.0f;
    if constexpr (BIAS)
      return __builtin_amdgcn_exp2f(
          __builtin_fmaf(-slope2, fabsf(dist), x * a.dot_scale));
    return __builtin_amdgcn_exp2f(x * a.dot_scale);
  }
}

template <int D, bool CAP, bool BIAS, bool SG>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void scored_dq_kernel(ScoredBwdArgs ba) {
  constexpr int R = D == 64 ? 64 : 32;  // staged keys per step; 32 at a time are computed
  using T = AttnTile<D, R>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kAttnStages * 2 * T::BYTES];
  __shared__ int box[8];
  const uint32_t lds0 = lds_address(smem);
  const ScoredArgs& a = ba.f;
  const rk_scored_attention_args& p = a.p;
  const int S = static_cast<int>(p.S);
  const int nqb = (S + kAttnRows - 1) / kAttnRows;
  const uint32_t blk = blockIdx.x / a.BH, ubh = blockIdx.x - blk * a.BH, ub = ubh / a.H;
  const int qb = nqb - 1 - static_cast<int>(blk);  // longest causal rows first; heads fastest
  const int64_t bh = ubh, b = ub, hd = ubh - ub * a.H, kvh = (ubh - ub * a.H) / a.G;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw0 = qb * kAttnRows + 32 * wave, qi = qw0 + l32;

  v8bf_a qf[D / 16], gf[D / 16];
  load_owned<D>(qf, p.q + b * p.sqb + hd * p.sqh, p.sqs, S, qi, h);
  load_owned<D>(gf, p.g + b * p.sgb + hd * p.sgh, p.sgs, S, qi, h);
  Span span = row_span(p, 0, b, qi);
  const WaveSpan ws(span);
  int lo, hi;
  block_range(ws, wave, lane, box, lo, hi);
  const int first = lo < hi ? lo / R : 0;
  const int end = lo < hi ? (hi + R - 1) / R : 0;
  const uint32_t width = static_cast<uint32_t>(span.hi - span.lo);

  const TileDma<D, R> kd(p.k + b * p.skb + kvh * p.skh, p.sks, S, wave, lane);
  const TileDma<D, R> vd(p.v + b * p.svb + kvh * p.svh, p.svs, S, wave, lane);
  auto issue = [&](int step) {
    const uint32_t st = lds0 + (step & 1) * 2 * T::BYTES;
    kd.issue(st, step * R, wave);
    vd.issue(st + T::BYTES, step * R, wave);
  };
  if (first < end) issue(first);  // under way while delta is formed

  // delta of this lane's query: half of the features here, the other half in lane ^ 32
  float dot = 0.0f;
  {
    v8bf_a of[D / 16];
    load_owned<D>(of, p.o + b * p.sob + hd * p.soh, p.sos, S, qi, h);
    uint2 rest[D / 16] = {};  // features 16 s + 8 h .. + 7: words 2 s + h of lanes l and l + 32
    if (p.rest) {
      const uint32_t* const at = rest_words<D>(a, bh, qw0) + 64 * h + l32;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) rest[s] = make_uint2(at[128 * s], at[128 * s + 32]);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const uint4 w = __builtin_bit_cast(uint4, of[s]);
      const uint32_t pairs[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int8_t r = static_cast<int8_t>((e < 4 ? rest[s].x : rest[s].y) >> (8 * (e % 4)));
        const uint32_t high = e % 2 ? pairs[e / 2] & 0xffff0000u : pairs[e / 2] << 16;
        const float ov = p.rest ? with_rest(high, r) : __uint_as_float(high);
        dot = __builtin_fmaf(static_cast<float>(gf[s][e]), ov, dot);
      }
    }
  }
  dot = dot + __shfl_xor(dot, 32, kWave);
  const float lse = span.valid ? p.lse[bh * S + qi] : 0.0f;
  // for the keys' launch, as score_p takes it there; this one subtracts lse after the product where
  // the score is modified (a sum that begins at -lse / scale rounds to its size, 1e-6 of p)
  const float term = CAP ? lse * kLog2e : -lse * ba.inv_scale;
  const float lse2 = lse * kLog2e;
  const float ndelta = span.valid ? -dot : 0.0f;
  if (h == 0) {  // Sp rows: the padded block's too
    float* const rows = ba.rows + bh * 2 * a.Sp + qi;
    rows[0] = term;
    rows[a.Sp] = ndelta;
  }
  float slope2 = 0.0f;
  if constexpr (BIAS) slope2 = p.slopes[hd] * kLog2e;

  v16f_a dq[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) dq[dt] = v16f_a{};
  float s_pd = 0.0f, s_pa = 0.0f, s_pda = 0.0f;  // sums of p dp, p |i - j|, p dp |i - j|
  for (int step = first; step < end; ++step) {
    const uint64_t pad = padding_bits<R>(a, b, step * R);
    dma_wait_barrier<0>();
    if (step + 1 < end) issue(step + 1);
    uint8_t* const kt = smem + (step & 1) * 2 * T::BYTES;
    uint8_t* const vt = kt + T::BYTES;
    if (pad) {  // the keys meet gradients of zero
      clear_rows<D, R>(kt, pad, tid);
      __syncthreads();
    }
    // (64 staged at head size 128 too: 65 -> 77 us with a bias and slope gradients at B 4, S 1001)
#pragma unroll
    for (int sub = 0; sub < R; sub += 32) {
      const int key0 = step * R + sub;
      if (ws.none(key0, 32)) continue;
      v16f_a st;
#pragma unroll
      for (int e = 0; e < 16; ++e) st[e] = CAP || BIAS ? 0.0f : term;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<D>(kt, sub, s, lane), qf[s], st,
                                                     0, 0, 0);
      const bool whole = ws.all(key0, 32);
      const int j0 = key0 + 4 * h - span.lo;
      const float d0 = static_cast<float>(qi - key0 - 4 * h);
      v16f_a dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] = ndelta;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<D>(vt, sub, s, lane), gf[s], dp,
                                                     0, 0, 0);
      // the masks in one uniform branch ahead of straight arithmetic (a masked score of -inf
      // gives p = 0, a capped one the cap's end, whose gradient is zero with dp; of a negative
      // slope its p may be infinite)
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (static_cast<uint32_t>(j0 + 8 * (e / 4) + (e % 4)) >= width) {
            st[e] = -INFINITY;
            dp[e] = 0.0f;
          }
      }
      bool near = false;
      if constexpr (CAP && SG) {
        float most = 0.0f;  // of the scores that count
#pragma unroll
        for (int e = 0; e < 16; ++e) most = fmaxf(most, st[e] == -INFINITY ? 0.0f : fabsf(st[e]));
        near = !__any(most > a.near_limit);
      }
      float ds[16];
      const auto gradient = [&](int e, float p1, float sl) {
        const float p2 = CAP && SG && st[e] == -INFINITY ? 0.0f
                         : CAP && BIAS && !SG            ? fminf(p1, 0x1p100f)
                                                         : p1;
        ds[e] = p2 * dp[e];
        if constexpr (SG) {
          const float dist = fabsf(d0 - static_cast<float>(8 * (e / 4) + (e % 4)));
          s_pd = s_pd + ds[e];
          s_pa = __builtin_fmaf(p2, dist, s_pa);
          s_pda = __builtin_fmaf(ds[e], dist, s_pda);
        }
        if constexpr (CAP) ds[e] = ds[e] * sl;
      };
      if (near) {  // (never without slope gradients)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float sl;
          const float y = st[e] == -INFINITY ? 0.0f : st[e];
          const float t = near_capped(a, y, sl) - lse2;
          const float dist = fabsf(d0 - static_cast<float>(8 * (e / 4) + (e % 4)));
          gradient(e, __builtin_amdgcn_exp2f(__builtin_fmaf(-slope2, dist, t)), sl);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float sl = 1.0f;
          const float dist = d0 - static_cast<float>(8 * (e / 4) + (e % 4));
          float p1;
          if constexpr (!CAP && BIAS)
            p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(
                -slope2, fabsf(dist), __builtin_fmaf(st[e], a.dot_scale, -lse2)));
          else
            p1 = score_p<CAP, BIAS>(a, st[e], lse2, slope2, dist, sl);
          gradient(e, p1, sl);
        }
      }
      uint4 dsf[2];
      pack16(dsf, ds);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
          dq[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              col_frag<D>(kt, sub + 16 * s2, dt, lane), frag_of(dsf[s2]), dq[dt], 0, 0, 0);
    }
  }
  if (!span.valid) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) dq[dt] = v16f_a{};
  }
  if (qi < S)
    store_owned<D>(p.dq + b * p.sxb + hd * p.sxh + static_cast<int64_t>(qi) * p.sxs, dq, p.scale,
                   h);
  if constexpr (SG) {
    s_pd = s_pd + __shfl_xor(s_pd, 32, kWave);
    s_pa = s_pa + __shfl_xor(s_pa, 32, kWave);
    s_pda = s_pda + __shfl_xor(s_pda, 32, kWave);
    if (h == 0) ba.slope_rows[bh * a.Sp + qi] = span.valid ? s_pda - s_pd * s_pa : 0.0f;
  }
}

// dslope[h] = -sum over the sequences and queries, in 64 bits and a fixed order; four loads in
// flight.
__global__ __launch_bounds__(1024) void scored_slope_kernel(ScoredBwdArgs ba) {
  __shared__ double red[1024];
  const ScoredArgs& a = ba.f;
  const int64_t hd = blockIdx.x;
  const int tid = threadIdx.x;
  double sum = 0.0;
  for (int64_t b = 0; b < a.p.B; ++b) {
    const float* rows = ba.slope_rows + (b * a.p.H + hd) * a.Sp;
    for (int64_t i = 4 * tid; i < a.Sp; i += 4096) {  // Sp is a multiple of 128
      const float4 x = *reinterpret_cast<const float4*>(rows + i);
      sum += (static_cast<double>(x.x) + x.y) + (static_cast<double>(x.z) + x.w);
    }
  }
  red[tid] = sum;
  for (int n = 512; n > 0; n >>= 1) {
    __syncthreads();
    if (tid < n) red[tid] += red[tid + n];
  }
  if (tid == 0) a.p.dslopes[hd] = static_cast<float>(-red[0]);
}

template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(D == 64 && !CAP ? 3 : 2, D == 64 && !CAP ? 3 : 2)))
void scored_dkv_kernel(ScoredBwdArgs ba) {
  using T = AttnTile<D, kBwdRows>;
  constexpr int STAGE = 2 * T::BYTES + 256;  // two tiles, 32 log-sum-exp terms, 32 -delta
  // the owned V rows stay in LDS (rk_attention_bwd.hip: in registers beside K the loop spills)
  constexpr int VTILE = kAttnRows * T::ROWB;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[VTILE + kAttnStages * STAGE];
  __shared__ int box[8];
  const uint32_t lds0 = lds_address(smem) + VTILE;
  const ScoredArgs& a = ba.f;
  const rk_scored_attention_args& p = a.p;
  const int S = static_cast<int>(p.S);
  const uint32_t uparts = static_cast<uint32_t>(ba.parts);
  const uint32_t ukv = static_cast<uint32_t>(p.Hkv), uBH = static_cast<uint32_t>(p.B) * ukv;
  const uint32_t blk = blockIdx.x / (uBH * uparts);  // heads fastest
  const uint32_t uidx = blockIdx.x - blk * (uBH * uparts), ubh = uidx / uparts, ub = ubh / ukv;
  const int64_t BH = uBH, bh = ubh, part = uidx - ubh * uparts, b = ub, kvh = ubh - ub * ukv;
  const int heads = static_cast<int>(a.G / uparts);
  const int64_t hq = kvh * static_cast<int64_t>(a.G) + part * heads;  // the first query head
  const int k0 = static_cast<int>(blk) * kAttnRows;  // the first keys have the longest walk
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kj = k0 + 32 * wave + l32;

  v8bf_a kf[D / 16];
  load_owned<D>(kf, p.k + b * p.skb + kvh * p.skh, p.sks, S, kj, h);
  Span span = row_span(p, 2, b, kj);
  const WaveSpan ws(span);
  int lo, hi;
  block_range(ws, wave, lane, box, lo, hi);
  const int first = lo < hi ? lo / kBwdRows : 0;
  const int steps = lo < hi ? (hi + kBwdRows - 1) / kBwdRows - first : 0;
  const uint32_t width = static_cast<uint32_t>(span.hi - span.lo);

  const TileDma<D, kBwdRows> vd(p.v + b * p.svb + kvh * p.svh, p.svs, S, wave, lane);
#pragma unroll
  for (int t = 0; t < kAttnRows / kBwdRows; ++t)
    vd.issue(lds_address(smem) + t * T::BYTES, k0 + t * kBwdRows, wave);

  // the query heads one after the other, the tiles of the next one behind the last of
  // this one: tile n of all is step n % steps of head n / steps
  const int total = steps * heads;
  int ihead = 0, istep = 0;  // the next tile to load
  TileDma<D, kBwdRows> qd(p.q + b * p.sqb + hq * p.sqh, p.sqs, S, wave, lane);
  TileDma<D, kBwdRows> gd(p.g + b * p.sgb + hq * p.sgh, p.sgs, S, wave, lane);
  // row statistics: lanes 0..31 take the first plane, lanes 32..63 the second (every wavefront
  // writes the same bytes)
  const int rvoff = static_cast<int>((h * a.Sp + l32) * 4);
  __amdgpu_buffer_rsrc_t rbuf = make_buffer(ba.rows + (b * p.H + hq) * 2 * a.Sp, 2 * a.Sp * 4);
  auto issue = [&](int n) {
    const uint32_t st = lds0 + (n & 1) * STAGE;
    const int row0 = (first + istep) * kBwdRows;
    dma4(rbuf, st + 2 * T::BYTES, rvoff, row0 * 4);
    qd.issue(st, row0, wave);
    gd.issue(st + T::BYTES, row0, wave);
    if (++istep == steps) {
      istep = 0;
      const int64_t hd = hq + ++ihead;
      if (ihead < heads) {
        qd.buf = make_buffer(p.q + b * p.sqb + hd * p.sqh, ((p.S - 1) * p.sqs + D) * 2);
        gd.buf = make_buffer(p.g + b * p.sgb + hd * p.sgh, ((p.S - 1) * p.sgs + D) * 2);
        rbuf = make_buffer(ba.rows + (b * p.H + hd) * 2 * a.Sp, 2 * a.Sp * 4);
      }
    }
  };

  v16f_a dk[D / 32], dv[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    dk[dt] = v16f_a{};
    dv[dt] = v16f_a{};
  }
  if (total > 0) issue(0);
  int chead = 0, cstep = 0;  // the tile computed
  float slope2 = 0.0f;
  for (int n = 0; n < total; ++n) {
    const int qs = (first + cstep) * kBwdRows;
    const uint64_t pad = padding_bits<kBwdRows>(a, b, qs);
    if constexpr (BIAS)
      if (cstep == 0) slope2 = p.slopes[hq + chead] * kLog2e;
    if (++cstep == steps) {
      cstep = 0;
      ++chead;
    }
    dma_wait_barrier<0>();
    if (n + 1 < total) issue(n + 1);
    uint8_t* const qt = smem + VTILE + (n & 1) * STAGE;
    uint8_t* const gt = qt + T::BYTES;
    const float* rows = reinterpret_cast<const float*>(gt + T::BYTES);
    if (pad) {  // the queries and their gradients meet probabilities of zero
      clear_rows<D, kBwdRows>(qt, pad, tid);
      clear_rows<D, kBwdRows>(gt, pad, tid);
      __syncthreads();
    }
    if (ws.none(qs, kBwdRows)) continue;
    // -lse / scale (plain: where the scores' sums begin), or lse log2(e)
    const auto row_terms = [&](int plane, v16f_a& x) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float4 v = *reinterpret_cast<const float4*>(rows + plane * kBwdRows + 8 * r + 4 * h);
        x[4 * r] = v.x; x[4 * r + 1] = v.y; x[4 * r + 2] = v.z; x[4 * r + 3] = v.w;
      }
    };
    v16f_a st{};
    if constexpr (!CAP) row_terms(0, st);
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<D>(qt, 0, s, lane), kf[s], st,
                                                   0, 0, 0);
    v16f_a dp;
    row_terms(1, dp);
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<D>(gt, 0, s, lane),
                                                   row_frag<D>(smem, 32 * wave, s, lane), dp,
                                                   0, 0, 0);
    // the masks sit in one uniform branch ahead of straight arithmetic: with the probabilities
    // formed before the second product, and the masks on them, the loop spilled or took a
    // quarter longer. A masked score of -inf gives p = 0; a capped one gives the cap's end, with
    // slope 0, and its p (infinite beside a negative slope, then with a gradient that is not a
    // number) is cleared below.
    const bool whole = ws.all(qs, kBwdRows);
    const int i0 = qs + 4 * h - span.lo;
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (static_cast<uint32_t>(i0 + 8 * (e / 4) + (e % 4)) >= width) {
          st[e] = -INFINITY;
          dp[e] = 0.0f;
        }
    }
    const float d0 = static_cast<float>(qs + 4 * h - kj);
    uint4 pf[2], dsf[2];
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      float pr[8], ds[8];
#pragma unroll
      for (int r = 2 * s2; r < 2 * s2 + 2; ++r) {
        float4 term{};
        if constexpr (CAP) term = *reinterpret_cast<const float4*>(rows + 8 * r + 4 * h);
        const float t4[4] = {term.x, term.y, term.z, term.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int e = 4 * r + x;
          float sl;
          const float p1 = score_p<CAP, BIAS>(a, st[e], t4[x], slope2,
                                              d0 + static_cast<float>(8 * r + x), sl);
          pr[e - 8 * s2] = p1;
          ds[e - 8 * s2] = (CAP ? p1 * sl : p1) * dp[e];
        }
      }
      pf[s2] = make_uint4(bf16_pair(pr[0], pr[1]), bf16_pair(pr[2], pr[3]),
                          bf16_pair(pr[4], pr[5]), bf16_pair(pr[6], pr[7]));
      dsf[s2] = make_uint4(bf16_pair(ds[0], ds[1]), bf16_pair(ds[2], ds[3]),
                           bf16_pair(ds[4], ds[5]), bf16_pair(ds[6], ds[7]));
    }
    if constexpr (CAP)
      if (!whole) {
        uint32_t* const w[8] = {&pf[0].x, &pf[0].y, &pf[0].z, &pf[0].w,
                                &pf[1].x, &pf[1].y, &pf[1].z, &pf[1].w};
        uint32_t* const d[8] = {&dsf[0].x, &dsf[0].y, &dsf[0].z, &dsf[0].w,
                                &dsf[1].x, &dsf[1].y, &dsf[1].z, &dsf[1].w};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (static_cast<uint32_t>(i0 + 8 * (e / 4) + (e % 4)) >= width) {
            const uint32_t keep = e % 2 ? 0x0000ffffu : 0xffff0000u;
            *w[e / 2] &= keep;
            if constexpr (BIAS) *d[e / 2] &= keep;
          }
      }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
        dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            col_frag<D>(gt, 16 * s2, dt, lane), frag_of(pf[s2]), dv[dt], 0, 0, 0);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
        dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            col_frag<D>(qt, 16 * s2, dt, lane), frag_of(dsf[s2]), dk[dt], 0, 0, 0);
  }
  // no load may still write this workgroup's LDS when it ends
  if (total == 0) dma_wait_barrier<0>();
  if (!span.valid) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      dk[dt] = v16f_a{};
      dv[dt] = v16f_a{};
    }
  }
  if (kj < S && ba.parts > 1) {
    float* const to = ba.part_rows + ((part * 2 * BH + bh) * S + kj) * D + 4 * h;
    const int64_t plane = BH * S * D;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float* const x = to + 32 * dt + 8 * r;
        *reinterpret_cast<float4*>(x) =
            make_float4(dk[dt][4 * r], dk[dt][4 * r + 1], dk[dt][4 * r + 2], dk[dt][4 * r + 3]);
        *reinterpret_cast<float4*>(x + plane) =
            make_float4(dv[dt][4 * r], dv[dt][4 * r + 1], dv[dt][4 * r + 2], dv[dt][4 * r + 3]);
      }
  } else if (kj < S) {
    const int64_t off = b * p.syb + kvh * p.syh + static_cast<int64_t>(kj) * p.sys;
    store_owned<D>(p.dk + off, dk, p.scale, h);
    store_owned<D>(p.dv + off, dv, 1.0f, h);
  }
}

// grid (S * D / 1024, B * Hkv, 2: dk, dv), 256 threads of 4 features: the parts, in order.
__global__ __launch_bounds__(256) void scored_parts_kernel(ScoredBwdArgs ba) {
  const rk_scored_attention_args& p = ba.f.p;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  const int64_t BH = p.B * p.Hkv, bh = blockIdx.y, plane = BH * p.S * p.D;
  if (i >= p.S * p.D) return;
  const float* at = ba.part_rows + blockIdx.z * plane + bh * p.S * p.D + i;
  float4 sum = *reinterpret_cast<const float4*>(at);
  for (int64_t n = 1; n < ba.parts; ++n) {
    const float4 x = *reinterpret_cast<const float4*>(at + 2 * n * plane);
    sum.x = sum.x + x.x;
    sum.y = sum.y + x.y;
    sum.z = sum.z + x.z;
    sum.w = sum.w + x.w;
  }
  const int64_t row = i / p.D, b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  uint16_t* const to = (blockIdx.z ? p.dv : p.dk) + b * p.syb + kvh * p.syh + row * p.sys +
                       (i - row * p.D);
  const float f = blockIdx.z ? 1.0f : p.scale;
  *reinterpret_cast<uint2*>(to) =
      make_uint2(bf16_pair(sum.x * f, sum.y * f), bf16_pair(sum.z * f, sum.w * f));
}

// Parts of the query heads that share a key head: enough for about 1024 workgroups.
static int64_t head_parts(int64_t B, int64_t H, int64_t Hkv, int64_t S) {
  const int64_t G = H / Hkv, have = B * Hkv * ((S + kAttnRows - 1) / kAttnRows);
  for (int64_t n = 1; n < G; ++n)
    if (G % n == 0 && have * n >= kBwdBlocks) return n;
  return G;
}

template <int D, bool CAP, bool BIAS>
static void launch_scored_bwd(const ScoredBwdArgs& a, hipStream_t st) {
  const rk_scored_attention_args& p = a.f.p;
  const unsigned blocks = static_cast<unsigned>(a.f.Sp / kAttnRows);
  const dim3 qgrid(static_cast<unsigned>(p.B * p.H) * blocks);
  const dim3 kgrid(static_cast<unsigned>(p.B * p.Hkv * a.parts) * blocks);
  if (BIAS && a.slope_rows) {
    scored_dq_kernel<D, CAP, BIAS, BIAS><<<qgrid, 256, 0, st>>>(a);
    scored_slope_kernel<<<static_cast<unsigned>(p.H), 1024, 0, st>>>(a);
  } else {
    scored_dq_kernel<D, CAP, BIAS, false><<<qgrid, 256, 0, st>>>(a);
  }
  scored_dkv_kernel<D, CAP, BIAS><<<kgrid, 256, 0, st>>>(a);
  if (a.parts > 1)
    scored_parts_kernel<<<dim3(static_cast<unsigned>((p.S * D + 1023) / 1024),
                               static_cast<unsigned>(p.B * p.Hkv), 2), 256, 0, st>>>(a);
}

template <int D>
static void dispatch_scored_bwd(const ScoredBwdArgs& a, hipStream_t st) {
  const bool cap = a.f.p.softcap > 0.0f, bias = a.f.p.slopes != nullptr;
  if (cap && bias) launch_scored_bwd<D, true, true>(a, st);
  else if (cap) launch_scored_bwd<D, true, false>(a, st);
  else if (bias) launch_scored_bwd<D, false, true>(a, st);
  else launch_scored_bwd<D, false, false>(a, st);
}

}  // namespace rk

using namespace rk;

extern "C" int64_t rk_scored_attention_backward_work(int64_t B, int64_t H, int64_t Hkv, int64_t S,
                                                     int64_t D, int slopes) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || S <= 0 || D <= 0 || H % Hkv != 0) return 0;
  const int64_t parts = head_parts(B, H, Hkv, S);
  return (slopes ? 3 : 2) * B * H * ((S + kAttnRows - 1) / kAttnRows * kAttnRows) +
         (parts > 1 ? parts * 2 * B * Hkv * S * D : 0);
}

extern "C" int rk_scored_attention_backward(const rk_scored_attention_args* args, float* work,
                                            void* stream) {
  clear_error();
  if (!args) return fail(RK_ERR_ARG, "null arguments");
  const rk_scored_attention_args& p = *args;
  if (int e = check_scored(p, true)) return e;
  if (p.dslopes && !p.slopes) return fail(RK_ERR_ARG, "a slope gradient needs slopes");
  if (p.H == 0 && p.Hkv > 0 && p.B > 0 && p.S > 0)
    return fail(RK_ERR_ARG, "no query heads: dk and dv would not be written");
  if (p.B == 0 || p.H == 0 || p.S == 0) return RK_OK;
  if (!p.dq || !p.dk || !p.dv || !work) return fail(RK_ERR_ARG, "null pointer");
  if (!aligned16(work)) return fail(RK_ERR_UNSUPPORTED, "the workspace needs 16-byte alignment");
  const void* out8[] = {p.dq, p.dk, p.dv};
  for (const void* t : out8)
    if (reinterpret_cast<uintptr_t>(t) & 7)
      return fail(RK_ERR_UNSUPPORTED, "dq, dk, dv need 8-byte alignment");
  ScoredBwdArgs a{};
  a.f = scored_args(p);
  a.inv_scale = 1.0f / p.scale;
  a.rows = work;
  a.slope_rows = p.dslopes ? work + 2 * p.B * p.H * a.f.Sp : nullptr;
  a.parts = head_parts(p.B, p.H, p.Hkv, p.S);
  a.part_rows = work + (p.dslopes ? 3 : 2) * p.B * p.H * a.f.Sp;
  if (a.parts > 1 && p.B * p.Hkv > 65535)
    return fail(RK_ERR_UNSUPPORTED, "more than 65535 sequence heads");
  if (p.D == 64) dispatch_scored_bwd<64>(a, as_stream(stream));
  else dispatch_scored_bwd<128>(a, as_stream(stream));
  return launch_status("scored_attention_backward");
}

// Causal self-attention whose scores are capped by a tanh, biased by the distance and masked by
// documents and their prefixes: the mask's plan and the forward (gfx950). It stands beside
// rk_attention_forward (model.py:117-123 attends without any of them) and shares its layout:
//   s_ij = scale q_i . k_j,  s = cap tanh(s / cap),  s -= slope_h |i - j|,
//   o_i = sum_j softmax_j(s_ij over the keys that i sees) v_j,  lse_i = log sum_j exp(s_ij).
// A query that sees nothing gets o = 0. Query head h reads key head h / (H / Hkv).
//
// One workgroup = 128 queries of a head, one wavefront = 32, one lane = half the keys of one
// query (rk_attention.hip describes the products). What differs:
//  * the key range comes from the queries' intervals, so tiles outside every document of the
//    workgroup are neither loaded nor computed; a wavefront skips tiles none of its rows sees and
//    tests elements only in tiles that some row does not see whole;
//  * capped or biased scores are modified before the running max, in base-2 units (rk_scored.h).
//
// B 8, H 16, S 1024, D 128: causal 68 us (34 GFLOP, 510 TFLOP/s; rk_attention_forward 55-60), in
// documents of 400 on average 44, with capped scores 69 and 50; B 32, H 8, S 512, D 64 in
// documents of 150 20.6 us, where reading q, k, v and writing o and its rest takes 16 at 5.3 TB/s.
// The vector unit is busy two fifths of the time (719 instructions a step of 64 keys, capped), the
// matrix unit an eighth: what is left is waiting between a step's dependent parts, and
// wavefronts of a workgroup that wait for the one whose rows see most.
#include "rk_scored.h"

namespace rk {

__device__ __forceinline__ float half_max2(float v) {
  const uint32_t b = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum2(float v) {
  const uint32_t b = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// R keys are staged per step, U of them make one update of the running max and sum.
// FINE: capped and biased scores of a pass whose gradients are wanted (near_capped).
// (Without a running max under a cap, relative to a reference known beforehand: 52 -> 49.8 us of
// the capped training shape, 288 -> 257 capped and biased at S 8192. But the largest p of a row
// is then no longer 1 and exact in bf16: gradients off by 2.6e-3 against 2.4e-3. Not kept.)
template <int D, int R, int U, bool CAP, bool BIAS, bool FINE = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 4)))
void scored_fwd_kernel(ScoredArgs a) {
  using T = AttnTile<D, R>;
  constexpr int UT = U / 32;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kAttnStages * 2 * T::BYTES];
  __shared__ int box[8];
  const uint32_t lds0 = lds_address(smem);
  const rk_scored_attention_args& p = a.p;
  const int S = static_cast<int>(p.S);
  const int nqb = (S + kAttnRows - 1) / kAttnRows;
  // 32-bit divisions (the host bounds the grid)
  const uint32_t blk = blockIdx.x / a.BH, ubh = blockIdx.x - blk * a.BH, ub = ubh / a.H;
  const int qb = nqb - 1 - static_cast<int>(blk);  // longest causal rows first; heads fastest
  const int64_t bh = ubh, b = ub, hd = ubh - ub * a.H, kvh = (ubh - ub * a.H) / a.G;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw0 = qb * kAttnRows + 32 * wave, qi = qw0 + l32;  // this lane's query

  v8bf_a qf[D / 16];
  load_owned<D>(qf, p.q + b * p.sqb + hd * p.sqh, p.sqs, S, qi, h);
  const TileDma<D, R> kd(p.k + b * p.skb + kvh * p.skh, p.sks, S, wave, lane);
  const TileDma<D, R> vd(p.v + b * p.svb + kvh * p.svh, p.svs, S, wave, lane);
  Span span = row_span(p, 0, b, qi);
  const WaveSpan ws(span);
  int lo, hi;
  block_range(ws, wave, lane, box, lo, hi);
  const int first = lo < hi ? lo / R : 0, end = lo < hi ? (hi + R - 1) / R : 0;
  const uint32_t width = static_cast<uint32_t>(span.hi - span.lo);
  float slope2 = 0.0f;
  if constexpr (BIAS) slope2 = p.slopes[hd] * kLog2e;

  auto issue = [&](int step) {
    const uint32_t st = lds0 + (step & 1) * 2 * T::BYTES;
    kd.issue(st, step * R, wave);
    vd.issue(st + T::BYTES, step * R, wave);
  };

  float m = -INFINITY, l = 0.0f;
  v16f_a o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) o[dt] = v16f_a{};
  if (first < end) issue(first);
  for (int step = first; step < end; ++step) {
    const uint64_t pad = padding_bits<R>(a, b, step * R);
    dma_wait_barrier<0>();
    if (step + 1 < end) issue(step + 1);
    uint8_t* const kt = smem + (step & 1) * 2 * T::BYTES;
    uint8_t* const vt = kt + T::BYTES;
    if (pad) {
      clear_rows<D, R>(vt, pad, tid);
      __syncthreads();
    }
    const int k0 = step * R;
    if (ws.none(k0, R)) continue;
    // S^T: lane holds keys k0 + 32 t + 8 (e / 4) + 4 h + e % 4 of its query
    v16f_a sc[R / 32];
#pragma unroll
    for (int t = 0; t < R / 32; ++t) {
      sc[t] = v16f_a{};
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
        sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<D>(kt, 32 * t, s, lane), qf[s],
                                                        sc[t], 0, 0, 0);
    }
    // capped and biased scores in base-2 units here; plain ones are scaled with the max
    const float mul = CAP || BIAS ? 1.0f : a.dot_scale;
    if constexpr (CAP || BIAS) {
      const float d0 = static_cast<float>(qi - k0 - 4 * h);
      bool near = false;
      if constexpr (FINE) {
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < R / 32; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(sc[t][e]));
        near = !__any(most > a.near_limit);
      }
      if (near) {
#pragma unroll
        for (int t = 0; t < R / 32; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float slack;
            sc[t][e] = __builtin_fmaf(-slope2, fabsf(d0 - (32 * t + 8 * (e / 4) + (e % 4))),
                                      near_capped(a, sc[t][e], slack));
          }
      } else {
#pragma unroll
        for (int t = 0; t < R / 32; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x = sc[t][e] * a.dot_scale;
            if constexpr (CAP) {
              const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x) + 1.0f);
              x = __builtin_fmaf(-2.0f * a.cap2, r, a.cap2);
            }
            if constexpr (BIAS)
              x = __builtin_fmaf(-slope2, fabsf(d0 - (32 * t + 8 * (e / 4) + (e % 4))), x);
            sc[t][e] = x;
          }
      }
    }
    if (!ws.all(k0, R)) {
      const int j0 = k0 + 4 * h - span.lo;
#pragma unroll
      for (int t = 0; t < R / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (static_cast<uint32_t>(j0 + 32 * t + 8 * (e / 4) + (e % 4)) >= width)
            sc[t][e] = -INFINITY;
    }
    // the updates' probabilities first, then their products
    float alpha[R / U], ps[R / U];
    uint4 pf[R / 32][2];
#pragma unroll
    for (int u = 0; u < R / U; ++u) {
      float mx = -INFINITY;
#pragma unroll
      for (int t = u * UT; t < (u + 1) * UT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[t][e]);
      mx = half_max2(mx);
      const float mnew = fmaxf(m, mx * mul);
      const float mref = mnew == -INFINITY ? 0.0f : mnew;  // a row with no key yet
      alpha[u] = __builtin_amdgcn_exp2f(m - mref);
      m = mnew;
      ps[u] = 0.0f;
#pragma unroll
      for (int t = u * UT; t < (u + 1) * UT; ++t) {
        float pr[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          pr[e] = __builtin_amdgcn_exp2f(CAP || BIAS ? sc[t][e] - mref
                                                     : __builtin_fmaf(sc[t][e], mul, -mref));
          ps[u] = ps[u] + pr[e];
        }
        pack16(pf[t], pr);
      }
    }
#pragma unroll
    for (int u = 0; u < R / U; ++u) {
      // keys that no row of the wavefront sees: every p is zero, but their values may not be finite
      if (ws.none(k0 + u * U, U)) continue;
      if (__any(alpha[u] != 1.0f)) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * alpha[u];
      }
      l = l * alpha[u] + half_sum2(ps[u]);
#pragma unroll
      for (int t = u * UT; t < (u + 1) * UT; ++t)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                col_frag<D>(vt, 32 * t + 16 * s2, dt, lane), frag_of(pf[t][s2]), o[dt], 0, 0, 0);
    }
  }

  uint32_t* const rest = p.rest ? rest_words<D>(a, bh, qw0) + lane : nullptr;
  if (qi >= S && rest) {
#pragma unroll
    for (int r = 0; r < D / 8; ++r) rest[64 * r] = 0;
  }
  if (qi < S) {
    if (!span.valid) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] = v16f_a{};
    }
    const float factor = span.valid ? 1.0f / l : 0.0f;
    uint16_t* const row = p.o + b * p.sob + hd * p.soh + static_cast<int64_t>(qi) * p.sos;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x[4] = {o[dt][4 * r] * factor, o[dt][4 * r + 1] * factor,
                            o[dt][4 * r + 2] * factor, o[dt][4 * r + 3] * factor};
        const uint32_t lo = bf16_pair(x[0], x[1]), hi = bf16_pair(x[2], x[3]);
        *reinterpret_cast<uint2*>(row + 32 * dt + 8 * r + 4 * h) = make_uint2(lo, hi);
        if (rest) rest[64 * (4 * dt + r)] = bf16_rest4(x, lo, hi);
      }
    if (h == 0)
      p.lse[bh * S + qi] = span.valid ? (m + __log2f(l)) * 0.69314718055994531f : 0.0f;
  }
}

// ---------------------------------------------------------------------------
// The plan: one workgroup per row, a thread 8 consecutive positions of a chunk of 8 * NT, scans
// over the threads' values by wavefront shuffles. From the left: the document's first position and
// whether the run of marked positions it begins with reaches here; from the right: the
// document's end and the end of that run. Up to one chunk the first pass stays in registers.
// (In 8-byte loads and stores of one position each, and through memory between the passes, a row
// of 8192 positions took 39 us; 11 this way.)
// ---------------------------------------------------------------------------
constexpr int kMaskEach = 8;

struct MaskArgs {
  const void* documents;  // int32 or int64 [B, S], or null (one document per row)
  int wide;
  const uint8_t* prefix;  // [B, S] 0 / 1, or null
  int64_t sdb, spb;       // row strides
  int64_t B, S, S32;
  int32_t* bounds;        // [4][B][S]
  uint8_t* padding;       // [B][S32][4]
};

// Two max scans over the threads of the workgroup, left to right or (BACK) right to left: each
// thread's x, y become those of the threads before it, tx, ty those of all. box: 2 NT / 64 ints.
template <int NT, bool BACK>
__device__ __forceinline__ void block_scan_max(int& x, int& y, int& tx, int& ty, int* box,
                                               int tid) {
  constexpr int NW = NT / 64, kNone = -0x7fffffff;
  const int lane = tid & 63, wave = tid >> 6;
  const int turn = BACK ? 63 - lane : lane, place = BACK ? NW - 1 - wave : wave;
  const auto before = [&](int v, int d) {
    return BACK ? __shfl_down(v, d, 64) : __shfl_up(v, d, 64);
  };
  int a = x, c = y;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int oa = before(a, d), oc = before(c, d);
    if (turn >= d) {
      a = a > oa ? a : oa;
      c = c > oc ? c : oc;
    }
  }
  __syncthreads();
  if (turn == 63) {
    box[place] = a;
    box[NW + place] = c;
  }
  __syncthreads();
  int ea = before(a, 1), ec = before(c, 1);
  if (turn == 0) ea = ec = kNone;
  tx = ty = kNone;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int ba = box[w], bc = box[NW + w];
    if (w < place) {
      ea = ea > ba ? ea : ba;
      ec = ec > bc ? ec : bc;
    }
    tx = tx > ba ? tx : ba;
    ty = ty > bc ? ty : bc;
  }
  x = ea;
  y = ec;
}

// 4-byte aligned vectors (rows of any length)
typedef int32_t v4i_u __attribute__((ext_vector_type(4), aligned(4)));
typedef int64_t v2l_u __attribute__((ext_vector_type(2), aligned(8)));

__device__ __forceinline__ int64_t document_of(const MaskArgs& a, int64_t b, int64_t i) {
  if (!a.documents) return 0;
  return a.wide ? static_cast<const int64_t*>(a.documents)[b * a.sdb + i]
                : static_cast<const int32_t*>(a.documents)[b * a.sdb + i];
}

// Ids of positions i0 .. i0 + 7 (-1 past the row).
__device__ __forceinline__ void documents_of(const MaskArgs& a, int64_t b, int i0, int S,
                                             int64_t (&id)[kMaskEach]) {
  if (a.documents && i0 + kMaskEach <= S) {
    if (a.wide) {
      const int64_t* at = static_cast<const int64_t*>(a.documents) + b * a.sdb + i0;
#pragma unroll
      for (int e = 0; e < kMaskEach; e += 2) {
        const v2l_u v = *reinterpret_cast<const v2l_u*>(at + e);
        id[e] = v.x;
        id[e + 1] = v.y;
      }
    } else {
      const int32_t* at = static_cast<const int32_t*>(a.documents) + b * a.sdb + i0;
#pragma unroll
      for (int e = 0; e < kMaskEach; e += 4) {
        const v4i_u v = *reinterpret_cast<const v4i_u*>(at + e);
        id[e] = v.x;
        id[e + 1] = v.y;
        id[e + 2] = v.z;
        id[e + 3] = v.w;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kMaskEach; ++e) id[e] = i0 + e < S ? document_of(a, b, i0 + e) : -1;
  }
}

__device__ __forceinline__ void store8(int32_t* to, const int (&v)[kMaskEach], int n) {
  if (n >= kMaskEach) {
    *reinterpret_cast<v4i_u*>(to) = v4i_u{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<v4i_u*>(to + 4) = v4i_u{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int e = 0; e < kMaskEach; ++e)
      if (e < n) to[e] = v[e];
  }
}

template <int NT>
__global__ __launch_bounds__(NT) void attention_mask_kernel(MaskArgs a) {
  constexpr int CHUNK = NT * kMaskEach, kNone = -0x7fffffff;
  __shared__ int box[2 * NT / 64];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, S = static_cast<int>(a.S);
  const int chunks = (S + CHUNK - 1) / CHUNK;
  int32_t* const key_lo = a.bounds + b * a.S;
  int32_t* const key_hi = key_lo + a.B * a.S;
  int32_t* const query_lo = key_hi + a.B * a.S;
  int32_t* const query_hi = query_lo + a.B * a.S;
  // left to right: the document's first position; bits: marked beginning, not padding
  int lo[kMaskEach] = {};
  uint32_t lead = 0, real = 0;
  int begin0 = 0, broken0 = -1;
  for (int c = 0; c < chunks; ++c) {
    const int i0 = c * CHUNK + tid * kMaskEach;
    int broken[kMaskEach] = {};
    int bx = kNone, by = kNone;
    lead = real = 0;
    if (i0 < S) {
      int64_t id[kMaskEach];
      documents_of(a, b, i0, S, id);
      int64_t before = i0 > 0 ? document_of(a, b, i0 - 1) : 0;
      uint32_t marks = 0;
#pragma unroll
      for (int e = 0; e < kMaskEach; ++e)
        marks |= static_cast<uint32_t>(a.prefix && i0 + e < S && a.prefix[b * a.spb + i0 + e]) << e;
#pragma unroll
      for (int e = 0; e < kMaskEach; ++e) {
        const int i = i0 + e;
        if (i == 0 || id[e] != before) bx = i;
        if (!(marks >> e & 1)) by = i;
        before = id[e];
        real |= static_cast<uint32_t>(i < S && id[e] >= 0) << e;
        lo[e] = bx;
        broken[e] = by;
      }
    }
    if (i0 < a.S32 * 32) {
      const uint32_t inside = S - i0 >= 8 ? 0xffu : S > i0 ? (1u << (S - i0)) - 1u : 0u;
      a.padding[b * a.S32 * 4 + i0 / 8] = static_cast<uint8_t>(~real & inside);
    }
    int ex = bx, ey = by, tx, ty;
    block_scan_max<NT, false>(ex, ey, tx, ty, box, tid);
    ex = ex > begin0 ? ex : begin0;
    ey = ey > broken0 ? ey : broken0;
#pragma unroll
    for (int e = 0; e < kMaskEach; ++e) {
      lo[e] = lo[e] > ex ? lo[e] : ex;
      const int br = broken[e] > ey ? broken[e] : ey;
      lead |= static_cast<uint32_t>(br < lo[e]) << e;
    }
    begin0 = tx > begin0 ? tx : begin0;
    broken0 = ty > broken0 ? ty : broken0;
    if (chunks > 1) {  // the same thread takes them up again
      store8(key_lo + i0, lo, S - i0);
      if (i0 < S) key_hi[i0] = static_cast<int>(lead | real << 8);
    }
  }
  // right to left, as a max scan of negated positions: the least later position where a
  // document begins (its end), and where one begins or the marked run is over
  int end0 = -S, stop0 = -S;
  for (int c = chunks - 1; c >= 0; --c) {
    const int i0 = c * CHUNK + tid * kMaskEach;
    if (chunks > 1 && i0 < S) {
#pragma unroll
      for (int e = 0; e < kMaskEach; ++e) lo[e] = i0 + e < S ? key_lo[i0 + e] : 0;
      lead = static_cast<uint32_t>(key_hi[i0]);
      real = lead >> 8;
    }
    int end[kMaskEach], stop[kMaskEach];
    int bx = kNone, by = kNone;
#pragma unroll
    for (int e = kMaskEach - 1; e >= 0; --e) {
      const int i = i0 + e;
      end[e] = bx;  // over the later positions of this thread
      stop[e] = by;
      if (i < S) {
        if (lo[e] == i) bx = -i;
        if (lo[e] == i || !(lead >> e & 1)) by = -i;
      }
    }
    int ex = bx, ey = by, tx, ty;
    block_scan_max<NT, true>(ex, ey, tx, ty, box, tid);
    ex = ex > end0 ? ex : end0;
    ey = ey > stop0 ? ey : stop0;
    int v[4][kMaskEach];
#pragma unroll
    for (int e = 0; e < kMaskEach; ++e) {
      const int i = i0 + e;
      const int en = -(end[e] > ex ? end[e] : ex), st = -(stop[e] > ey ? stop[e] : ey);
      const bool r = real >> e & 1, ld = lead >> e & 1;
      v[0][e] = r ? lo[e] : 0;
      v[1][e] = r ? (ld ? st : i + 1) : 0;
      v[2][e] = r ? (ld ? lo[e] : i) : 0;
      v[3][e] = r ? en : 0;
    }
    if (i0 < S) {
      store8(key_lo + i0, v[0], S - i0);
      store8(key_hi + i0, v[1], S - i0);
      store8(query_lo + i0, v[2], S - i0);
      store8(query_hi + i0, v[3], S - i0);
    }
    end0 = tx > end0 ? tx : end0;
    stop0 = ty > stop0 ? ty : stop0;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_scored(const rk_scored_attention_args& p, bool backward) {
  if (p.B < 0 || p.H < 0 || p.Hkv < 0 || p.S < 0) return fail(RK_ERR_ARG, "negative size");
  if (p.D != 64 && p.D != 128)
    return fail(RK_ERR_UNSUPPORTED, "head size %lld (64 or 128 only)", static_cast<long long>(p.D));
  if (p.B == 0 || p.H == 0 || p.S == 0) return RK_OK;
  if (p.Hkv == 0 || p.H % p.Hkv != 0)
    return fail(RK_ERR_ARG, "query heads must be a multiple of the key heads");
  if (!(p.scale > 0.0f) || !(p.scale < INFINITY))
    return fail(RK_ERR_ARG, "scale must be positive and finite");
  if (!(p.softcap >= 0.0f) || !(p.softcap < INFINITY))
    return fail(RK_ERR_ARG, "softcap must be finite and not negative (0: none)");
  if (p.softcap != 0.0f && !(p.softcap >= 1e-3f && p.softcap <= 1e3f))
    return fail(RK_ERR_UNSUPPORTED, "softcap outside 1e-3 .. 1e3");
  if (!p.q || !p.k || !p.v || !p.o || !p.lse) return fail(RK_ERR_ARG, "null pointer");
  if (p.bounds && p.mask_batch != 1 && p.mask_batch != p.B)
    return fail(RK_ERR_ARG, "a mask holds one row or one per sequence");
  if ((p.bounds == nullptr) != (p.padding == nullptr))
    return fail(RK_ERR_ARG, "a mask's intervals and padding bits go together");
  if (reinterpret_cast<uintptr_t>(p.rest) & 3)
    return fail(RK_ERR_UNSUPPORTED, "rest needs 4-byte alignment");
  const void* in16[] = {p.q, p.k, p.v, backward ? p.o : p.q, backward ? p.g : p.q};
  for (const void* t : in16)
    if (!t || !aligned16(t)) return fail(RK_ERR_UNSUPPORTED, "operands need 16-byte alignment");
  const int64_t strides[] = {p.sqb, p.sqh, p.sqs, p.skb, p.skh, p.sks, p.svb, p.svh, p.svs,
                             p.sob, p.soh, p.sos, backward ? p.sgb : 0, backward ? p.sgh : 0,
                             backward ? p.sgs : 0, backward ? p.sxb : 0, backward ? p.sxh : 0,
                             backward ? p.sxs : 0, backward ? p.syb : 0, backward ? p.syh : 0,
                             backward ? p.sys : 0};
  for (int64_t st : strides)
    if (st < 0 || st % 8 != 0)
      return fail(RK_ERR_UNSUPPORTED, "strides must be non-negative multiples of 8 elements");
  // buffer offsets are 32-bit: the rows of one head up to the last tile's end, and its row
  // statistics, lie below 2^31 bytes
  const int64_t rows[] = {p.sqs, p.sks, p.svs, backward ? p.sos : 0, backward ? p.sgs : 0};
  for (int64_t st : rows)
    if (st >= (int64_t{1} << 31) || ((p.S + 192) * st + p.D) * 2 >= (int64_t{1} << 31))
      return fail(RK_ERR_UNSUPPORTED, "sequence extent exceeds 2^31 bytes per head");
  const int64_t blocks = (p.S + kAttnRows - 1) / kAttnRows;
  if (p.S > (int64_t{1} << 27) || p.B > (int64_t{1} << 24) || p.H > (int64_t{1} << 24) ||
      p.B * p.H >= (int64_t{1} << 24) || p.B * p.H * blocks >= (int64_t{1} << 24))
    return fail(RK_ERR_UNSUPPORTED, "2^24 blocks of 128 positions and more");
  return RK_OK;
}

ScoredArgs scored_args(const rk_scored_attention_args& p) {
  ScoredArgs a{};
  a.p = p;
  a.BH = static_cast<uint32_t>(p.B * p.H);
  a.H = static_cast<uint32_t>(p.H);
  a.G = static_cast<uint32_t>(p.H / p.Hkv);
  a.S32 = (p.S + 31) / 32;
  a.Sp = (p.S + kAttnRows - 1) / kAttnRows * kAttnRows;
  const bool cap = p.softcap > 0.0f;
  a.dot_scale = cap ? 2.0f * kLog2e * (p.scale / p.softcap) : p.scale * kLog2e;
  a.cap2 = p.softcap * kLog2e;
  if (cap) {
    const double c2 = static_cast<double>(a.cap2), step = 1.0 / (c2 * c2);
    const double fit[4] = {-0.3333323001861572, 0.13327749073505402, -0.053165826946496964,
                           0.0174802765250206};
    double power = step;
    for (int i = 0; i < 4; ++i, power *= step) a.near[i] = static_cast<float>(fit[i] * power);
    a.near_scale = p.scale * kLog2e;
    a.near_limit = 0.5f * p.softcap / p.scale;
    a.inv_cap2 = static_cast<float>(1.0 / c2);
  }
  return a;
}

template <int D, int R, int U>
static void launch_scored_fwd(const ScoredArgs& a, dim3 grid, hipStream_t st) {
  const bool cap = a.p.softcap > 0.0f, bias = a.p.slopes != nullptr;
  if (cap && bias && a.p.rest)
    scored_fwd_kernel<D, R, U, true, true, true><<<grid, 256, 0, st>>>(a);
  else if (cap && bias) scored_fwd_kernel<D, R, U, true, true><<<grid, 256, 0, st>>>(a);
  else if (cap) scored_fwd_kernel<D, R, U, true, false><<<grid, 256, 0, st>>>(a);
  else if (bias) scored_fwd_kernel<D, R, U, false, true><<<grid, 256, 0, st>>>(a);
  else scored_fwd_kernel<D, R, U, false, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace rk

using namespace rk;

extern "C" int64_t rk_scored_attention_rest(int64_t B, int64_t H, int64_t S, int64_t D) {
  if (B <= 0 || H <= 0 || S <= 0 || D <= 0) return 0;
  return B * H * ((S + kAttnRows - 1) / kAttnRows * kAttnRows) * D;
}

extern "C" int rk_scored_attention_forward(const rk_scored_attention_args* args, void* stream) {
  clear_error();
  if (!args) return fail(RK_ERR_ARG, "null arguments");
  const rk_scored_attention_args& p = *args;
  if (int e = check_scored(p, false)) return e;
  if (p.B == 0 || p.H == 0 || p.S == 0) return RK_OK;
  if (reinterpret_cast<uintptr_t>(p.o) & 7)
    return fail(RK_ERR_UNSUPPORTED, "o needs 8-byte alignment");
  const ScoredArgs a = scored_args(p);
  const dim3 grid(static_cast<unsigned>(p.B * p.H * (a.Sp / kAttnRows)));
  if (p.D == 64) launch_scored_fwd<64, 64, 64>(a, grid, as_stream(stream));
  else launch_scored_fwd<128, 64, 32>(a, grid, as_stream(stream));
  return launch_status("scored_attention_forward");
}

extern "C" int rk_attention_mask(const void* documents, int wide, int64_t sdb,
                                 const uint8_t* prefix, int64_t spb, int64_t B, int64_t S,
                                 int32_t* bounds, uint32_t* padding, void* stream) {
  clear_error();
  if (B < 0 || S < 0) return fail(RK_ERR_ARG, "negative size");
  if (B == 0 || S == 0) return RK_OK;
  if (!bounds || !padding) return fail(RK_ERR_ARG, "null pointer");
  if (B > 0x7fffff || S > (int64_t{1} << 27)) return fail(RK_ERR_UNSUPPORTED, "mask too large");
  const int64_t S32 = (S + 31) / 32;
  MaskArgs a{documents, wide, prefix, sdb, spb, B, S, S32, bounds,
             reinterpret_cast<uint8_t*>(padding)};
  const unsigned grid = static_cast<unsigned>(B);
  if (S <= 256 * kMaskEach) attention_mask_kernel<256><<<grid, 256, 0, as_stream(stream)>>>(a);
  else attention_mask_kernel<1024><<<grid, 1024, 0, as_stream(stream)>>>(a);
  return launch_status("attention_mask");
}

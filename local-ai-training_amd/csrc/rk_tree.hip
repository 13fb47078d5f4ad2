// Attention for a tree of drafted tokens over the 8-bit cache (gfx950), and the tree's plan. The
// reference drafts nothing (generate.py:183-201 runs the window for every token).
//
// Node i of a sequence with `start` cached tokens stands at position start + depth_i. It sees the
// cached tokens and its own way from the root: itself and its ancestors, whose keys and values lie
// beside the cache (only those that are accepted are appended to it).
//   s_j = scale q . k_j;  capped and biased as in rk_scored.h;  o = sum_j softmax(s_j) v_j
#include "rk_kv8.h"
#include "rk_tree.h"

#include <math.h>

#include <type_traits>

namespace rk {

// ---------------------------------------------------------------------------
// The plan: grid (trees), 256 threads; thread i walks from node i to the root. A launch's latency
// bounds it (16 trees of 32 nodes: 4.6 us).
// ---------------------------------------------------------------------------
struct TreePlan {
  const void* parents;  // int32 or int64 [R][N], row stride ldp
  int wide;
  int64_t ldp, N, W;
  int32_t* kept;    // [R][N]: the parents, -1 for the root, kTreeOff for nodes that are off
  int32_t* depths;  // [R][N]
  uint64_t* seen;   // [R][N][W]
};

__global__ __launch_bounds__(kTreeNodes) void draft_tree_kernel(TreePlan a) {
  __shared__ int parent[kTreeNodes];
  const int i = threadIdx.x;
  const int64_t r = blockIdx.x;
  if (i < a.N) {
    const int64_t p = a.wide ? static_cast<const int64_t*>(a.parents)[r * a.ldp + i]
                             : static_cast<const int32_t*>(a.parents)[r * a.ldp + i];
    // a root is node 0, any other node's parent comes before it
    const bool ok = i == 0 ? p == -1 : p >= 0 && p < i;
    parent[i] = ok ? static_cast<int>(p) : kTreeOff;
  }
  __syncthreads();
  if (i >= a.N) return;
  uint64_t bits[kTreeNodes / 64] = {};
  int depth = -1, at = i;
  while (at >= 0) {  // strictly down
    bits[0] |= at < 64 ? 1ull << (at & 63) : 0;
    bits[1] |= at >= 64 && at < 128 ? 1ull << (at & 63) : 0;
    bits[2] |= at >= 128 && at < 192 ? 1ull << (at & 63) : 0;
    bits[3] |= at >= 192 ? 1ull << (at & 63) : 0;
    ++depth;
    at = parent[at];
  }
  const bool off = at == kTreeOff;
  a.kept[r * a.N + i] = off ? kTreeOff : parent[i];
  a.depths[r * a.N + i] = off ? 0 : depth;
  for (int w = 0; w < a.W; ++w) a.seen[(r * a.N + i) * a.W + w] = off ? 0 : bits[w];
}

// ---------------------------------------------------------------------------
// Attention. The first launch takes the cached tokens, the second joins its parts and adds the
// nodes a column sees.
//
// Columns of a product are the N * G queries that share a key head (G = query heads per key head);
// a wavefront holds CT tiles of 16 of them and walks blocks of 64 tokens with its own running max,
// sum and output, so that a block's codes are loaded and widened to bf16 (which holds them exactly)
// once for all its columns. Lane l holds the scores of column l % 16 against keys
// 16 (l / 16) .. + 15: key 16 g + 4 t + e is row 4 g + e of product t, and the same 16 keys are
// the lane's k slots of the second product (8 for each half), whose other operand, 16 tokens of one
// feature, lies side by side in the cache. bf16 queries enter as they are, float32 ones as sums of
// three bf16 numbers; probabilities as sums of three for float32 results and of two (2^-16 of
// themselves) for bf16 ones, whatever the tree's size. (One, 2^-8 of themselves, beside more than 32
// columns took 116 us where two take 137 at 64 nodes of 8 query heads a key head, and left a result off
// by 2.2e-3 of the norm instead of the 1.7e-3 of its own rounding.)
//
// What bounds it: up to 32 columns, the cache's bytes (16 sequences of 2.7 to 8 thousand tokens, 16 heads
// of 128, 32 nodes: 349 MB in 82 us, 4.3 TB/s of the 5.0 that a copy reaches); with more, vector
// instructions (8 sequences of 6 to 15 thousand, 32 heads of 64 on 4, 64 nodes, capped: 137 us a call;
// the two products alone, 38 us at the rate of a large matrix product). Of a block and two tiles of
// columns a lane widens 128 codes with 192 instructions, 6 for each of its 32 scores, more than a cap (5), an
// exponential (1) or the two roundings (3) take; every two tiles widen the block anew. Few tokens: the
// latency of one pass, 5 us at 300. Two tiles of columns a wavefront: the codes are widened once for both;
// four spill or leave one wavefront a SIMD (172 us where two took 147). The join takes 4 us for a few
// rows, 14 for 16384 columns.
// ---------------------------------------------------------------------------
struct TreeAttn {
  Kv8 c;
  const void *q, *k, *v;
  int64_t sqb, sqh, sqs, skb, skh, sks, svb, svh, svs;
  const int64_t* start;
  const int64_t* lengths;
  const uint64_t* seen;
  const int32_t* depths;
  const float* slopes;
  int64_t start_step, tree_step, N, W, Hq, G, nsplit, tiles;
  float dot_scale;        // scale log2(e)
  float cap2, inv_cap2;   // cap log2(e); 0: none
  float near[3];          // tree_near
  float* work;  // [B * H][N * G][nsplit][D + 4]: max, sum, 2 pad, unnormalized output
  void* out;    // [B, N, Hq, D]
};

// The capped score C tanh(y / C) of a score y, both in base-2 units, C = cap log2(e). The exponential
// form is off by a few 2^-24 of C whatever the score; where float32 results show it (FINE), scores of
// up to a third of the cap take tanh's series (its next term is below 2^-26 there).
template <bool FINE>
__device__ __forceinline__ float tree_capped(float y, float cap2, float inv_cap2) {
  const float u = y * inv_cap2;
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(u * (2.0f * kLog2e8)) + 1.0f);
  float t = __builtin_fmaf(-2.0f * cap2, r, cap2);
  if constexpr (FINE) {
    const float z = u * u;
    float s = __builtin_fmaf(z, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    s = __builtin_fmaf(z, s, -17.0f / 315.0f);
    s = __builtin_fmaf(z, s, 2.0f / 15.0f);
    s = __builtin_fmaf(z, s, -1.0f / 3.0f);
    t = fabsf(u) < 0.34f ? __builtin_fmaf(y * z, s, y) : t;
  }
  return t;
}
// The same for |y| <= kNear C by y (1 + z (c0 + c1 z + c2 z^2)), z = y^2: half the instructions (64 nodes
// of 8 query heads a key head: 146 us with the exponential form, 137 with this one). The host interpolates
// (tanh(u) / u - 1) / u^2 at Chebyshev nodes of u^2 (off by at most 4.0e-7 of the score, at kNear).
constexpr float kNear = 0.4f;
__device__ __forceinline__ float tree_near(float y, const float (&c)[3]) {
  const float z = y * y;
  float s = __builtin_fmaf(z, c[2], c[1]);
  s = __builtin_fmaf(z, s, c[0]);
  return __builtin_fmaf(y, z * s, y);
}

// What is done to the scores: nothing; a cap of so little (kBounded) that their exponentials need no
// maximum, 2^60 being the most (155 us with the maximum, 137 without, at 64 nodes of 8 query heads a key
// head); a cap, a bias or both.
enum { kPlain, kBounded, kModified };
constexpr float kBound = 60.0f;

template <int D, int CT, int QDT, int ODT, int MODE>
__global__ __launch_bounds__(256) void tree_cache_kernel(TreeAttn a) {
  constexpr int KK = D / 64, FT = D / 16, NW = 4;
  constexpr int QP = QDT == RK_F32 ? 3 : 1;
  constexpr bool FINE = ODT == RK_F32;
  constexpr int NP = FINE ? 3 : 2;  // bf16 numbers of a probability
  __shared__ float box[2][CT * (4 * FT + 2)][64];
  const int split = blockIdx.x;
  const int64_t tile = blockIdx.y, bh = blockIdx.z;
  const uint32_t uh = static_cast<uint32_t>(a.c.H), ub = blockIdx.z / uh;  // 32-bit divisions
  const int64_t b = ub, kvh = blockIdx.z - ub * uh;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t start = a.start[b * a.start_step];
  const int64_t cols = a.N * a.G;
  const uint32_t ug = static_cast<uint32_t>(a.G);
  int64_t nb = start > 0 ? (start + kTok - 1) >> 6 : 0;
  nb = nb < a.c.NB ? nb : a.c.NB;
  const int64_t per = (static_cast<uint32_t>(nb) + static_cast<uint32_t>(a.nsplit) - 1) /
                      static_cast<uint32_t>(a.nsplit);
  const int64_t j0 = split * per, j1 = j0 + per < nb ? j0 + per : nb;

  // the sum is a product too, of ones (its four rows are equal): the MFMAs have time for it
  float m[CT], o[CT][FT][4];
  v4f_a sums[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    m[c] = -INFINITY;
    sums[c] = v4f_a{};
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][f][e] = 0.0f;
  }

  if (j0 + wave < j1) {
    const int bytes = static_cast<int>(j1 - j0) * (kTok * D);  // the host bounds a head's codes
    const __amdgpu_buffer_rsrc_t kbuf =
        make_buffer(a.c.keys + (bh * a.c.NB + j0) * kTok * D, bytes);
    const __amdgpu_buffer_rsrc_t vbuf =
        make_buffer(a.c.values + (bh * a.c.NB + j0) * kTok * D, bytes);
    const float* const ks = a.c.ks + bh * a.c.NB;
    const float* const vs = a.c.vs + bh * a.c.NB;
    const int koff = (16 * (col >> 2) + (col & 3)) * D + 16 * g;  // row 4 g' + e' of product 0
    const int voff = col * kTok + 16 * g;
    v4i8 kf[4][KK], vf[FT];
    // loads past the split's last block return zeros without going to memory
    auto load_k = [&](int64_t j) {
      const int at = static_cast<int>(j - j0) * (kTok * D);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kf[t][kk] = __builtin_bit_cast(
              v4i8, __builtin_amdgcn_raw_buffer_load_b128(kbuf, koff + 4 * t * D + 64 * kk, at, 0));
    };
    auto load_v = [&](int64_t j) {
      const int at = static_cast<int>(j - j0) * (kTok * D);
#pragma unroll
      for (int f = 0; f < FT; ++f)
        vf[f] = __builtin_bit_cast(
            v4i8, __builtin_amdgcn_raw_buffer_load_b128(vbuf, voff + 16 * f * kTok, at, 0));
    };
    int64_t j = j0 + wave;
    load_k(j);
    load_v(j);
    // the queries: features 64 kk + 16 g .. + 15 of each tile's column
    v8bf_a qf[CT][QP][KK][2];
    float slope2[CT];
    int depth[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int64_t ct = (tile * CT + c) * 16 + col, cc = ct < cols ? ct : cols - 1;
      const int64_t i = static_cast<uint32_t>(cc) / ug, hd = kvh * a.G + (cc - i * a.G);
      const int64_t base = b * a.sqb + hd * a.sqh + i * a.sqs + 16 * g;
      slope2[c] = a.slopes ? a.slopes[hd] * kLog2e8 : 0.0f;
      depth[c] = a.depths[b * a.tree_step * a.N + i];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if constexpr (QDT == RK_BF16) {
          const uint4* const at =
              reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + base + 64 * kk);
          qf[c][0][kk][0] = frag_of(at[0]);
          qf[c][0][kk][1] = frag_of(at[1]);
        } else {
          float x[16];
#pragma unroll
          for (int v = 0; v < 4; ++v) load_vec16<QDT>(a.q, base + 64 * kk + 4 * v, x + 4 * v);
          v8bf_a part[3][2];
          split_bf16<3>(x, part);
#pragma unroll
          for (int n = 0; n < QP; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) qf[c][n][kk][u] = part[n][u];
        }
      }
    }
    const uint32_t one2 = 0x3f803f80u;
    const v8bf_a ones = frag_of(make_uint4(one2, one2, one2, one2));
    // widened codes: 16 features of a key, 16 tokens of a feature
    const auto widen = [](const v4i8& codes, v8bf_a (&to)[2]) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        widen_codes(static_cast<uint32_t>(codes[e]), w[2 * e], w[2 * e + 1]);
      to[0] = frag_of(make_uint4(w[0], w[1], w[2], w[3]));
      to[1] = frag_of(make_uint4(w[4], w[5], w[6], w[7]));
    };
    const auto product = [&](int c, const v8bf_a (&kw)[KK][2]) {
      v4f_a acc{};
#pragma unroll
      for (int n = QP - 1; n >= 0; --n)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kw[kk][u], qf[c][n][kk][u], acc, 0, 0, 0);
      return acc;
    };
    for (; j < j1; j += NW) {
      const float vscale = vs[j], mul = ks[j] * a.dot_scale;
      // key 16 g + x of the block is cached for x < left
      const int64_t ahead = start - (j * kTok + 16 * g);
      const int left = ahead > 16 ? 16 : ahead < 0 ? 0 : static_cast<int>(ahead);
      const bool whole = (j + 1) * kTok <= start;
      // a tile's probabilities from its scores, with the running maximum and sum
      const auto weigh = [&](int c, const v4f_a (&s)[4], v8bf_a (&p)[NP][2]) {
        float y[16];
        // plain scores are scaled with the subtraction of the maximum
        const float unit = MODE == kPlain ? mul : 1.0f;
#pragma unroll
        for (int x = 0; x < 16; ++x) y[x] = s[x / 4][x % 4] * (MODE == kPlain ? 1.0f : mul);
        if (MODE == kBounded || (MODE == kModified && a.cap2 != 0.0f)) {
          float far = 0.0f, raw[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) far = fmaxf(far, fabsf(y[x]));
          const bool near = !FINE && !__any(!(far <= kNear * a.cap2));
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            raw[x] = y[x];
            if constexpr (!FINE) y[x] = tree_near(y[x], a.near);
          }
          if (!near) {
#pragma unroll
            for (int x = 0; x < 16; ++x) y[x] = tree_capped<FINE>(raw[x], a.cap2, a.inv_cap2);
          }
        }
        if (MODE == kModified && a.slopes) {
          // (whole numbers: positions pass 2^24; a head's codes bound them to 2^25)
          const float d0 = static_cast<float>(static_cast<int>(ahead) + depth[c]);
#pragma unroll
          for (int x = 0; x < 16; ++x) y[x] = __builtin_fmaf(-slope2[c], d0 - x, y[x]);
        }
        if (!whole) {
#pragma unroll
          for (int x = 0; x < 16; ++x) y[x] = x < left ? y[x] : -INFINITY;
        }
        if constexpr (MODE == kBounded) {
          m[c] = 0.0f;
#pragma unroll
          for (int x = 0; x < 16; ++x) y[x] = __builtin_amdgcn_exp2f(y[x]);
        } else {
          float mx = y[0];
#pragma unroll
          for (int x = 1; x < 16; ++x) mx = fmaxf(mx, y[x]);
          mx = col_max(mx) * unit;
          const float mnew = fmaxf(m[c], mx), ref = mnew == -INFINITY ? 0.0f : mnew;
          const float alpha = __builtin_amdgcn_exp2f(m[c] - ref);
          m[c] = mnew;
#pragma unroll
          for (int x = 0; x < 16; ++x)
            y[x] = __builtin_amdgcn_exp2f(MODE == kPlain ? __builtin_fmaf(y[x], unit, -ref)
                                                         : y[x] - ref);
          if (MODE == kPlain && !whole) {  // (a zero key scale makes NaN of a masked score)
#pragma unroll
            for (int x = 0; x < 16; ++x) y[x] = x < left ? y[x] : 0.0f;
          }
          if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[c][e] = sums[c][e] * alpha;
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[c][f][e] = o[c][f][e] * alpha;
          }
        }
        split_bf16<NP>(y, p);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            sums[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[n][u], sums[c], 0, 0, 0);
      };
      const auto values = [&](int c, int f, const v8bf_a (&v)[2], const v8bf_a (&p)[NP][2]) {
        v4f_a acc{};
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], p[n][u], acc, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][f][e] = __builtin_fmaf(acc[e], vscale, o[c][f][e]);
      };
      if constexpr (D == 64) {
        // the widened block fits the registers: a tile at a time, one's products beside the next one's
        // exponentials
        v8bf_a kw[4][KK][2], vw[FT][2];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) widen(kf[t][kk], kw[t][kk]);
        load_k(j + NW);
#pragma unroll
        for (int f = 0; f < FT; ++f) widen(vf[f], vw[f]);
        load_v(j + NW);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          v4f_a s[4];
          v8bf_a p[NP][2];
#pragma unroll
          for (int t = 0; t < 4; ++t) s[t] = product(c, kw[t]);
          weigh(c, s, p);
#pragma unroll
          for (int f = 0; f < FT; ++f) values(c, f, vw[f], p);
        }
      } else {
        v4f_a s[CT][4];
        v8bf_a p[CT][NP][2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          v8bf_a kw[KK][2];
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) widen(kf[t][kk], kw[kk]);
#pragma unroll
          for (int c = 0; c < CT; ++c) s[c][t] = product(c, kw);
        }
        load_k(j + NW);
#pragma unroll
        for (int c = 0; c < CT; ++c) weigh(c, s[c], p[c]);
#pragma unroll
        for (int f = 0; f < FT; ++f) {
          v8bf_a v[2];
          widen(vf[f], v);
#pragma unroll
          for (int c = 0; c < CT; ++c) values(c, f, v, p[c]);
        }
        load_v(j + NW);
      }
    }
  }

  // the wavefronts: 2 and 3 into 0 and 1, then 1 into 0
  float l[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) l[c] = sums[c][0];
  const auto merge = [&](int half) {
    if (wave >= half && wave < 2 * half) {
      float(*const to)[64] = box[wave - half];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        to[c * (4 * FT + 2)][lane] = m[c];
        to[c * (4 * FT + 2) + 1][lane] = l[c];
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
          for (int e = 0; e < 4; ++e) to[c * (4 * FT + 2) + 2 + 4 * f + e][lane] = o[c][f][e];
      }
    }
    __syncthreads();
    if (wave < half) {
      const float(*const from)[64] = box[wave];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const float m1 = from[c * (4 * FT + 2)][lane], l1 = from[c * (4 * FT + 2) + 1][lane];
        const float mn = fmaxf(m[c], m1);
        const float c0 = m[c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[c] - mn);
        const float c1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - mn);
        // a NaN sum with no maximum still has to be seen
        l[c] = (l[c] == l[c] ? l[c] * c0 : l[c]) + (l1 == l1 ? l1 * c1 : l1);
        m[c] = mn;
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[c][f][e] = __builtin_fmaf(from[c * (4 * FT + 2) + 2 + 4 * f + e][lane], c1,
                                        o[c][f][e] * c0);
      }
    }
  };
  merge(2);
  __syncthreads();
  merge(1);
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int64_t ct = (tile * CT + c) * 16 + col;
    if (ct >= cols) continue;
    float* const w = a.work + ((bh * cols + ct) * a.nsplit + split) * (D + 4);
    if (g == 0) {
      w[0] = m[c];
      w[1] = l[c];
    }
#pragma unroll
    for (int f = 0; f < FT; ++f)
      *reinterpret_cast<float4*>(w + 4 + 16 * f + 4 * g) =
          make_float4(o[c][f][0], o[c][f][1], o[c][f][2], o[c][f][3]);
  }
}

// A column's running softmax over parts: each has a maximum, a sum and D / 16 features a lane.
template <int F>
struct TreeState {
  float m = -INFINITY, l = 0.0f, o[F];
  __device__ __forceinline__ TreeState() {
#pragma unroll
    for (int e = 0; e < F; ++e) o[e] = 0.0f;
  }
  // a part whose maximum is -inf holds nothing, unless its sum is NaN
  __device__ __forceinline__ void add(float m1, float l1, const float (&o1)[F]) {
    const float mn = fmaxf(m, m1);
    const float c0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float c1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - mn);
    l = (l == l ? l * c0 : l) + (l1 == l1 ? l1 * c1 : l1);
    m = mn;
#pragma unroll
    for (int e = 0; e < F; ++e)
      o[e] = m1 == -INFINITY ? o[e] : __builtin_fmaf(o1[e], c1, o[e] * c0);
  }
};

// grid (columns / 4, B * H), a wavefront a column: its splits and the nodes it sees, in float32. Four
// groups of 16 lanes, D / 16 features a lane, take every fourth of both.
template <int D, int QDT, int ODT>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeAttn a) {
  constexpr int F = D / 16;
  const uint32_t uh = static_cast<uint32_t>(a.c.H), ub = blockIdx.y / uh;
  const int64_t ct = 4 * static_cast<int64_t>(blockIdx.x) +
                     __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (ct >= a.N * a.G) return;
  const int64_t bh = blockIdx.y, b = ub, kvh = blockIdx.y - ub * uh;
  const int64_t i = static_cast<uint32_t>(ct) / static_cast<uint32_t>(a.G);
  const int64_t hd = kvh * a.G + (ct - i * a.G);
  const int lane = threadIdx.x & 63, grp = lane >> 4, f0 = (lane & 15) * F;
  const int64_t start = a.start[b * a.start_step];
  const int64_t tree = b * a.tree_step;
  const uint64_t* const seen = a.seen + (tree * a.N + i) * a.W;
  // bits past the last node are not looked at
  const uint64_t tail = a.N % 64 ? (1ull << (a.N % 64)) - 1 : ~0ull;
  uint64_t any = 0;
  for (int64_t w = 0; w < a.W; ++w) any |= seen[w] & (w + 1 < a.W ? ~0ull : tail);
  const bool on = start >= 0 && any != 0 && !(a.lengths && i >= a.lengths[b]);
  const bool past = start > a.c.NB * kTok;
  TreeState<F> st;
  if (on && !past) {
    const float* const work =
        a.work + (bh * a.N * a.G + ct) * a.nsplit * (D + 4);
    for (int64_t s = grp; s < a.nsplit; s += 4) {
      const float* const at = work + s * (D + 4);
      float o1[F];
#pragma unroll
      for (int e = 0; e < F; e += 4) load_vec16<RK_F32>(at, 4 + f0 + e, o1 + e);
      st.add(at[0], at[1], o1);
    }
    constexpr int PER = F < Vec<QDT>::N ? F : Vec<QDT>::N;
    const auto load = [&](const void* src, int64_t idx, float (&x)[F]) {
      if constexpr (PER == Vec<QDT>::N) {
#pragma unroll
        for (int e = 0; e < F; e += PER) load_vec16<QDT>(src, idx + e, x + e);
      } else {  // four bf16 features
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(src) + idx);
        x[0] = __uint_as_float(w.x << 16);
        x[1] = __uint_as_float(w.x & 0xffff0000u);
        x[2] = __uint_as_float(w.y << 16);
        x[3] = __uint_as_float(w.y & 0xffff0000u);
      }
    };
    float q[F];
    load(a.q, b * a.sqb + hd * a.sqh + i * a.sqs + f0, q);
    const float slope2 = a.slopes ? a.slopes[hd] * kLog2e8 : 0.0f;
    const int32_t* const depths = a.depths + tree * a.N;
    const int depth = depths[i];
    for (int64_t w = 0; w < a.W; ++w) {
      uint64_t left = seen[w] & (w + 1 < a.W ? ~0ull : tail);
      while (left) {  // the next eight nodes, two for each group, loaded together
        int node[2] = {-1, -1};
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int at = left ? static_cast<int>(__builtin_ctzll(left)) : -1;
          if (grp == n % 4) node[n / 4] = at;
          left &= left - 1;
        }
        float k[2][F], v[2][F], s[2];
        int depth_at[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int64_t at = 64 * w + (node[n] < 0 ? 0 : node[n]);
          load(a.k, b * a.skb + kvh * a.skh + at * a.sks + f0, k[n]);
          load(a.v, b * a.svb + kvh * a.svh + at * a.svs + f0, v[n]);
          depth_at[n] = depths[at];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          s[n] = 0.0f;
#pragma unroll
          for (int e = 0; e < F; ++e) s[n] = __builtin_fmaf(q[e], k[n][e], s[n]);
          const auto bits = [&] { return __float_as_uint(s[n]); };
          s[n] = s[n] + __uint_as_float(dpp_u32<0x128>(bits()));  // over the group's lanes
          s[n] = s[n] + __uint_as_float(dpp_u32<0x141>(dpp_u32<0x1b>(bits())));
          s[n] = s[n] + __uint_as_float(dpp_u32<0x4e>(bits()));
          s[n] = s[n] + __uint_as_float(dpp_u32<0xb1>(bits()));
          s[n] = s[n] * a.dot_scale;
          if (a.cap2 != 0.0f) s[n] = tree_capped<ODT == RK_F32>(s[n], a.cap2, a.inv_cap2);
          if (a.slopes)
            s[n] = __builtin_fmaf(-slope2, static_cast<float>(depth - depth_at[n]), s[n]);
          if (node[n] >= 0) st.add(s[n], 1.0f, v[n]);
        }
      }
    }
  }
  // the groups
  float r[F];
#pragma unroll
  for (int off = 16; off <= 32; off *= 2) {
    float o1[F];
    const float m1 = __shfl_xor(st.m, off), l1 = __shfl_xor(st.l, off);
#pragma unroll
    for (int e = 0; e < F; ++e) o1[e] = __shfl_xor(st.o[e], off);
    st.add(m1, l1, o1);
  }
#pragma unroll
  for (int e = 0; e < F; ++e)
    r[e] = !on ? 0.0f : past ? __uint_as_float(0x7fc00000u) : st.o[e] / st.l;
  if (grp == 0) {
#pragma unroll
    for (int e = 0; e < F; e += 4) {
      const float x[4] = {r[e], r[e + 1], r[e + 2], r[e + 3]};
      store4<ODT>(a.out, ((b * a.N + i) * a.Hq + hd) * D + f0 + e, x);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct TreeLaunch {
  int ct;  // tiles of 16 columns a wavefront holds
  int64_t tiles, splits;
};

static TreeLaunch tree_launch(const rk_tree_attention_args& p) {
  const rk_int8_kv& c = p.cache;
  const int64_t cols = p.N * (p.Hq / c.H);
  TreeLaunch t{};
  const bool many = cols > 32 && p.dtype == RK_BF16 && p.out_dtype == RK_BF16;
  t.ct = c.D > 128 || cols <= 16 || (c.D == 128 && p.dtype == RK_F32) ? 1 : 2;
  t.tiles = (cols + 16 * t.ct - 1) / (16 * t.ct);
  const int64_t have = t.tiles * c.B * c.H;
  const auto splits = [&](int64_t wgs, int64_t least) {
    const int64_t n = wgs / (have > 0 ? have : 1), most = (c.blocks + least - 1) / least;
    return n < 1 || most < 1 ? 1 : n < most ? n : most;
  };
  // Up to 512 workgroups of a block for each wavefront at least; of 16 blocks and more, up to 1024
  // (2048 with many columns, which are slower): sequences of several lengths are not even. 16
  // sequences of 2.7 to 8 thousand tokens, 16 heads of 128, 32 nodes: 512 85 us, 1024 82, 2048 88; 8 of
  // 6 to 15 thousand, 32 heads of 64 on 4, 64 nodes: 1024 155, 2048 137, 4096 146. (4 of 1 to 3
  // thousand, float32: 512 17 us, 1024 of fewer than 16 blocks 19.)
  const int64_t few = splits(512, 4), more = splits(many ? 2048 : 1024, 16);
  t.splits = few > more ? few : more;
  return t;
}

template <int D, int CT, int MODE>
static void launch_tree_cache(const TreeAttn& a, int qdt, int odt, hipStream_t st) {
  constexpr int F32 = RK_F32, BF16 = RK_BF16;
  const dim3 grid(static_cast<unsigned>(a.nsplit), static_cast<unsigned>(a.tiles),
                  static_cast<unsigned>(a.c.B * a.c.H));
  if (qdt == RK_F32) {
    if constexpr (D != 128 || CT == 1) {
      if (odt == RK_F32) tree_cache_kernel<D, CT, F32, F32, MODE><<<grid, 256, 0, st>>>(a);
      else tree_cache_kernel<D, CT, F32, BF16, MODE><<<grid, 256, 0, st>>>(a);
    }
  } else if (odt == RK_F32) {
    tree_cache_kernel<D, CT, BF16, F32, MODE><<<grid, 256, 0, st>>>(a);
  } else {
    tree_cache_kernel<D, CT, BF16, BF16, MODE><<<grid, 256, 0, st>>>(a);
  }
}

template <int D>
static void launch_tree(const TreeAttn& a, const TreeLaunch& t, int qdt, int odt, hipStream_t st) {
  const auto run = [&](auto mode) {
    constexpr int M = decltype(mode)::value;
    if constexpr (D <= 128) {
      if (t.ct == 2) return launch_tree_cache<D, 2, M>(a, qdt, odt, st);
    }
    launch_tree_cache<D, 1, M>(a, qdt, odt, st);
  };
  if (a.slopes || a.cap2 > kBound) run(std::integral_constant<int, kModified>{});
  else if (a.cap2 != 0.0f) run(std::integral_constant<int, kBounded>{});
  else run(std::integral_constant<int, kPlain>{});
  const dim3 grid(static_cast<unsigned>((a.N * a.G + 3) / 4),
                  static_cast<unsigned>(a.c.B * a.c.H));
  if (qdt == RK_F32 && odt == RK_F32) tree_join_kernel<D, RK_F32, RK_F32><<<grid, 256, 0, st>>>(a);
  else if (qdt == RK_F32) tree_join_kernel<D, RK_F32, RK_BF16><<<grid, 256, 0, st>>>(a);
  else if (odt == RK_F32) tree_join_kernel<D, RK_BF16, RK_F32><<<grid, 256, 0, st>>>(a);
  else tree_join_kernel<D, RK_BF16, RK_BF16><<<grid, 256, 0, st>>>(a);
}

// tree_near's coefficients: the quadratic through g(z) = (tanh(u) / u - 1) / z, z = u^2, at three
// Chebyshev nodes of 0 .. kNear^2, in units of C^2.
static void near_coefficients(double cap2, float (&c)[3]) {
  double z[3], g[3];
  for (int i = 0; i < 3; ++i) {
    z[i] = 0.5 * kNear * kNear * (1.0 + cos((2 * i + 1) * M_PI / 6.0));
    const double u = sqrt(z[i]);
    g[i] = (tanh(u) / u - 1.0) / z[i];
  }
  const double d01 = (g[1] - g[0]) / (z[1] - z[0]), d12 = (g[2] - g[1]) / (z[2] - z[1]);
  const double d = (d12 - d01) / (z[2] - z[0]);
  const double k[3] = {g[0] - d01 * z[0] + d * z[0] * z[1], d01 - d * (z[0] + z[1]), d};
  double unit = 1.0;
  for (int i = 0; i < 3; ++i) {
    unit /= cap2 * cap2;
    c[i] = static_cast<float>(k[i] * unit);
  }
}

static int check_tree(const rk_tree_attention_args& p) {
  const rk_int8_kv& c = p.cache;
  if (int e = check_cache(c)) return e;
  if (p.N < 0 || p.Hq < 0 || p.trees < 0) return fail(RK_ERR_ARG, "negative size");
  if (p.N > kTreeNodes) return fail(RK_ERR_UNSUPPORTED, "a tree has at most %d nodes", kTreeNodes);
  if (c.H == 0 ? p.Hq != 0 : p.Hq % c.H != 0)
    return fail(RK_ERR_ARG, "query heads must be a multiple of the key heads");
  if ((p.dtype != RK_F32 && p.dtype != RK_BF16) || (p.out_dtype != RK_F32 && p.out_dtype != RK_BF16))
    return fail(RK_ERR_ARG, "queries, keys, values and outputs are float32 or bfloat16");
  if (p.start_count != 1 && p.start_count != c.B)
    return fail(RK_ERR_ARG, "one start, or one per sequence");
  if (p.trees != 1 && p.trees != c.B) return fail(RK_ERR_ARG, "one tree, or one per sequence");
  if (!(p.scale > 0.0f) || !(p.scale < INFINITY))
    return fail(RK_ERR_ARG, "scale must be positive and finite");
  if (!(p.softcap >= 0.0f) || !(p.softcap < INFINITY))
    return fail(RK_ERR_ARG, "softcap must be finite and not negative (0: none)");
  if (p.softcap != 0.0f && !(p.softcap >= 1e-3f && p.softcap <= 1e3f))
    return fail(RK_ERR_UNSUPPORTED, "softcap outside 1e-3 .. 1e3");
  if (c.blocks == 0 && c.B > 0 && p.Hq > 0 && p.N > 0) return fail(RK_ERR_ARG, "an empty cache");
  return RK_OK;
}

}  // namespace rk

using namespace rk;

extern "C" int rk_draft_tree(const void* parents, int wide, int64_t ldp, int64_t R, int64_t N,
                             int32_t* kept, int32_t* depths, uint64_t* seen, void* stream) {
  clear_error();
  if (R < 0 || N < 0 || ldp < 0) return fail(RK_ERR_ARG, "negative size");
  if (N > kTreeNodes) return fail(RK_ERR_UNSUPPORTED, "a tree has at most %d nodes", kTreeNodes);
  if (R == 0 || N == 0) return RK_OK;
  if (!parents || !kept || !depths || !seen) return fail(RK_ERR_ARG, "null pointer");
  // a launch holds fewer than 2^24 blocks of 256 threads
  if (R >= (int64_t{1} << 24)) return fail(RK_ERR_UNSUPPORTED, "too many trees");
  const TreePlan a{parents, wide, ldp, N, (N + 63) / 64, kept, depths, seen};
  draft_tree_kernel<<<static_cast<unsigned>(R), kTreeNodes, 0, as_stream(stream)>>>(a);
  return launch_status("draft_tree");
}

extern "C" int64_t rk_tree_attention_work(const rk_tree_attention_args* args) {
  if (!args || args->cache.B <= 0 || args->cache.H <= 0 || args->Hq <= 0 || args->N <= 0 ||
      args->Hq % args->cache.H)
    return 0;
  return args->cache.B * args->Hq * args->N * tree_launch(*args).splits * (args->cache.D + 4);
}

extern "C" int rk_tree_attention(const rk_tree_attention_args* args, float* work,
                                 int64_t work_floats, void* stream) {
  clear_error();
  if (!args) return fail(RK_ERR_ARG, "null arguments");
  const rk_tree_attention_args& p = *args;
  if (int e = check_tree(p)) return e;
  const rk_int8_kv& c = p.cache;
  if (c.B == 0 || p.Hq == 0 || p.N == 0) return RK_OK;
  if (!p.q || !p.k || !p.v || !p.start || !p.seen || !p.depths || !p.out)
    return fail(RK_ERR_ARG, "null pointer");
  const int64_t per = p.dtype == RK_F32 ? 4 : 8;
  const int64_t strides[] = {p.sqb, p.sqh, p.sqs, p.skb, p.skh, p.sks, p.svb, p.svh, p.svs};
  for (int64_t st : strides)
    if (st < 0 || st % per != 0)
      return fail(RK_ERR_UNSUPPORTED, "rows and strides must be whole 16-byte vectors");
  if (!aligned16(p.q) || !aligned16(p.k) || !aligned16(p.v) || !aligned16(p.out))
    return fail(RK_ERR_UNSUPPORTED, "queries, keys, values and outputs need 16-byte alignment");
  const int64_t G = p.Hq / c.H;
  const TreeLaunch t = tree_launch(p);
  // a launch holds fewer than 2^24 blocks of 256 threads
  if (p.N * G >= (int64_t{1} << 24) || t.tiles > 65535 ||
      t.tiles * c.B * c.H * t.splits >= (int64_t{1} << 24) ||
      p.N * p.Hq * c.B >= (int64_t{1} << 26))
    return fail(RK_ERR_UNSUPPORTED, "too many queries for one launch");
  if (!work || !aligned16(work) || work_floats < rk_tree_attention_work(args))
    return fail(RK_ERR_ARG, "attention workspace too small");
  const float cap2 = p.softcap * kLog2e8;
  TreeAttn a{cache_args(c), p.q, p.k, p.v, p.sqb, p.sqh, p.sqs, p.skb, p.skh, p.sks, p.svb,
             p.svh, p.svs, p.start, p.lengths, p.seen, p.depths, p.slopes,
             p.start_count > 1 ? 1 : 0, p.trees > 1 ? 1 : 0, p.N, (p.N + 63) / 64, p.Hq, G,
             t.splits, t.tiles, p.scale * kLog2e8, cap2, cap2 > 0.0f ? 1.0f / cap2 : 0.0f, {},
             work, p.out};
  if (cap2 > 0.0f) near_coefficients(cap2, a.near);
  hipStream_t st = as_stream(stream);
  if (c.D == 64) launch_tree<64>(a, t, p.dtype, p.out_dtype, st);
  else if (c.D == 128) launch_tree<128>(a, t, p.dtype, p.out_dtype, st);
  else launch_tree<256>(a, t, p.dtype, p.out_dtype, st);
  return launch_status("tree_attention");
}

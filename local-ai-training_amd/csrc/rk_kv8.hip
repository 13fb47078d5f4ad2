// A key/value cache in 8 bits (gfx950): appended keys and values quantized per block of 64 tokens
// and key head, attention of new tokens over it, and the values read back. It stands beside the
// bf16 / float32 cache (rk_kv_append, rk_decode_attention) at half or a quarter of its bytes; the
// reference keeps no cache (generate.py:183-201 recomputes the window).
//
// Layout: keys int8 [B, Hkv, NB, 64, D], values int8 [B, Hkv, NB, D, 64] (by feature), one
// float32 scale per block and head for each. Both products of the attention then read their
// operand 16 bytes per lane straight from memory, in the order in which the MFMA takes it.
//
// Quantization: s = absmax / 127 over the block's tokens, code = rint(x / s) (IEEE float32
// quotients, the rule of rk_quantize_rows). Tokens appended to a block that holds some can only
// raise its scale; the codes there are then rounded again, rint(c (s_old / s)). A block's first
// token starts it anew, whatever it held.
#include "rk_attention.h"
#include "rk_rowquant.h"

#include <math.h>

namespace rk {

constexpr int kTok = 64;  // tokens of a block
constexpr int64_t kChunkTokens = 32;  // a wavefront's queries: from here on kv8_chunk_kernel
constexpr float kLog2e8 = 1.4426950408889634f;

typedef int v4i8 __attribute__((ext_vector_type(4)));
typedef float v4f_a __attribute__((ext_vector_type(4)));

struct Kv8 {
  int8_t* keys;
  int8_t* values;
  float* ks;
  float* vs;
  int64_t B, H, NB;  // H: key heads
};

struct Kv8Append {
  Kv8 c;
  const void* k;
  const void* v;
  int64_t skb, skh, sks, svb, svh, svs;
  const int64_t* start;    // [1] or [B] (start_step 0 or 1)
  const int64_t* lengths;  // [B] or null
  int64_t start_step, S;
};

// The new tokens first .. last - 1 of block `blk` of sequence b, first past what it keeps.
__device__ __forceinline__ bool append_range(const Kv8Append& a, int64_t b, int64_t touched,
                                             int64_t& blk, int64_t& start, int& first, int& last) {
  start = a.start[b * a.start_step];
  if (start < 0) return false;
  int64_t n = a.lengths ? a.lengths[b] : a.S;
  n = n < a.S ? n : a.S;
  blk = (start >> 6) + touched;
  if (n <= 0 || blk >= a.c.NB) return false;
  const int64_t base = blk * kTok, f = start - base, l = start + n - base;
  first = static_cast<int>(f > 0 ? f : 0);
  last = static_cast<int>(l < kTok ? l : kTok);
  return first < last;
}

__device__ __forceinline__ float fmed3(float x) {
  return __builtin_amdgcn_fmed3f(x, -127.0f, 127.0f);
}

// code of x under scale s; only denormal scales reach the clamp, only NaN and infinite scales
// the zero of a NaN quotient
__device__ __forceinline__ int code_of(float x, float s) {
  const float y = __builtin_rintf(x / s);
  const int c = static_cast<int>(fminf(fmaxf(y, -127.0f), 127.0f));
  return s > 0.0f && y == y ? c : 0;
}
// The same for 8 values, by the reciprocal r of s where that decides (rk_rowquant.h: the rounded
// product, redone by the quotient when one of the 8 lies near a rounding boundary). With the IEEE
// quotient for every value the divisions were most of its instructions.
__device__ __forceinline__ void codes_of(const float (&x)[8], float s, float r, int (&c)[8]) {
  bool exact = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = static_cast<int>(fmed3(round_fast(x[e], r, exact)));
  if (exact) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = code_of(x[e], s);
  }
}
__device__ __forceinline__ int code_again(int c, float ratio) {
  return static_cast<int>(
      fminf(fmaxf(__builtin_rintf(static_cast<float>(c) * ratio), -127.0f), 127.0f));
}

// grid (touched blocks, B * H, 2: keys, values), 256 threads; a thread takes D / 32 pieces of 8
// features. The block's absmax by the bits of |x| (a NaN is the largest), so a block that takes
// in a NaN or an infinity has such a scale and reads back as NaN. 4 x 777 tokens, 16 heads of 128:
// 14.8 us for 39 MB (a load, a reduction and a store in workgroups that are all resident at once;
// 262 MB of float32 80 us, 4.1 TB/s); a token for 16 sequences 5.4 us.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8Append a) {
  constexpr int PER = D / 8, EACH = kTok * PER / 256, PITCH = kTok + 4;
  __shared__ uint32_t red[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[D * PITCH];
  const uint32_t uh = static_cast<uint32_t>(a.c.H), ub = blockIdx.y / uh;
  const int64_t bh = blockIdx.y, b = ub, h = blockIdx.y - ub * uh;
  const int tid = threadIdx.x;
  int64_t blk, start;
  int first, last;
  if (!append_range(a, b, blockIdx.x, blk, start, first, last)) return;
  const bool val = blockIdx.z != 0;
  const int64_t at = (bh * a.c.NB + blk);
  float* const scale = (val ? a.c.vs : a.c.ks) + at;
  int8_t* const codes = (val ? a.c.values : a.c.keys) + at * kTok * D;
  const void* src = val ? a.v : a.k;
  const int64_t ss = val ? a.svs : a.sks;
  // element offset of the token at the block's first position (never read before `first`)
  const int64_t off = b * (val ? a.svb : a.skb) + h * (val ? a.svh : a.skh) +
                      (blk * kTok - start) * ss;
  const float old = first > 0 ? *scale : 0.0f;

  // every thread loads, tokens outside first .. last - 1 the nearest one inside: a condition
  // around the loads let only one be in flight (16 -> 14.5 us at 4 x 777 tokens, 16 heads of 128)
  float x[EACH][8];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int unit = tid + 256 * i, t = unit / PER, f = unit % PER * 8;
    const int tc = t < first ? first : t < last ? t : last - 1;
    load_vec16<DT>(src, off + tc * ss + f, x[i]);
    if constexpr (DT == RK_F32) load_vec16<DT>(src, off + tc * ss + f + 4, x[i] + 4);
  }
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = __float_as_uint(x[i][e]) & 0x7fffffffu;
      most = bits > most ? bits : most;
    }
  most = wave_butterfly(most, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
  if ((tid & 63) == 0) red[tid >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) most = red[w] > most ? red[w] : most;
  float s = __uint_as_float(most) / 127.0f;
  if (first > 0 && __float_as_uint(old) > __float_as_uint(s)) s = old;
  const bool grown = first > 0 && __float_as_uint(old) != __float_as_uint(s);
  const float ratio = old / (s > 0.0f ? s : 1.0f), recip = 1.0f / s;
  if (tid == 0) *scale = s;

  if (!val) {
    if (grown) {
      for (int i = tid; i < first * (D / 4); i += 256) {
        uint32_t* const w = reinterpret_cast<uint32_t*>(codes) + i;
        const uint32_t c = *w;
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          r |= static_cast<uint32_t>(code_again(static_cast<int8_t>(c >> (8 * e)), ratio) & 255)
               << (8 * e);
        *w = r;
      }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int unit = tid + 256 * i, t = unit / PER, f = unit % PER * 8;
      if (t >= first && t < last) {
        int c[8];
        codes_of(x[i], s, recip, c);
        *reinterpret_cast<uint2*>(codes + t * D + f) =
            make_uint2(pack_bytes4(c[0], c[1], c[2], c[3]), pack_bytes4(c[4], c[5], c[6], c[7]));
      }
    }
    return;
  }
  // values: the block by features in LDS, what it keeps first, then written whole
  for (int i = tid; i < D * (kTok / 4); i += 256) {
    const int f = i / (kTok / 4), w = i % (kTok / 4);
    uint32_t r = 0;
    if (4 * w < first) {
      const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[i];
      r = c;
      if (grown) {
        r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          r |= static_cast<uint32_t>(code_again(static_cast<int8_t>(c >> (8 * e)), ratio) & 255)
               << (8 * e);
      }
    }
    *reinterpret_cast<uint32_t*>(tile + f * PITCH + 4 * w) = r;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int unit = tid + 256 * i, t = unit / PER, f = unit % PER * 8;
    if (t >= first && t < last) {
      int c[8];
      codes_of(x[i], s, recip, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[(f + e) * PITCH + t] = static_cast<uint8_t>(c[e]);
    }
  }
  __syncthreads();
  for (int i = tid; i < D * (kTok / 4); i += 256)
    reinterpret_cast<uint32_t*>(codes)[i] =
        *reinterpret_cast<const uint32_t*>(tile + i / (kTok / 4) * PITCH + 4 * (i % (kTok / 4)));
}

struct Kv8Read {
  Kv8 c;
  int64_t begin, n;
  void* keys;  // [B, H, n, D] contiguous, float32 or bf16
  void* values;
};

// grid (blocks, B * H, 2), 256 threads: the values codes stand for, code x scale in float32. Bound
// by its bytes: 64 MB, mostly written, in 12.5 us.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8Read a) {
  constexpr int PER = D / 8, PITCH = kTok + 4;
  __shared__ __attribute__((aligned(16))) uint8_t tile[D * PITCH];
  const int64_t bh = blockIdx.y, blk = a.begin / kTok + blockIdx.x;
  const int tid = threadIdx.x;
  const bool val = blockIdx.z != 0;
  const int64_t at = bh * a.c.NB + blk;
  const float s = (val ? a.c.vs : a.c.ks)[at];
  const int8_t* const codes = (val ? a.c.values : a.c.keys) + at * kTok * D;
  if (val) {
    for (int i = tid; i < D * (kTok / 4); i += 256)
      *reinterpret_cast<uint32_t*>(tile + i / (kTok / 4) * PITCH + 4 * (i % (kTok / 4))) =
          reinterpret_cast<const uint32_t*>(codes)[i];
    __syncthreads();
  }
  char* const out = static_cast<char*>(val ? a.values : a.keys);
  for (int unit = tid; unit < kTok * PER; unit += 256) {
    const int t = unit / PER, f = unit % PER * 8;
    const int64_t tok = blk * kTok + t - a.begin;
    if (tok < 0 || tok >= a.n) continue;
    float x[8];
    if (val) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = static_cast<int8_t>(tile[(f + e) * PITCH + t]) * s;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + t * D + f);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = static_cast<int8_t>((e < 4 ? w.x : w.y) >> (8 * (e % 4))) * s;
    }
    const int64_t idx = (bh * a.n + tok) * D + f;
    if constexpr (DT == RK_F32) {
      float4* const o = reinterpret_cast<float4*>(out + idx * 4);
      o[0] = make_float4(x[0], x[1], x[2], x[3]);
      o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = f32_to_bf16(x[2 * e]) | (static_cast<uint32_t>(f32_to_bf16(x[2 * e + 1])) << 16);
      *reinterpret_cast<uint4*>(out + idx * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention of S new tokens per sequence (positions start .. start + S - 1, their keys and values
// appended before) over the cache: query i sees positions 0 .. start + i.
//   s_j = scale q . k_j;  capped and biased as in rk_scored.h;  o = sum_j softmax(s_j) v_j
// with k_j, v_j what the codes stand for. Columns of a product are the S * G queries that share a
// key head (G = query heads per key head), 16 at a time; rows are keys, then features.
//
// The first product runs on the codes as they are, in exact integers: the query is written as a
// fixed-point number of three signed base-256 digits (23 bits) relative to its largest feature,
// which may be thousands of times the others (in two, one of 500 times took bf16 results from 1.7e-3
// to 4e-3), and each digit's product is its own MFMA.
// The second takes codes widened to bf16, which holds them exactly, and probabilities as sums of bf16
// numbers: three for float32 results (24 bits of each probability), two for bf16 (16 bits). A
// probability needs its own exponent: as fixed-point numbers relative to their block's largest, those
// beside a token that takes nearly all of the attention lost their bits, and where that token's
// value is small they are the result (with 1e-3 left to the others, bf16 results off by a tenth;
// widening and splitting cost 137 -> 142 us at 16 sequences of 5 to 16 thousand tokens, 30 -> 33 at
// 48 of 2.7 to 8.1 thousand with shared heads). For one query per head, 56 MFMAs (72 with three
// parts) and about 500 vector instructions per 16 KB of codes at D = 128.
//
// A wavefront walks blocks of 64 tokens with its own running max, sum and output. Lane l holds the
// scores of column l % 16 against keys 16 (l / 16) .. + 15: key 16 g + 4 t + e is row 4 g + e of
// product t, and the same 16 keys are the lane's k slots of the second product (8 for each half),
// whose other operand, 16 tokens of one feature, lies side by side in the cache. The wavefronts of a
// workgroup are joined in LDS, splits of a long cache by a second launch.
//
// 16 sequences of 5 to 16 thousand tokens, 16 heads of 128: 143-147 us, 820 MB of codes at 5.6 TB/s
// (the device's own copy reaches 5.3); 48 sequences of 2.7 to 8.1 thousand, 32 heads of 64 on 4,
// capped: 31 + 4 us for 125 MB; one of 1000, 16 heads of 128: 11.4 us, a chain of load latencies.
// ---------------------------------------------------------------------------
struct Kv8Attn {
  Kv8 c;
  const void* q;
  int64_t sqb, sqh, sqs;
  const int64_t* start;
  const int64_t* lengths;
  const float* slopes;
  int64_t start_step, S, Hq, G, nsplit, tiles;
  int64_t nfull;  // chunks: splits of whole tiles (1 or nsplit; the last, partial one has nsplit)
  int64_t col0;   // the first column that is joined
  float dot_scale, cap2;
  float* work;  // [B * H][S * G - col0][nsplit][D + 4]: max, sum, 2 pad, unnormalized output
  void* out;    // [B, S, Hq, D], of type ODT
};

__device__ __forceinline__ float col_max(float v) {  // over the four lanes of a column
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float col_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ uint32_t col_umax(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = r[0] > r[1] ? r[0] : r[1];
  const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return s[0] > s[1] ? s[0] : s[1];
}

constexpr int kDigits = 3;  // of a query's number, signed, base 256: the largest is kFixed
constexpr float kFixed = 127.0f * 65536.0f;

// Digits of 4 numbers, each given as the word whose low bytes are the number plus 128 in every
// digit but the first (which makes them unsigned, without a carry to take back), as one word a
// digit, the first digit first.
__device__ __forceinline__ void digits4(const uint32_t (&w)[4], int (&d)[kDigits]) {
  const uint32_t p01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // low bytes, second bytes
  const uint32_t p23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t low = __builtin_amdgcn_perm(p23, p01, 0x05040100u);
  const uint32_t mid = __builtin_amdgcn_perm(p23, p01, 0x07060302u);
  const uint32_t h01 = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0602u);
  const uint32_t h23 = __builtin_amdgcn_perm(w[3], w[2], 0x0c0c0602u);
  d[0] = static_cast<int>(__builtin_amdgcn_perm(h23, h01, 0x05040100u));
  d[1] = static_cast<int>(mid ^ 0x80808080u);
  d[2] = static_cast<int>(low ^ 0x80808080u);
}

// The sum that the digits' sums make (each below 2^22, so two of them fit an integer).
__device__ __forceinline__ float from_digits(const v4i8 (&d)[kDigits], int e) {
  return __builtin_fmaf(static_cast<float>(d[0][e]), 65536.0f,
                        static_cast<float>(d[1][e] * 256 + d[2][e]));
}

template <bool SCALED = false>
__device__ __forceinline__ void widen_codes(uint32_t w, uint32_t& lo, uint32_t& hi,
                                            float power = 1.0f) {
  uint32_t f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
    f[e] = __float_as_uint(SCALED ? x * power : x);
  }
  lo = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);  // small integers: the low halves are zero
  hi = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
}

// 16 probabilities as sums of N bf16 numbers each, the largest parts first: off by 2^-8N of
// themselves.
template <int N>
__device__ __forceinline__ void split_bf16(float (&p)[16], v8bf_a (&part)[N][2]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = bf16_pair(p[2 * i], p[2 * i + 1]);
      if (n + 1 < N) {  // what is left, exactly
        p[2 * i] = p[2 * i] - __uint_as_float(w[i] << 16);
        p[2 * i + 1] = p[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    part[n][0] = frag_of(make_uint4(w[0], w[1], w[2], w[3]));
    part[n][1] = frag_of(make_uint4(w[4], w[5], w[6], w[7]));
  }
}

template <int QDT>
__device__ __forceinline__ void store4(void* out, int64_t idx, const float (&x)[4]) {
  if constexpr (QDT == RK_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + idx) =
        make_float4(x[0], x[1], x[2], x[3]);
  } else {
    const uint32_t lo = f32_to_bf16(x[0]) | (static_cast<uint32_t>(f32_to_bf16(x[1])) << 16);
    const uint32_t hi = f32_to_bf16(x[2]) | (static_cast<uint32_t>(f32_to_bf16(x[3])) << 16);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + idx) = make_uint2(lo, hi);
  }
}

// What a row of the output holds where it is not a plain quotient: zeros for a sequence or token
// that is switched off, NaN for a position past the cache.
__device__ __forceinline__ float row_factor(const Kv8Attn& a, int64_t b, int64_t i, float l) {
  const int64_t start = a.start[b * a.start_step];
  if (start < 0 || (a.lengths && i >= a.lengths[b])) return 0.0f;
  if (start + i >= a.c.NB * kTok) return __uint_as_float(0x7fc00000u);
  return 1.0f / l;
}

template <int D, int QDT, int ODT, int NW, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * NW) void kv8_attn_kernel(Kv8Attn a) {
  constexpr int KK = D / 64, FT = D / 16, NT = 64 * NW;
  constexpr int NP = ODT == RK_F32 ? 3 : 2;  // parts of a probability
  __shared__ __attribute__((aligned(16))) float so[NW][16][D + 4];
  __shared__ float sm[NW][16], sl[NW][16];
  const int split = blockIdx.x;
  const int64_t tile = blockIdx.y, bh = blockIdx.z;
  const uint32_t uh = static_cast<uint32_t>(a.c.H), ub = blockIdx.z / uh;  // 32-bit divisions
  const int64_t b = ub, kvh = blockIdx.z - ub * uh;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t start = a.start[b * a.start_step];
  const int64_t cols = a.S * a.G;
  // this lane's column: query i of head kvh * G + hg; lanes past the last take the last's
  const int64_t cc = tile * 16 + col < cols ? tile * 16 + col : cols - 1;
  const uint32_t ug = static_cast<uint32_t>(a.G);  // (the host bounds the columns)
  const int64_t i = static_cast<uint32_t>(cc) / ug, hd = kvh * a.G + (cc - i * a.G);
  int64_t n = a.lengths ? a.lengths[b] : a.S;
  n = n < a.S ? n : a.S;
  // the blocks that the tile's last active query sees
  const int64_t c_last = tile * 16 + 15 < cols ? tile * 16 + 15 : cols - 1;
  int64_t i_last = static_cast<uint32_t>(c_last) / ug;
  i_last = i_last < n ? i_last : n - 1;
  const bool on = start >= 0 && n > 0 && static_cast<uint32_t>(tile * 16) / ug < n;
  int64_t nb = on ? ((start + i_last) >> 6) + 1 : 0;
  nb = nb < a.c.NB ? nb : a.c.NB;
  const int64_t per = (static_cast<uint32_t>(nb) + static_cast<uint32_t>(a.nsplit) - 1) /
                      static_cast<uint32_t>(a.nsplit);
  const int64_t j0 = split * per, j1 = j0 + per < nb ? j0 + per : nb;

  float m = -INFINITY, l = 0.0f, o[FT][4];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[f][e] = 0.0f;

  if (j0 + wave < j1) {
    float slope2 = 0.0f;
    if constexpr (BIAS) slope2 = a.slopes[hd] * kLog2e8;
    const int64_t pos = start + i;
    // loads past the split's last block return zeros without going to memory, so the next
    // block's are issued without a branch (which doubled the registers that hold them)
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
    // the query's digits: features 64 kk + 16 g .. + 15
    v4i8 qd[kDigits][KK];
    float qscale;
    {
      float x[KK][16];
      uint32_t most = 0;
      const int64_t base = b * a.sqb + hd * a.sqh + i * a.sqs + 16 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
        for (int v = 0; v < 16 / Vec<QDT>::N; ++v)
          load_vec16<QDT>(a.q, base + 64 * kk + v * Vec<QDT>::N, x[kk] + v * Vec<QDT>::N);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t bits = __float_as_uint(x[kk][e]) & 0x7fffffffu;
          most = bits > most ? bits : most;
        }
      }
      most = col_umax(most);
      const float big = __uint_as_float(most);
      const float up = big > 0.0f ? kFixed / big : 0.0f;
      qscale = big / kFixed;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t y[4];
          int d[kDigits];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = fminf(fmaxf(x[kk][4 * w + e] * up, -kFixed), kFixed);
            y[e] = static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v)) + 0x8080);
          }
          digits4(y, d);
#pragma unroll
          for (int n = 0; n < kDigits; ++n) qd[n][kk][w] = d[n];
        }
    }
    for (; j < j1; j += NW) {
      const float kscale = ks[j], vscale = vs[j];
      float s[16];
      const float mul = qscale * kscale * a.dot_scale;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        v4i8 acc[kDigits];
#pragma unroll
        for (int d = 0; d < kDigits; ++d) {
          acc[d] = v4i8{0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][kk], qd[d][kk], acc[d], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[4 * t + e] = from_digits(acc, e) * mul;
      }
      load_k(j + NW);
      const int64_t ahead = pos - (j * kTok + 16 * g);
      const int left = ahead > 16 ? 16 : ahead < -1 ? -1 : static_cast<int>(ahead);
      const float d0 = static_cast<float>(ahead);  // key 16 g + x is seen for x <= left
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        float t = s[x];
        if constexpr (CAP) {
          const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(t) + 1.0f);
          t = __builtin_fmaf(-2.0f * a.cap2, r, a.cap2);
        }
        if constexpr (BIAS) t = __builtin_fmaf(-slope2, d0 - x, t);
        s[x] = x <= left ? t : -INFINITY;
        mx = fmaxf(mx, s[x]);
      }
      mx = col_max(mx);  // the block's own, the probabilities' unit
      const float mnew = fmaxf(m, mx);
      const float ref = mx == -INFINITY ? 0.0f : mx, nref = mnew == -INFINITY ? 0.0f : mnew;
      const float alpha = __builtin_amdgcn_exp2f(m - nref);
      const float beta = __builtin_amdgcn_exp2f(mx - nref);
      m = mnew;
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[x] = __builtin_amdgcn_exp2f(s[x] - ref);
        sum = sum + s[x];
      }
      v8bf_a p[NP][2];
      split_bf16<NP>(s, p);
      l = l * alpha + beta * col_sum(sum);
      // a block that the column does not see at all adds nothing, whatever its scale
      const float add = mx == -INFINITY && sum == 0.0f ? 0.0f : beta * vscale;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[f][e] = o[f][e] * alpha;
      }
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          widen_codes(static_cast<uint32_t>(vf[f][e]), w[2 * e], w[2 * e + 1]);
        const v8bf_a v[2] = {frag_of(make_uint4(w[0], w[1], w[2], w[3])),
                             frag_of(make_uint4(w[4], w[5], w[6], w[7]))};
        v4f_a acc{};
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], p[n][u], acc, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[f][e] = __builtin_fmaf(acc[e], add, o[f][e]);
      }
      load_v(j + NW);
    }
  }

  // the wavefronts
  if (g == 0) {
    sm[wave][col] = m;
    sl[wave][col] = l;
  }
#pragma unroll
  for (int f = 0; f < FT; ++f)
    *reinterpret_cast<float4*>(&so[wave][col][16 * f + 4 * g]) =
        make_float4(o[f][0], o[f][1], o[f][2], o[f][3]);
  __syncthreads();
  // a thread takes 4 features of one column at a time
  for (int idx = tid; idx < 16 * (D / 4); idx += NT) {
    const int c = idx / (D / 4), f = idx % (D / 4) * 4;
    const int64_t ct = tile * 16 + c;
    if (ct >= cols) break;
    float mm = sm[0][c];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w][c]);
    float ll = 0.0f, r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float x = sm[w][c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][c] - mm);
      // a NaN sum with no maximum still has to be seen
      ll = ll + (sl[w][c] == sl[w][c] ? x * sl[w][c] : sl[w][c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = __builtin_fmaf(x, so[w][c][f + e], r[e]);
    }
    if (a.nsplit == 1) {
      const int64_t qi = static_cast<uint32_t>(ct) / ug, h = kvh * a.G + (ct - qi * a.G);
      const float factor = row_factor(a, b, qi, ll);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = factor == 0.0f ? 0.0f : r[e] * factor;
      store4<ODT>(a.out, ((b * a.S + qi) * a.Hq + h) * D + f, r);
    } else {
      float* const w = a.work + ((bh * cols + ct) * a.nsplit + split) * (D + 4);
      *reinterpret_cast<float4*>(w + 4 + f) = make_float4(r[0], r[1], r[2], r[3]);
      if (f == 0) {
        w[0] = mm;
        w[1] = ll;
      }
    }
  }
}

// grid (columns, B * H), D / 4 threads: the splits of one column.
template <int D, int ODT>
__global__ __launch_bounds__(64) void kv8_join_kernel(Kv8Attn a) {
  const uint32_t uh = static_cast<uint32_t>(a.c.H), ub = blockIdx.y / uh;
  const int64_t ct = a.col0 + blockIdx.x, bh = blockIdx.y, b = ub, kvh = blockIdx.y - ub * uh;
  const int f = threadIdx.x * 4;
  const float* w = a.work + (bh * (a.S * a.G - a.col0) + blockIdx.x) * a.nsplit * (D + 4);
  const int64_t step = D + 4;
  float mm = -INFINITY, ll = 0.0f, r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  // eight splits' loads in flight, in one pass with a running maximum
  for (int64_t s0 = 0; s0 < a.nsplit; s0 += 8) {
    float ms[8], ls[8];
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float* at = w + (s0 + u < a.nsplit ? s0 + u : s0) * step;
      ms[u] = s0 + u < a.nsplit ? at[0] : -INFINITY;
      ls[u] = s0 + u < a.nsplit ? at[1] : 0.0f;
      v[u] = *reinterpret_cast<const float4*>(at + 4 + f);
    }
    float mn = mm;
#pragma unroll
    for (int u = 0; u < 8; ++u) mn = fmaxf(mn, ms[u]);
    const float c = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mm - mn);
    mm = mn;
    ll = ll == ll ? ll * c : ll;  // a NaN sum with no maximum still has to be seen
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = r[e] * c;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float x = ms[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[u] - mm);
      ll = ll + (ls[u] == ls[u] ? x * ls[u] : ls[u]);
      const float o4[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = ms[u] == -INFINITY ? r[e] : __builtin_fmaf(x, o4[e], r[e]);
    }
  }
  const int64_t qi = static_cast<uint32_t>(ct) / static_cast<uint32_t>(a.G);
  const int64_t h = kvh * a.G + (ct - qi * a.G);
  const float factor = row_factor(a, b, qi, ll);
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = factor == 0.0f ? 0.0f : r[e] * factor;
  store4<ODT>(a.out, ((b * a.S + qi) * a.Hq + h) * D + f, r);
}

// ---------------------------------------------------------------------------
// The same for chunks of many bf16 tokens with bf16 results (a prompt's next part): one workgroup
// takes 128 queries of a head, in two halves of four wavefronts that walk every other block; a
// wavefront takes 32 queries of its half, the halves are joined in LDS at the end, and the products
// run on the bf16 MFMA as in rk_attention.hip (scores transposed, a lane holds one query). The codes
// become bf16 once per half and block, exactly (8 bits), on their way into LDS; the key scale goes
// into the score, the value scale into the probabilities before they are rounded to bf16. Values lie
// by feature, so the second product's operand is a row read too: the tokens of a row are stored in
// the order in which a lane holds its probabilities. The next block's codes are in registers
// meanwhile.
//
// 4 x 517 tokens behind 1500, 16 heads of 128 (30 GFLOP): 73 us and 5 for the last tile's join;
// kv8_attn_kernel in its place took 176. A last tile of few queries is split over the keys
// (attention_plan): its workgroups were 25 of 96 us. Four wavefronts without the halves 82-86; the next block converted
// between the two products instead of behind them 99. The wavefronts of a half keep step with each
// other, so its MFMAs (1024 cycles a block and wavefront) and its vector instructions (590) overlap
// little: those two are what it spends its time on.
// ---------------------------------------------------------------------------
// A block's value scale: `fold` goes into the exponent of its probabilities, whose sum is
// multiplied by `inv`, and `rest` into its values. Scales whose products could leave float32's
// range leave a power of two to the values; one that is not finite makes its values zero and the
// sum NaN, which only the queries that see the block take over.
struct ValueScale {
  float fold, inv, rest;
  __device__ __forceinline__ explicit ValueScale(float s) : fold(s), inv(0.0f), rest(1.0f) {
    const bool finite = s <= 3.4028235e38f;
    if (!(s >= 0x1p-60f && s <= 0x1p60f)) {
      fold = !finite || s == 0.0f ? 1.0f : s < 1.0f ? s * 0x1p96f : s * 0x1p-96f;
      rest = !finite || s == 0.0f ? 0.0f : s < 1.0f ? 0x1p-96f : 0x1p96f;
    }
    inv = finite ? 1.0f / fold : __uint_as_float(0x7fc00000u);
  }
};

template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void kv8_chunk_kernel(Kv8Attn a) {
  constexpr int TILE = kTok * D * 2;    // bf16 keys [64][D] or values [D][64]
  constexpr int EACH = kTok * D / 16 / 256;  // 16-code pieces per thread and operand
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * 2 * 2 * TILE];
  // whole tiles first, the last queries, which see most, before the others; heads fastest
  const uint32_t uhq = static_cast<uint32_t>(a.Hq), uBHq = static_cast<uint32_t>(a.c.B) * uhq;
  const uint32_t full = static_cast<uint32_t>(a.S) / 128, nfull = static_cast<uint32_t>(a.nfull);
  const uint32_t turn = blockIdx.x / uBHq, ubh = blockIdx.x - turn * uBHq, ub = ubh / uhq;
  const bool whole_tile = turn < full * nfull;
  const int64_t qt = whole_tile ? full - 1 - turn / nfull : full;
  const int64_t split = whole_tile ? turn % nfull : turn - full * nfull;
  const uint32_t nsplit = static_cast<uint32_t>(whole_tile ? a.nfull : a.nsplit);
  const int64_t b = ub, hd = ubh - ub * uhq, kvh = (ubh - ub * uhq) / static_cast<uint32_t>(a.G);
  const int64_t bh = b * a.c.H + kvh;
  const int tid = threadIdx.x & 255, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);  // blocks half, half + 2, ..
  uint8_t* const smem = lds + half * 2 * 2 * TILE;
  const int64_t start = a.start[b * a.start_step];
  int64_t n = a.lengths ? a.lengths[b] : a.S;
  n = n < a.S ? n : a.S;
  const int64_t i0 = qt * 128, iw = i0 + 32 * wave, i = iw + l32;
  const bool on = start >= 0 && i0 < n;
  const int64_t last = i0 + 128 < n ? i0 + 127 : n - 1;  // the last active query
  int64_t nb = on ? ((start + last) >> 6) + 1 : 0;
  nb = nb < a.c.NB ? nb : a.c.NB;
  const int64_t per = (static_cast<uint32_t>(nb) + nsplit - 1) / nsplit;
  const int64_t j0 = split * per, j1 = j0 + per < nb ? j0 + per : nb;
  // positions relative to the split's first key
  const int64_t base = start - j0 * kTok;
  const int64_t pw = base + iw;                       // of the wavefront's first query
  const int64_t pos = base + (i < n ? i : n - 1);     // of this lane's

  float m = -INFINITY, l = 0.0f;
  v16f_a o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) o[dt] = v16f_a{};
  if (j0 < j1) {
    v8bf_a qf[D / 16];
    {
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.sqb + hd * a.sqh +
                          (i < a.S ? i : a.S - 1) * a.sqs + 8 * h;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
        qf[s] = frag_of(*reinterpret_cast<const uint4*>(q + 16 * s));
    }
    float slope2 = 0.0f;
    if constexpr (BIAS) slope2 = a.slopes[hd] * kLog2e8;
    const uint4* const kc =
        reinterpret_cast<const uint4*>(a.c.keys + (bh * a.c.NB + j0) * kTok * D) + tid;
    const uint4* const vc =
        reinterpret_cast<const uint4*>(a.c.values + (bh * a.c.NB + j0) * kTok * D) + tid;
    const float* const ks = a.c.ks + bh * a.c.NB + j0;
    const float* const vs = a.c.vs + bh * a.c.NB + j0;
    uint4 rk[EACH], rv[EACH];
    auto load = [&](int j) {
#pragma unroll
      for (int c = 0; c < EACH; ++c) {
        rk[c] = kc[static_cast<int64_t>(j) * (kTok * D / 16) + 256 * c];
        rv[c] = vc[static_cast<int64_t>(j) * (kTok * D / 16) + 256 * c];
      }
    };
    auto store = [&](int j) {
      uint8_t* const kt = smem + (j >> 1 & 1) * 2 * TILE;
      uint8_t* const vt = kt + TILE;
      const float power = ValueScale(vs[j]).rest;
#pragma unroll
      for (int c = 0; c < EACH; ++c) {
        const int p = tid + 256 * c;
        uint4 x[2];
        {
          const int row = p / (D / 16), seg = p % (D / 16) * 2, sw = seg_swizzle<D>(row);
          widen_codes(rk[c].x, x[0].x, x[0].y);
          widen_codes(rk[c].y, x[0].z, x[0].w);
          widen_codes(rk[c].z, x[1].x, x[1].y);
          widen_codes(rk[c].w, x[1].z, x[1].w);
          uint8_t* const to = kt + row * (2 * D);
          *reinterpret_cast<uint4*>(to + 16 * (seg ^ sw)) = x[0];
          *reinterpret_cast<uint4*>(to + 16 * ((seg + 1) ^ sw)) = x[1];
        }
        {  // tokens 0-3, 8-11 | 4-7, 12-15 of each 16: a lane's slots
          const int row = p / 4, seg = p % 4 * 2, sw = seg_swizzle<64>(row);
          if (power == 1.0f) {
            widen_codes(rv[c].x, x[0].x, x[0].y);
            widen_codes(rv[c].z, x[0].z, x[0].w);
            widen_codes(rv[c].y, x[1].x, x[1].y);
            widen_codes(rv[c].w, x[1].z, x[1].w);
          } else {
            widen_codes<true>(rv[c].x, x[0].x, x[0].y, power);
            widen_codes<true>(rv[c].z, x[0].z, x[0].w, power);
            widen_codes<true>(rv[c].y, x[1].x, x[1].y, power);
            widen_codes<true>(rv[c].w, x[1].z, x[1].w, power);
          }
          uint8_t* const to = vt + row * (2 * kTok);
          *reinterpret_cast<uint4*>(to + 16 * (seg ^ sw)) = x[0];
          *reinterpret_cast<uint4*>(to + 16 * ((seg + 1) ^ sw)) = x[1];
        }
      }
    };
    const int blocks = static_cast<int>(j1 - j0);
    if (half < blocks) {
      load(half);
      store(half);
      if (half + 2 < blocks) load(half + 2);
    }
    __syncthreads();
    for (int n2 = 0; n2 < blocks; n2 += 2) {
      const int j = n2 + half;
      const uint8_t* const kt = smem + (j >> 1 & 1) * 2 * TILE;
      const uint8_t* const vt = kt + TILE;
      const int64_t k0 = static_cast<int64_t>(j) * kTok;
      if (j < blocks && iw < n && k0 <= pw + 31) {  // some query of the wavefront sees some key
        const float kscale = ks[j] * a.dot_scale;
        const ValueScale v(vs[j]);
        const float vlog = __log2f(v.fold);
        v16f_a sc[2] = {v16f_a{}, v16f_a{}};
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<D>(kt, 32 * t, s, lane),
                                                            qf[s], sc[t], 0, 0, 0);
        const int64_t ahead = pos - k0 - 4 * h;
        const float d0 = static_cast<float>(ahead);
        // capped and biased scores in base-2 units here; plain ones are scaled with the max
        const float mul = CAP || BIAS ? 1.0f : kscale;
        if constexpr (CAP || BIAS) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int x = 32 * t + 8 * (e / 4) + (e % 4);
              float y = sc[t][e];
              if constexpr (CAP) {
                const float r =
                    __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y * kscale) + 1.0f);
                y = __builtin_fmaf(-2.0f * a.cap2, r, a.cap2);
                if constexpr (BIAS) y = __builtin_fmaf(-slope2, d0 - x, y);
              } else {
                y = __builtin_fmaf(y, kscale, -slope2 * (d0 - x));
              }
              sc[t][e] = y;
            }
        }
        const bool whole = k0 + kTok - 1 <= pw;
        const int left = ahead > kTok ? kTok : ahead < -1 ? -1 : static_cast<int>(ahead);
        if (!whole) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (32 * t + 8 * (e / 4) + (e % 4) > left) sc[t][e] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[t][e]);
        {
          const uint32_t bits = __float_as_uint(mx);
          const auto r = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
          mx = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
        // a zero key scale: every score is zero, also times a maximum of -inf
        const float mnew = fmaxf(m, mx == -INFINITY ? mx : mx * mul);
        const float mref = mnew == -INFINITY ? 0.0f : mnew;
        const float alpha = __builtin_amdgcn_exp2f(m - mref), shift = vlog - mref;
        m = mnew;
        float sum = 0.0f;
        uint4 pf[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            p[e] = __builtin_amdgcn_exp2f(CAP || BIAS ? sc[t][e] + shift
                                                      : __builtin_fmaf(sc[t][e], mul, shift));
          if (!whole) {  // (a zero key scale makes NaN of a masked score)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (32 * t + 8 * (e / 4) + (e % 4) > left) p[e] = 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) sum = sum + p[e];
          pack16(pf[t], p);
        }
        {
          const uint32_t bits = __float_as_uint(sum);
          const auto r = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
          sum = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        if (__any(alpha != 1.0f)) {
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * alpha;
        }
        l = l * alpha + (sum == 0.0f ? 0.0f : sum * v.inv);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                row_frag<64>(vt, 32 * dt, s, lane), frag_of(pf[s / 2][s % 2]), o[dt], 0, 0, 0);
      }
      if (j + 2 < blocks) {
        store(j + 2);
        if (j + 4 < blocks) load(j + 4);
      }
      if (n2 + 2 < blocks) __syncthreads();
    }
  }
  // the second half's state into the first's
  {
    float* const box = reinterpret_cast<float*>(lds) + tid;
    __syncthreads();
    if (half == 1) {
      box[0] = m;
      box[256] = l;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) box[256 * (2 + 16 * dt + e)] = o[dt][e];
    }
    __syncthreads();
    if (half == 1) return;
    const float m1 = box[0], l1 = box[256], mn = fmaxf(m, m1);
    const float c0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float c1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - mn);
    // a NaN sum with no maximum still has to be seen
    l = (l == l ? l * c0 : l) + (l1 == l1 ? l1 * c1 : l1);
    m = mn;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        o[dt][e] = __builtin_fmaf(box[256 * (2 + 16 * dt + e)], c1, o[dt][e] * c0);
  }
  if (i >= a.S) return;
  if (nsplit == 1) {
    uint16_t* const row = static_cast<uint16_t*>(a.out) + ((b * a.S + i) * a.Hq + hd) * D;
    const float factor = row_factor(a, b, i, l);
    if (factor == 0.0f) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] = v16f_a{};
    }
    store_owned<D>(row, o, factor, h);
  } else {
    const int64_t ct = i * a.G + (hd - kvh * a.G);
    float* const w =
        a.work + ((bh * (a.S * a.G - a.col0) + ct - a.col0) * a.nsplit + split) * (D + 4);
    if (h == 0) {
      w[0] = m;
      w[1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<float4*>(w + 4 + 32 * dt + 8 * r + 4 * h) =
            make_float4(o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static int check_cache(const rk_int8_kv& c) {
  if (c.B < 0 || c.H < 0 || c.blocks < 0) return fail(RK_ERR_ARG, "negative size");
  if (c.D != 64 && c.D != 128 && c.D != 256)
    return fail(RK_ERR_UNSUPPORTED, "head size %lld (64, 128 or 256)", static_cast<long long>(c.D));
  if (c.B == 0 || c.H == 0 || c.blocks == 0) return RK_OK;
  if (!c.keys || !c.values || !c.key_scales || !c.value_scales)
    return fail(RK_ERR_ARG, "null cache");
  if (!aligned16(c.keys) || !aligned16(c.values))
    return fail(RK_ERR_UNSUPPORTED, "the cache needs 16-byte alignment");
  if (c.B * c.H > 65535) return fail(RK_ERR_UNSUPPORTED, "more than 65535 sequence heads");
  if (c.blocks * kTok * c.D >= (int64_t{1} << 31) - (int64_t{1} << 20))
    return fail(RK_ERR_UNSUPPORTED, "a head's codes reach 2^31 bytes");
  return RK_OK;
}

static Kv8 cache_args(const rk_int8_kv& c) {
  return Kv8{c.keys, c.values, c.key_scales, c.value_scales, c.B, c.H, c.blocks};
}

// How a call is cut up: chunks of 128 queries of a head, or tiles of 16 columns; splits of the
// cache up to about `want` workgroups, each at least `least` blocks.
struct Kv8Plan {
  bool chunk;
  int waves;  // of a workgroup
  int64_t tiles, splits, full_splits, col0;
};

static Kv8Plan attention_plan(const rk_int8_kv& c, int64_t Hq, int64_t S, int qdtype, int odtype) {
  const int64_t G = Hq / c.H;
  Kv8Plan p{};
  p.chunk = qdtype == RK_BF16 && odtype == RK_BF16 && c.D <= 128 && S >= kChunkTokens;
  p.tiles = p.chunk ? (S + 127) / 128 : (S * G + 15) / 16;
  const int64_t have = p.tiles * c.B * (p.chunk ? Hq : c.H);
  const auto splits = [&](int64_t want, int64_t least) {
    const int64_t n = want / (have > 0 ? have : 1), most = (c.blocks + least - 1) / least;
    return n < 1 || most < 1 ? 1 : n < most ? n : most;
  };
  if (!p.chunk) {
    // few workgroups: eight wavefronts in each, so that up to 16 blocks need no join (16 and 128
    // heads of 128, 1000 tokens: 9.3 and 12.7 us a call; four wavefronts in splits 12.7 and 13.2; of
    // 4000 tokens 12.8 and 26, against 13.0 and 22.7, and above 128 always slower from there on);
    // otherwise as many workgroups as the device holds (twice as many gained nothing)
    // (head size 256 needs more registers than eight wavefronts have: 66 us with them, 40 with
    // four, at 8 sequences of 1.3 to 4 thousand tokens and 16 heads)
    p.waves = have <= 128 && c.D <= 128 ? 8 : 4;
    p.splits = splits(c.D == 64 ? 1024 : 512, p.waves == 8 ? 16 : 4);
    return p;
  }
  p.splits = p.full_splits = splits(256, 8);
  // a last tile of less than 64 queries behind whole ones: its few busy wavefronts would be the
  // launch's tail, so its keys are split (512 + 5 to 512 + 63 tokens behind 2000, 4 sequences, 16 heads
  // of 128: 86-91 us, unsplit 108-113; fuller ones would gain as much, 512 + 120: 93, unsplit 116)
  const int64_t full = S / 128, rest = S % 128;
  if (p.splits == 1 && full > 0 && rest > 0 && rest < 64 && c.blocks >= 16) {
    p.splits = c.blocks / 8 < 8 ? c.blocks / 8 : 8;
    p.col0 = full * 128 * G;
  }
  return p;
}

template <int D, int QDT, int ODT, int NW>
static void launch_kv8_attn(const Kv8Attn& a, bool cap, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.nsplit), static_cast<unsigned>(a.tiles),
                  static_cast<unsigned>(a.c.B * a.c.H));
  if (cap && a.slopes) kv8_attn_kernel<D, QDT, ODT, NW, true, true><<<grid, 64 * NW, 0, st>>>(a);
  else if (cap) kv8_attn_kernel<D, QDT, ODT, NW, true, false><<<grid, 64 * NW, 0, st>>>(a);
  else if (a.slopes) kv8_attn_kernel<D, QDT, ODT, NW, false, true><<<grid, 64 * NW, 0, st>>>(a);
  else kv8_attn_kernel<D, QDT, ODT, NW, false, false><<<grid, 64 * NW, 0, st>>>(a);
}

template <int D, int QDT, int ODT>
static void launch_kv8_waves(const Kv8Attn& a, const Kv8Plan& plan, bool cap, hipStream_t st) {
  if constexpr (D <= 128) {
    if (plan.waves == 8) return launch_kv8_attn<D, QDT, ODT, 8>(a, cap, st);
  }
  launch_kv8_attn<D, QDT, ODT, 4>(a, cap, st);
}

template <int D>
static void launch_kv8_chunk(const Kv8Attn& a, bool cap, hipStream_t st) {
  const int64_t turns = a.S / 128 * a.nfull + (a.S % 128 ? a.nsplit : 0);
  const dim3 grid(static_cast<unsigned>(turns * a.c.B * a.Hq));
  if (cap && a.slopes) kv8_chunk_kernel<D, true, true><<<grid, 512, 0, st>>>(a);
  else if (cap) kv8_chunk_kernel<D, true, false><<<grid, 512, 0, st>>>(a);
  else if (a.slopes) kv8_chunk_kernel<D, false, true><<<grid, 512, 0, st>>>(a);
  else kv8_chunk_kernel<D, false, false><<<grid, 512, 0, st>>>(a);
}

template <int D>
static void dispatch_kv8_attn(const Kv8Attn& a, const Kv8Plan& plan, bool cap, int qdt, int odt,
                              hipStream_t st) {
  if (plan.chunk) {
    if constexpr (D <= 128) launch_kv8_chunk<D>(a, cap, st);
  } else if (qdt == RK_F32) {
    if (odt == RK_F32) launch_kv8_waves<D, RK_F32, RK_F32>(a, plan, cap, st);
    else launch_kv8_waves<D, RK_F32, RK_BF16>(a, plan, cap, st);
  } else {
    if (odt == RK_F32) launch_kv8_waves<D, RK_BF16, RK_F32>(a, plan, cap, st);
    else launch_kv8_waves<D, RK_BF16, RK_BF16>(a, plan, cap, st);
  }
  if (a.nsplit > 1) {
    const dim3 grid(static_cast<unsigned>(a.S * a.G - a.col0),
                    static_cast<unsigned>(a.c.B * a.c.H));
    if (odt == RK_F32) kv8_join_kernel<D, RK_F32><<<grid, D / 4, 0, st>>>(a);
    else kv8_join_kernel<D, RK_BF16><<<grid, D / 4, 0, st>>>(a);
  }
}

}  // namespace rk

using namespace rk;

extern "C" int rk_int8_kv_append(const rk_int8_kv* cache, const void* k, int64_t skb, int64_t skh,
                                 int64_t sks, const void* v, int64_t svb, int64_t svh, int64_t svs,
                                 int dtype, int64_t S, const int64_t* start, int64_t start_count,
                                 const int64_t* lengths, void* stream) {
  clear_error();
  if (!cache) return fail(RK_ERR_ARG, "null cache");
  const rk_int8_kv& c = *cache;
  if (int e = check_cache(c)) return e;
  if (S < 0) return fail(RK_ERR_ARG, "negative size");
  if (dtype != RK_F32 && dtype != RK_BF16)
    return fail(RK_ERR_ARG, "keys and values must be float32 or bfloat16");
  if (start_count != 1 && start_count != c.B)
    return fail(RK_ERR_ARG, "one start, or one per sequence");
  if (c.B == 0 || c.H == 0 || c.blocks == 0 || S == 0) return RK_OK;
  if (!k || !v || !start) return fail(RK_ERR_ARG, "null pointer");
  const int64_t per = dtype == RK_F32 ? 4 : 8;
  const int64_t strides[] = {skb, skh, sks, svb, svh, svs};
  for (int64_t st : strides)
    if (st < 0 || st % per != 0)
      return fail(RK_ERR_UNSUPPORTED, "rows and strides must be whole 16-byte vectors");
  if (!aligned16(k) || !aligned16(v))
    return fail(RK_ERR_UNSUPPORTED, "keys and values need 16-byte alignment");
  if (S > (int64_t{1} << 29)) return fail(RK_ERR_UNSUPPORTED, "too many tokens");
  Kv8Append a{cache_args(c), k, v, skb, skh, sks, svb, svh, svs, start, lengths,
              start_count > 1 ? 1 : 0, S};
  // S tokens from any position touch at most this many blocks
  const dim3 grid(static_cast<unsigned>((S + kTok - 2) / kTok + 1),
                  static_cast<unsigned>(c.B * c.H), 2);
  hipStream_t st = as_stream(stream);
  const auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (c.D == 64) kv8_append_kernel<DT, 64><<<grid, 256, 0, st>>>(a);
    else if (c.D == 128) kv8_append_kernel<DT, 128><<<grid, 256, 0, st>>>(a);
    else kv8_append_kernel<DT, 256><<<grid, 256, 0, st>>>(a);
  };
  if (dtype == RK_F32) run(std::integral_constant<int, RK_F32>{});
  else run(std::integral_constant<int, RK_BF16>{});
  return launch_status("int8_kv_append");
}

extern "C" int rk_int8_kv_read(const rk_int8_kv* cache, int64_t begin, int64_t end, int dtype,
                               void* keys, void* values, void* stream) {
  clear_error();
  if (!cache) return fail(RK_ERR_ARG, "null cache");
  const rk_int8_kv& c = *cache;
  if (int e = check_cache(c)) return e;
  if (begin < 0 || end < begin || end > c.blocks * kTok)
    return fail(RK_ERR_ARG, "positions past the cache");
  if (dtype != RK_F32 && dtype != RK_BF16)
    return fail(RK_ERR_ARG, "values are read as float32 or bfloat16");
  if (c.B == 0 || c.H == 0 || end == begin) return RK_OK;
  if (!keys || !values) return fail(RK_ERR_ARG, "null pointer");
  if (!aligned16(keys) || !aligned16(values))
    return fail(RK_ERR_UNSUPPORTED, "keys and values need 16-byte alignment");
  Kv8Read a{cache_args(c), begin, end - begin, keys, values};
  const dim3 grid(static_cast<unsigned>((end + kTok - 1) / kTok - begin / kTok),
                  static_cast<unsigned>(c.B * c.H), 2);
  hipStream_t st = as_stream(stream);
  const auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (c.D == 64) kv8_read_kernel<DT, 64><<<grid, 256, 0, st>>>(a);
    else if (c.D == 128) kv8_read_kernel<DT, 128><<<grid, 256, 0, st>>>(a);
    else kv8_read_kernel<DT, 256><<<grid, 256, 0, st>>>(a);
  };
  if (dtype == RK_F32) run(std::integral_constant<int, RK_F32>{});
  else run(std::integral_constant<int, RK_BF16>{});
  return launch_status("int8_kv_read");
}

extern "C" int64_t rk_int8_kv_attention_work(const rk_int8_kv* cache, int64_t Hq, int64_t S,
                                             int qdtype, int odtype) {
  if (!cache || cache->B <= 0 || cache->H <= 0 || Hq <= 0 || S <= 0 || Hq % cache->H) return 0;
  const Kv8Plan p = attention_plan(*cache, Hq, S, qdtype, odtype);
  return p.splits == 1 ? 0
                       : cache->B * (Hq * S - cache->H * p.col0) * p.splits * (cache->D + 4);
}

extern "C" int rk_int8_kv_attention(const rk_int8_kv* cache, const void* q, int qdtype, int64_t sqb,
                                    int64_t sqh, int64_t sqs, int64_t Hq, int64_t S,
                                    const int64_t* start, int64_t start_count,
                                    const int64_t* lengths, float scale, float softcap,
                                    const float* slopes, float* work, int64_t work_floats,
                                    void* out, int odtype, void* stream) {
  clear_error();
  if (!cache) return fail(RK_ERR_ARG, "null cache");
  const rk_int8_kv& c = *cache;
  if (int e = check_cache(c)) return e;
  if (S < 0 || Hq < 0) return fail(RK_ERR_ARG, "negative size");
  if (c.H == 0 ? Hq != 0 : Hq % c.H != 0)
    return fail(RK_ERR_ARG, "query heads must be a multiple of the key heads");
  if ((qdtype != RK_F32 && qdtype != RK_BF16) || (odtype != RK_F32 && odtype != RK_BF16))
    return fail(RK_ERR_ARG, "queries and outputs are float32 or bfloat16");
  if (start_count != 1 && start_count != c.B)
    return fail(RK_ERR_ARG, "one start, or one per sequence");
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return fail(RK_ERR_ARG, "scale must be positive and finite");
  if (!(softcap >= 0.0f) || !(softcap < INFINITY))
    return fail(RK_ERR_ARG, "softcap must be finite and not negative (0: none)");
  if (softcap != 0.0f && !(softcap >= 1e-3f && softcap <= 1e3f))
    return fail(RK_ERR_UNSUPPORTED, "softcap outside 1e-3 .. 1e3");
  if (c.B == 0 || Hq == 0 || S == 0) return RK_OK;
  if (c.blocks == 0) return fail(RK_ERR_ARG, "an empty cache");
  if (!q || !start || !out) return fail(RK_ERR_ARG, "null pointer");
  const int64_t per = qdtype == RK_F32 ? 4 : 8;
  const int64_t strides[] = {sqb, sqh, sqs};
  for (int64_t st : strides)
    if (st < 0 || st % per != 0)
      return fail(RK_ERR_UNSUPPORTED, "query rows and strides must be whole 16-byte vectors");
  if (!aligned16(q) || !aligned16(out))
    return fail(RK_ERR_UNSUPPORTED, "queries and outputs need 16-byte alignment");
  const int64_t G = Hq / c.H;
  const Kv8Plan plan = attention_plan(c, Hq, S, qdtype, odtype);
  // a launch holds fewer than 2^23 blocks of 512 threads
  if (S * G >= (int64_t{1} << 24) || (!plan.chunk && plan.tiles > 65535) ||
      plan.tiles * c.B * Hq * plan.splits >= (int64_t{1} << 23))
    return fail(RK_ERR_UNSUPPORTED, "too many queries for one launch");
  const int64_t n = plan.splits;
  if (n > 1 && (!work || !aligned16(work) ||
                work_floats < rk_int8_kv_attention_work(&c, Hq, S, qdtype, odtype)))
    return fail(RK_ERR_ARG, "attention workspace too small");
  const bool cap = softcap > 0.0f;
  Kv8Attn a{cache_args(c), q, sqb, sqh, sqs, start, lengths, slopes, start_count > 1 ? 1 : 0, S,
            Hq, G, n, plan.tiles, plan.full_splits, plan.col0,
            cap ? 2.0f * kLog2e8 * (scale / softcap) : scale * kLog2e8, softcap * kLog2e8, work,
            out};
  hipStream_t st = as_stream(stream);
  if (c.D == 64) dispatch_kv8_attn<64>(a, plan, cap, qdtype, odtype, st);
  else if (c.D == 128) dispatch_kv8_attn<128>(a, plan, cap, qdtype, odtype, st);
  else dispatch_kv8_attn<256>(a, plan, cap, qdtype, odtype, st);
  return launch_status("int8_kv_attention");
}

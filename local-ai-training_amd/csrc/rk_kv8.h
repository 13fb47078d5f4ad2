// Pieces shared by the kernels of the 8-bit key/value cache (rk_kv8.hip) and those that attend over
// it from elsewhere (rk_tree.hip): its layout, codes widened to bf16, probabilities as sums of bf16
// numbers, reductions over the four lanes of a column of a 16 x 16 product.
#pragma once

#include "rk_attention.h"

namespace rk {

constexpr int kTok = 64;  // tokens of a block
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

int check_cache(const rk_int8_kv& c);

inline Kv8 cache_args(const rk_int8_kv& c) {
  return Kv8{c.keys, c.values, c.key_scales, c.value_scales, c.B, c.H, c.blocks};
}

}  // namespace rk

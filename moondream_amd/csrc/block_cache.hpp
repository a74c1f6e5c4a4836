// What the kernels over the 8-bit cache with block scales share: the numbers' form, and a block's quantisation by one wave.
#pragma once
#include "md_common.hpp"

typedef float md_f32x2v __attribute__((ext_vector_type(2)));

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// the least e with amax <= 448 * 2^e = 1.75 * 2^(e + 8), within the cache's range (amax == 0: the least)
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, MD_KV8_MIN_EXP), MD_KV8_MAX_EXP);
}

// four numbers times `inv` as e4m3, ties to even, saturated; NaN counts as 0 (a NaN in the cache would reach every query of its tile: a masked
// key's weight is 0, and 0 * NaN is not)
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d, float inv) {
  a = a == a ? a : 0.f;
  b = b == b ? b : 0.f;
  c = c == c ? c : 0.f;
  d = d == d ? d : 0.f;
  return pack_fp8x4(a * inv, b * inv, c * inv, d * inv);
}

__device__ __forceinline__ void kv8_unpack4(uint32_t w, float (&f)[4]) {
  const md_f32x2v lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  f[0] = lo[0];
  f[1] = lo[1];
  f[2] = hi[0];
  f[3] = hi[1];
}

// |x| where x is finite, else 0
__device__ __forceinline__ float kv8_magnitude(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;
}

constexpr int64_t MOST_GROUPS = (1 << 24) - 1;  // of 256 threads: a launch has fewer than 2^32

inline bool kv8_cache_ok(const md_kv8_cache* c) {
  return c && c->k && c->v && c->k_exp && c->v_exp && (c->head_dim == 64 || c->head_dim == 128) && c->slots > 0 && c->kv_heads > 0 && c->ctx > 0 &&
         c->ctx % MD_KV8_BLOCK == 0 && c->slot_stride % 16 == 0 && c->slot_stride >= (int64_t)c->kv_heads * c->ctx * c->head_dim &&
         c->exp_stride >= (int64_t)c->kv_heads * (c->ctx / MD_KV8_BLOCK) && (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0;
}

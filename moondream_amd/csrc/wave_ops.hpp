// Reductions and scans over a wave with DPP moves: neighbours' registers through the vector ALU.  A shuffle goes through LDS, where the waves of a
// compute unit queue: sixteen waves' chains of them took 3 us a round.
#pragma once
#include "md_common.hpp"

// v of the lane that CTRL names, `none` where there is none (or its row is not in ROWS)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false);
}

// op folded over rows of 16 lanes (shifts by 1, 2, 4, 8), then row 0 into 1 and 2 into 3, then rows 0, 1 into 2, 3: lane i has the fold over lanes 0 .. i
#define MD_DPP_STEPS(STEP) \
  STEP(0x111, 0xf)         \
  STEP(0x112, 0xf)         \
  STEP(0x114, 0xf)         \
  STEP(0x118, 0xf)         \
  STEP(0x142, 0xa)         \
  STEP(0x143, 0xc)

// sum over the lanes up to this one
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
#define MD_STEP(C, R) v += dpp<C, R>(v, 0u);
  MD_DPP_STEPS(MD_STEP)
#undef MD_STEP
  return v;
}

__device__ __forceinline__ uint32_t lane_63(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }

__device__ __forceinline__ uint32_t wave_most_u32(uint32_t v) {
#define MD_STEP(C, R) v = max(v, dpp<C, R>(v, 0u));
  MD_DPP_STEPS(MD_STEP)
#undef MD_STEP
  return lane_63(v);
}
// by the upper halves, which mostly differ; by the lower ones where they do not
__device__ __forceinline__ uint64_t wave_most_u64(uint64_t v) {
  const uint32_t hi = wave_most_u32((uint32_t)(v >> 32));
  const bool mine = (uint32_t)(v >> 32) == hi;
  const uint64_t who = __ballot(mine);
  const uint32_t lo = who & (who - 1) ? wave_most_u32(mine ? (uint32_t)v : 0u) : (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, __builtin_ctzll(who));
  return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ float wave_most_f32(float v) {
#define MD_STEP(C, R) v = fmaxf(v, __uint_as_float(dpp<C, R>(__float_as_uint(v), __float_as_uint(-INFINITY))));
  MD_DPP_STEPS(MD_STEP)
#undef MD_STEP
  return __uint_as_float(lane_63(__float_as_uint(v)));
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#define MD_STEP(C, R)                                                                                                                            \
  {                                                                                                                                              \
    const uint64_t u = __builtin_bit_cast(uint64_t, v);                                                                                          \
    v += __builtin_bit_cast(double, ((uint64_t)dpp<C, R>((uint32_t)(u >> 32), 0u) << 32) | dpp<C, R>((uint32_t)u, 0u));                          \
  }
  MD_DPP_STEPS(MD_STEP)
#undef MD_STEP
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, ((uint64_t)lane_63((uint32_t)(u >> 32)) << 32) | lane_63((uint32_t)u));
}

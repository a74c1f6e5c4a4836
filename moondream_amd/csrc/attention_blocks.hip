// Attention over the 8-bit cache with block scales.
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i . k_j) / sum over the rows j < limit(i)
//
// A COLUMN is one (query, head of the group): the heads that share a key head are columns of one matrix product, so a key is read and
// converted once for all of them.  A wave holds NT tiles of 16 columns and walks over blocks of 32 keys, everything in registers:
//   S^T [32 keys x 16 columns] = K Q^T       two tiles of v_mfma 16x16x32 bf16 per 32 coordinates; a lane's 16 bytes of a key row are its operand
//                                            of two products (an e4m3 number is exact in bf16; which coordinates share a product is free)
//   P = 2^(S * c + v_exp - m)                c = scale * log2(e) * 2^k_exp;  m the running maximum of the exponent
//   O^T [head_dim x 16 columns] += V^T P     v_mfma 16x16x32 f16.  The accumulator layout of S^T is the operand layout of P (keys 4 q .. 4 q + 3 of
//                                            both tiles in lane group q); V's operand is eight rows' bytes of one coordinate: a lane loads the
//                                            same 4 (8) coordinates of its eight rows and transposes them with byte permutes
// The value block's scale stands in the exponent (P holds p times 2^v_exp, V the bare codes), so blocks of any scales share one accumulator and
// fp16's range is spent where the output is made: l = sum over blocks of 2^-v_exp * (the block's sum of P), and o = O / l.
// m moves only when a column's exponent exceeds it by more than 8 (P <= 2^8): mostly one comparison instead of a reduction and a rescaling.
//
// Few columns (decode): the four waves of a workgroup share a column tile and take every fourth block, several workgroups share the keys, and
// a second kernel joins their (O, m, l).  Many columns (prompts): every wave has its own columns.
#include "block_cache.hpp"

#include <algorithm>

namespace {

constexpr int BLK = MD_KV8_BLOCK;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NO_MAX = -3.0e38f;   // running maximum before any key: 2^(-inf - NO_MAX) is 0, not NaN
constexpr float SLACK = 8.f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

struct Params {
  const uint8_t *k, *v, *ke, *ve;
  int64_t slot_stride, exp_stride;
  int slots, ctx, kv_heads;
  const bf16_t* q;
  int64_t q_bs, q_ts, q_hs;
  bf16_t* o;
  int64_t o_bs, o_ts, o_hs;
  const int32_t *slot, *q_pos0, *q_rows, *kv_len;
  int group, q_len, max_len, prefix, splits, col_groups, cols;
  float scale_log2, decay;
  float *part, *part_ml, *lse, *weights;  // part: [batch][kv_heads][cols][splits][head_dim], part_ml: ... [splits][2], lse: [batch][kv_heads][cols]
};

// What a sequence has: its slot (-1: none), keys, queries, and the row of query 0
struct Seq {
  int slot, len, rows, pos0;
};
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
  Seq s;
  s.slot = p.slot ? p.slot[b] : b;
  if (s.slot >= p.slots) s.slot = -1;
  s.len = s.slot < 0 ? 0 : min(max(p.kv_len[b], 0), p.max_len);
  s.rows = p.q_rows ? min(max(p.q_rows[b], 0), p.q_len) : p.q_len;
  s.pos0 = p.q_pos0 ? min(max(p.q_pos0[b], -p.q_len), p.max_len) : s.len - s.rows;
  return s;
}
// how many keys the query in row `pos` sees
__device__ __forceinline__ int limit_of(const Params& p, const Seq& s, int pos) {
  const int n = pos < 0 ? 0 : (pos < p.prefix ? max(pos + 1, p.prefix) : pos + 1);
  return min(n, s.len);
}

template <int HD>
struct Block {             // one lane's share of 32 keys and values
  u32x4 k[2][HD / 64];     // tile, 64 coordinates: row (lane & 15), bytes 16 (lane >> 4) ..
  uint32_t v[8][HD / 64];  // rows 4 q .. 4 q + 3 and 16 + 4 q .., bytes (HD / 16) (lane & 15) ..
  int ke, ve;
};

template <int HD>
__device__ __forceinline__ void load_block(Block<HD>& f, const uint8_t* k, const uint8_t* v, const uint8_t* ke, const uint8_t* ve, int block, int lane) {
  const int r = lane & 15, q = lane >> 4;
  const uint8_t* kb = k + (int64_t)block * BLK * HD;
  const uint8_t* vb = v + (int64_t)block * BLK * HD;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) f.k[t][c] = *(const u32x4*)(kb + (t * 16 + r) * HD + c * 64 + q * 16);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint8_t* at = vb + ((j < 4 ? 4 * q + j : 12 + 4 * q + j)) * HD + (HD / 16) * r;
    if constexpr (HD == 64) {
      f.v[j][0] = *(const uint32_t*)at;
    } else {
      const u32x2 w = *(const u32x2*)at;
      f.v[j][0] = w[0];
      f.v[j][1] = w[1];
    }
  }
  f.ke = ke[block];
  f.ve = ve[block];
}

// eight e4m3 codes -> bf16, eight -> fp16 (exact)
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t a, uint32_t b) {
  union {
    b16x2 h[4];
    bf16x8 v;
  } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return u.v;
}
__device__ __forceinline__ f16x8 codes_f16(uint32_t a, uint32_t b) {
  union {
    f16x2 h[4];
    f16x8 v;
  } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
  return u.v;
}

// w[j]: four coordinates of row j -> out[c]: coordinate c of the four rows
__device__ __forceinline__ void transpose4(const uint32_t (&w)[4], uint32_t (&out)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// the scores' product: 32 keys x 16 columns
template <int HD>
__device__ __forceinline__ void scores(const bf16x8 (&a)[2][HD / 32], const bf16x8 (&qf)[HD / 32], f32x4 (&s)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a[t][c]), __builtin_bit_cast(b16x8, qf[c]), s[t], 0, 0, 0);
  }
}

// a column's query as the scores' second operand: coordinates in the order in which a lane's bytes of a key hold them
template <int HD>
__device__ __forceinline__ void load_query(const Params& p, int b, int kvh, int col, int rows, int q, bf16x8 (&qf)[HD / 32]) {
  const int t = col / p.group, g = col - t * p.group;
#pragma unroll
  for (int c = 0; c < HD / 32; ++c) {
    qf[c] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (t < rows) qf[c] = *(const bf16x8*)(p.q + (int64_t)b * p.q_bs + (int64_t)t * p.q_ts + (int64_t)(kvh * p.group + g) * p.q_hs + (c >> 1) * 64 + q * 16 + (c & 1) * 8);
  }
}

__device__ __forceinline__ float over_q_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ float over_q_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}

// WK: waves of a workgroup that share columns and take the key blocks in turn; the other 4 / WK have columns of their own.
template <int HD, int NT, int WK>
__global__ __launch_bounds__(256) void attention_kernel(Params p) {
  constexpr int VT = HD / 16;  // tiles of 16 coordinates of the output
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x % p.splits, cg = blockIdx.x / p.splits, kvh = blockIdx.y, b = blockIdx.z;
  const Seq sq = sequence(p, b);
  const int n_cols = sq.rows * p.group;
  const int col0 = (cg * (4 / WK) + wave / WK) * 16 * NT;
  if constexpr (WK == 1) {
    if (col0 >= n_cols) return;
  } else {
    if (cg * 16 * NT >= n_cols) return;  // (all four waves)
  }

  bf16x8 qf[NT][HD / 32];
  int lim[NT], most = 0, least = 0x7fffffff;
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    const int col = col0 + ct * 16 + r;
    load_query<HD>(p, b, kvh, col, sq.rows, q, qf[ct]);
    lim[ct] = col < n_cols ? limit_of(p, sq, sq.pos0 + col / p.group) : 0;
    most = max(most, lim[ct]);
    if (col < n_cols) least = min(least, lim[ct]);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    most = max(most, __shfl_xor(most, o, 64));
    least = min(least, __shfl_xor(least, o, 64));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);

  f32x4 acc[NT][VT];
  float m[NT], l[NT];
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    m[ct] = NO_MAX;
    l[ct] = 0.f;
#pragma unroll
    for (int t = 0; t < VT; ++t) acc[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int blocks = (most + BLK - 1) / BLK, per = (blocks + p.splits - 1) / p.splits;
  const int begin = split * per, end = min(begin + per, blocks);
  const int64_t head = (int64_t)max(sq.slot, 0) * p.slot_stride + (int64_t)kvh * p.ctx * HD;
  const int64_t ehead = (int64_t)max(sq.slot, 0) * p.exp_stride + (int64_t)kvh * (p.ctx / BLK);
  const uint8_t *k = p.k + head, *v = p.v + head, *ke = p.ke + ehead, *ve = p.ve + ehead;

  const auto step = [&](Block<HD>& f, int block) {
    const int key0 = block * BLK;
    const float ck = p.scale_log2 * kv8_pow2(f.ke - 127), ev = (float)(f.ve - 127), back = kv8_pow2(127 - f.ve);
    if (key0 + BLK > sq.len) {  // rows behind the last may hold anything
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key0 + (j < 4 ? 4 * q + j : 12 + 4 * q + j) >= sq.len) {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) f.v[j][c] = 0;
        }
    }
    bf16x8 a[2][HD / 32];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) a[t][c] = codes_bf16(f.k[t][c >> 1][2 * (c & 1)], f.k[t][c >> 1][2 * (c & 1) + 1]);
    f32x4 s[NT][2];
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) scores<HD>(a, qf[ct], s[ct]);
    float top[NT];
    bool over = false;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      top[ct] = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[ct][t][i] = __builtin_fmaf(s[ct][t][i], ck, ev);
      if (key0 + BLK > least) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + t * 16 + 4 * q + i >= lim[ct]) s[ct][t][i] = -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[ct] = fmaxf(top[ct], s[ct][t][i]);
      over |= top[ct] > m[ct] + SLACK;
    }
    if (__any(over)) {
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const float now = fmaxf(m[ct], over_q_max(top[ct])), f0 = __builtin_amdgcn_exp2f(m[ct] - now);
        m[ct] = now;
        l[ct] *= f0;
#pragma unroll
        for (int t = 0; t < VT; ++t) acc[ct][t] *= f0;
      }
    }
    f16x8 pf[NT];
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      float sum = 0.f, e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = __builtin_amdgcn_exp2f(s[ct][j >> 2][j & 3] - m[ct]);
        sum += e[j];
      }
      l[ct] = __builtin_fmaf(sum, back, l[ct]);
      union {
        f16x2 h[4];
        f16x8 v;
      } u;
#pragma unroll
      for (int j = 0; j < 4; ++j) u.h[j] = __builtin_convertvector((md_f32pair{e[2 * j], e[2 * j + 1]}), f16x2);
      pf[ct] = u.v;
    }
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const uint32_t w0[4] = {f.v[0][c], f.v[1][c], f.v[2][c], f.v[3][c]}, w1[4] = {f.v[4][c], f.v[5][c], f.v[6][c], f.v[7][c]};
      uint32_t t0[4], t1[4];
      transpose4(w0, t0);
      transpose4(w1, t1);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f16x8 va = codes_f16(t0[t], t1[t]);
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) acc[ct][4 * c + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[ct], acc[ct][4 * c + t], 0, 0, 0);
      }
    }
  };

  // two blocks' registers in turn: one on its way while the other is worked on (a block past the end is the last one again)
  const int first = begin + (WK == 1 ? 0 : wave);
  if (first < end) {
    Block<HD> f0, f1;
    load_block<HD>(f0, k, v, ke, ve, first, lane);
    for (int block = first; block < end; block += 2 * WK) {
      load_block<HD>(f1, k, v, ke, ve, min(block + WK, end - 1), lane);
      step(f0, block);
      load_block<HD>(f0, k, v, ke, ve, min(block + 2 * WK, end - 1), lane);
      if (block + WK < end) step(f1, block + WK);
    }
  }
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) l[ct] = over_q_sum(l[ct]);

  // a lane holds, of column r, coordinates VT (4 q + i) + t at acc[t][i]: VT * 4 neighbours
  const int64_t bh = (int64_t)b * p.kv_heads + kvh;
  if constexpr (WK == 1) {
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const int col = col0 + ct * 16 + r;
      if (col >= n_cols) continue;
      if (p.splits > 1) {
        const int64_t at = (bh * p.cols + col) * p.splits + split;
        float* out = p.part + at * HD + 4 * VT * q;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < VT; t += 4) *(f32x4*)(out + VT * i + t) = f32x4{acc[ct][t][i], acc[ct][t + 1][i], acc[ct][t + 2][i], acc[ct][t + 3][i]};
        if (q == 0) {
          p.part_ml[at * 2] = m[ct];
          p.part_ml[at * 2 + 1] = l[ct];
        }
        continue;
      }
      const float inv = l[ct] == 0.f ? 0.f : 1.f / l[ct];
      const int t0 = col / p.group, g = col - t0 * p.group;
      bf16_t* out = p.o + (int64_t)b * p.o_bs + (int64_t)t0 * p.o_ts + (int64_t)(kvh * p.group + g) * p.o_hs + 4 * VT * q;
      uint32_t w[2 * VT];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < VT; t += 2) w[(VT * i + t) / 2] = pack_bf16x2(acc[ct][t][i] * inv, acc[ct][t + 1][i] * inv);
#pragma unroll
      for (int i = 0; i < VT / 2; ++i) *(u32x4*)(out + 8 * i) = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      if (p.lse && q == 0) p.lse[bh * p.cols + col] = l[ct] == 0.f ? INFINITY : m[ct] + __builtin_amdgcn_logf(l[ct]);
    }
  } else {
    static_assert(WK == 4 || WK == 1, "");
    __shared__ float so[4][VT * 4][64];
    __shared__ float sm[4][16], sl[4][16];
    for (int ct = 0; ct < NT; ++ct) {
      if (ct) __syncthreads();
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) so[wave][t * 4 + i][lane] = acc[ct][t][i];
      if (q == 0) {
        sm[wave][r] = m[ct];
        sl[wave][r] = l[ct];
      }
      __syncthreads();
      float f[4], mm = NO_MAX, ll = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w][r]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f[w] = __builtin_amdgcn_exp2f(sm[w][r] - mm);
        ll = __builtin_fmaf(sl[w][r], f[w], ll);
      }
      const int col = col0 + ct * 16 + r;
      if (col < n_cols) {  // wave i: coordinates VT (4 q + i) ..
        float out[VT];
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          out[t] = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) out[t] = __builtin_fmaf(so[w][t * 4 + wave][lane], f[w], out[t]);
        }
        const int at0 = VT * (4 * q + wave);
        if (p.splits > 1) {
          const int64_t at = (bh * p.cols + col) * p.splits + split;
#pragma unroll
          for (int t = 0; t < VT; t += 4) *(f32x4*)(p.part + at * HD + at0 + t) = f32x4{out[t], out[t + 1], out[t + 2], out[t + 3]};
          if (q == 0 && wave == 0) {
            p.part_ml[at * 2] = mm;
            p.part_ml[at * 2 + 1] = ll;
          }
        } else {
          const float inv = ll == 0.f ? 0.f : 1.f / ll;
          const int t0 = col / p.group, g = col - t0 * p.group;
          bf16_t* o = p.o + (int64_t)b * p.o_bs + (int64_t)t0 * p.o_ts + (int64_t)(kvh * p.group + g) * p.o_hs + at0;
#pragma unroll
          for (int t = 0; t < VT; t += 4) *(u32x2*)(o + t) = u32x2{pack_bf16x2(out[t] * inv, out[t + 1] * inv), pack_bf16x2(out[t + 2] * inv, out[t + 3] * inv)};
          if (p.lse && q == 0 && wave == 0) p.lse[bh * p.cols + col] = ll == 0.f ? INFINITY : mm + __builtin_amdgcn_logf(ll);
        }
      }
    }
  }
}

// Joins the workgroups that shared a column's keys: one wave per column, in the splits' order.
template <int HD>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr int N = HD / 64;
  const int lane = threadIdx.x & 63, col = blockIdx.x * 4 + (threadIdx.x >> 6), kvh = blockIdx.y, b = blockIdx.z;
  const int rows = p.q_rows ? min(max(p.q_rows[b], 0), p.q_len) : p.q_len;
  if (col >= rows * p.group) return;
  const int64_t c0 = ((int64_t)b * p.kv_heads + kvh) * p.cols + col;
  const float* ml = p.part_ml + c0 * p.splits * 2;
  const float* part = p.part + c0 * p.splits * HD + lane * N;
  float m = NO_MAX, l = 0.f, o[N] = {};
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * s]);
  for (int s = 0; s < p.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * s] - m);
    l = __builtin_fmaf(ml[2 * s + 1], f, l);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = __builtin_fmaf(part[(int64_t)s * HD + i], f, o[i]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int t = col / p.group, g = col - t * p.group;
  bf16_t* out = p.o + (int64_t)b * p.o_bs + (int64_t)t * p.o_ts + (int64_t)(kvh * p.group + g) * p.o_hs + lane * N;
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = f2bf(o[i] * inv);
  if (p.lse && lane == 0) p.lse[c0] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// The weight that every row got: one wave per block of 32 rows, the block's keys in registers, all columns that see it pass by; scores are the ones of
// the attention kernel again (the same products in the same order), exp2(score - lse) is their softmax.
template <int HD>
__global__ __launch_bounds__(256) void weights_kernel(Params p) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, kvh = blockIdx.y, b = blockIdx.z;
  const int block = blockIdx.x * 4 + (threadIdx.x >> 6), key0 = block * BLK;
  const Seq sq = sequence(p, b);
  if (key0 >= sq.len) return;
  const int64_t head = (int64_t)sq.slot * p.slot_stride + (int64_t)kvh * p.ctx * HD;
  const int64_t ehead = (int64_t)sq.slot * p.exp_stride + (int64_t)kvh * (p.ctx / BLK);
  const uint8_t* kb = p.k + head + (int64_t)key0 * HD;
  bf16x8 a[2][HD / 32];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const u32x4 w = *(const u32x4*)(kb + (t * 16 + r) * HD + c * 64 + q * 16);
      a[t][2 * c] = codes_bf16(w[0], w[1]);
      a[t][2 * c + 1] = codes_bf16(w[2], w[3]);
    }
  const float ck = p.scale_log2 * kv8_pow2((int)p.ke[ehead + block] - 127);
  float w[2][4] = {};
  const float* lse = p.lse + ((int64_t)b * p.kv_heads + kvh) * p.cols;
  const int n_cols = sq.rows * p.group;
  // queries from row key0 on see something of the block, those of the prefix if it begins within
  const int t0 = key0 < p.prefix ? 0 : min(max(key0 - sq.pos0, 0), sq.rows);
  for (int c0 = t0 * p.group; c0 < n_cols; c0 += 16) {
    const int col = c0 + r;
    bf16x8 qf[HD / 32];
    load_query<HD>(p, b, kvh, col, sq.rows, q, qf);
    const float ls = col < n_cols ? lse[col] : INFINITY;
    const int lim = col < n_cols ? limit_of(p, sq, sq.pos0 + col / p.group) : 0;
    f32x4 s[2];
    scores<HD>(a, qf, s);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[t][i] += key0 + t * 16 + 4 * q + i < lim ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], ck, -ls)) : 0.f;
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) w[t][i] += __shfl_xor(w[t][i], o, 64);
  if (r < 8) {
    const int t = r >> 2, i = r & 3, key = key0 + t * 16 + 4 * q + i;
    float mine = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine = j == r ? w[j >> 2][j & 3] : mine;
    if (key < sq.len) {
      float* out = p.weights + ((int64_t)sq.slot * p.kv_heads + kvh) * p.ctx + key;
      *out = p.decay == 0.f ? mine : __builtin_fmaf(p.decay, *out, mine);
    }
  }
}

// How a call is cut.  Up to 32 columns a wave's tiles would stand empty, and its keys are what there is to read: the four waves of a
// workgroup share them.  Splits: enough workgroups for 256 CUs of 4 workgroups each, none with less than 8 blocks (decode) or 16.
struct Plan {
  int nt, wk, col_groups, splits, cols;
  size_t part, ml, lse, bytes;
};

Plan plan_of(const md_kv8_cache* c, const md_kv8_attn_args* a) {
  Plan pl;
  pl.cols = a->q_len * (a->n_heads / c->kv_heads);
  pl.wk = pl.cols <= 32 ? 4 : 1;
  pl.nt = pl.wk == 4 ? (pl.cols <= 16 ? 1 : 2) : (c->head_dim == 64 ? 4 : 2);
  const int per = 16 * pl.nt * (4 / pl.wk);
  pl.col_groups = (pl.cols + per - 1) / per;
  const int max_len = a->max_len > 0 ? std::min(a->max_len, c->ctx) : c->ctx, blocks = (max_len + BLK - 1) / BLK;
  const int64_t groups = (int64_t)pl.col_groups * c->kv_heads * a->batch;
  const int64_t want = (1024 + groups - 1) / groups, most = std::max(1, blocks / (pl.wk == 4 ? 8 : 16));
  pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, 64}));
  const int64_t cols = (int64_t)a->batch * c->kv_heads * pl.cols;
  pl.part = 0;
  pl.ml = pl.splits > 1 ? cols * pl.splits * c->head_dim * 4 : 0;
  pl.lse = pl.ml + (pl.splits > 1 ? cols * pl.splits * 2 * 4 : 0);
  pl.bytes = pl.lse + (a->weights ? cols * 4 : 0);
  return pl;
}

bool args_ok(const md_kv8_cache* c, const md_kv8_attn_args* a) {
  if (!kv8_cache_ok(c) || !a || a->batch <= 0 || a->q_len <= 0 || a->n_heads <= 0 || a->n_heads % c->kv_heads != 0 || a->max_len < 0) return false;
  const int64_t cols = (int64_t)a->q_len * (a->n_heads / c->kv_heads);
  return cols <= 0x7fffff && a->batch <= 65535 && c->kv_heads <= 65535 && (a->slot || a->batch <= c->slots);
}

}  // namespace

extern "C" size_t md_kv8_attention_workspace_bytes(const md_kv8_cache* cache, const md_kv8_attn_args* args) {
  return args_ok(cache, args) ? plan_of(cache, args).bytes : 0;
}

extern "C" md_status md_kv8_attention(const md_kv8_cache* cache, const md_kv8_attn_args* a, void* stream) {
  MD_CHECK_ARG(args_ok(cache, a) && a->q && a->o && a->kv_len && a->prefix_len >= 0);
  MD_CHECK_ARG((((uintptr_t)a->q | (uintptr_t)a->o) & 15) == 0 && (a->q_bs | a->q_ts | a->q_hs | a->o_bs | a->o_ts | a->o_hs) % 8 == 0);
  MD_CHECK_ARG(a->scale > -INFINITY && a->scale < INFINITY && (!a->weights || (a->decay >= 0.f && a->decay < INFINITY)));
  const Plan pl = plan_of(cache, a);
  if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes)) return MD_ERR_WORKSPACE;
  MD_CHECK_ARG(((uintptr_t)a->workspace & 15) == 0);
  Params p;
  p.k = (const uint8_t*)cache->k;
  p.v = (const uint8_t*)cache->v;
  p.ke = (const uint8_t*)cache->k_exp;
  p.ve = (const uint8_t*)cache->v_exp;
  p.slot_stride = cache->slot_stride;
  p.exp_stride = cache->exp_stride;
  p.slots = cache->slots;
  p.ctx = cache->ctx;
  p.kv_heads = cache->kv_heads;
  p.q = (const bf16_t*)a->q;
  p.q_bs = a->q_bs, p.q_ts = a->q_ts, p.q_hs = a->q_hs;
  p.o = (bf16_t*)a->o;
  p.o_bs = a->o_bs, p.o_ts = a->o_ts, p.o_hs = a->o_hs;
  p.slot = a->slot, p.q_pos0 = a->q_pos0, p.q_rows = a->q_rows, p.kv_len = a->kv_len;
  p.group = a->n_heads / cache->kv_heads;
  p.q_len = a->q_len;
  p.max_len = a->max_len > 0 ? std::min(a->max_len, cache->ctx) : cache->ctx;
  p.prefix = a->prefix_len;
  p.splits = pl.splits, p.col_groups = pl.col_groups, p.cols = pl.cols;
  p.scale_log2 = a->scale * LOG2E;
  p.decay = a->decay;
  char* ws = (char*)a->workspace;
  p.part = (float*)(ws + pl.part);
  p.part_ml = (float*)(ws + pl.ml);
  p.lse = a->weights ? (float*)(ws + pl.lse) : nullptr;
  p.weights = a->weights;
  MD_CHECK_ARG((int64_t)pl.col_groups * pl.splits <= 0x7fffffff);
  const dim3 grid(pl.col_groups * pl.splits, cache->kv_heads, a->batch), block(256);
  hipStream_t s = (hipStream_t)stream;
#define MD_ATTN(HD, NT, WK) hipLaunchKernelGGL((attention_kernel<HD, NT, WK>), grid, block, 0, s, p)
  if (cache->head_dim == 64) {
    if (pl.wk == 1) MD_ATTN(64, 4, 1);
    else if (pl.nt == 1) MD_ATTN(64, 1, 4);
    else MD_ATTN(64, 2, 4);
  } else {
    if (pl.wk == 1) MD_ATTN(128, 2, 1);
    else if (pl.nt == 1) MD_ATTN(128, 1, 4);
    else MD_ATTN(128, 2, 4);
  }
#undef MD_ATTN
  MD_TRY(md_launch_status());
  if (pl.splits > 1) {
    const dim3 jg((pl.cols + 3) / 4, cache->kv_heads, a->batch);
    if (cache->head_dim == 64) hipLaunchKernelGGL(join_kernel<64>, jg, block, 0, s, p);
    else hipLaunchKernelGGL(join_kernel<128>, jg, block, 0, s, p);
    MD_TRY(md_launch_status());
  }
  if (a->weights) {
    const dim3 wg((((p.max_len + BLK - 1) / BLK) + 3) / 4, cache->kv_heads, a->batch);
    if (cache->head_dim == 64) hipLaunchKernelGGL(weights_kernel<64>, wg, block, 0, s, p);
    else hipLaunchKernelGGL(weights_kernel<128>, wg, block, 0, s, p);
    MD_TRY(md_launch_status());
  }
  return MD_OK;
}

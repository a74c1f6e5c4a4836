// Attention over the 8-bit cache with block scales.
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i . k_j) / sum over the rows j < limit(i)
//
// A COLUMN is one (query, head of the group): the heads that share a key head are columns of one matrix product, so a key is read and
// converted once for all of them.  A wave holds NT tiles of 16 columns and walks over blocks of 32 keys, everything in registers:
//   S^T [32 keys x 16 columns] = K Q^T       two tiles of v_mfma 16x16x32 bf16 per 32 coordinates; a lane's 16 bytes of a key row are its operand
//                                            of two products (an e4m3 number is exact in bf16; which coordinates share a product is free)
//   P = 2^(S * c + v_exp - m)                c = scale * log2(e) * 2^k_exp;  m the running maximum of the exponent less 7
//   O^T [head_dim x 16 columns] += V^T P     v_mfma 16x16x32 f16.  The accumulator layout of S^T is the operand layout of P (keys 4 q .. 4 q + 3 of
//                                            both tiles in lane group q); V's operand is eight rows' bytes of one coordinate: a lane loads the
//                                            same 4 (8) coordinates of its eight rows and transposes them with byte permutes
// The value block's scale stands in the exponent (P holds p times 2^v_exp, V the bare codes), so blocks of any scales share one accumulator and
// fp16's range is spent where the output is made: l = sum over blocks of 2^-v_exp * (the block's sum of P), and o = O / l.
// The largest P lies between 2^7 and 2^15, the top of fp16's range: a P keeps its 11 bits down to 2^-21 of the largest and something down to 2^-31.  (With the
// largest at 1 the many small weights behind a first row that takes 0.99 of the sum were subnormal or lost: 32768 rows' outputs off by 13 to 28 %.)  fp16 because bf16 would keep 8 bits of
// every weight, and a second product for the rest would double the work of the bound that there is.
// m moves only when a column's exponent exceeds it by more than 15 (P <= 2^15): mostly one comparison instead of a reduction and a rescaling.
//
// Few columns (decode): the waves of a workgroup share a column tile and take its blocks in turn, several workgroups share the keys, and a second
// kernel joins their (O, m, l).  Bound by the cache's bytes: 64 x 1003 rows of 32 heads of 64 (198 MB) in 38 us, 5.2 TB/s, the rate of a large copy.
// Many columns (prompts): every wave has its own columns, the converted operands come through LDS.  Bound by the sum of matrix and vector instructions, which
// take turns on a SIMD where accumulators are in vector registers: 8 x 767 queries of 32 heads of 64 at 700 TFLOP/s (53 us among other passes, 59 under the profiler; per block and wave 256 cycles of
// products and 650 of softmax and conversion come to the time measured), 2 x 2048 queries of 32 on 8 heads of 128 over 6101 rows at 850 (280 us).
// Accumulators in the other half of the registers, which overlap, were slower (68 and 345 us: inline assembly that the compiler does not schedule), as were
// scores of the next block made beside the softmax of this one (63 and 302 us: registers).
#include "block_cache.hpp"
#include "layout.hpp"
#include "wave_ops.hpp"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int BLK = MD_KV8_BLOCK;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NO_MAX = -3.0e38f;   // running maximum before any key: 2^(-inf - NO_MAX) is 0, not NaN
constexpr float LIFT = 7.f;          // the largest P stands at 2^LIFT when the maximum moves,
constexpr float SLACK = LIFT + 8.f;  // and at 2^SLACK, within fp16's 65504, before it does

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
  uint32_t per_group, all;  // 2^32 / group rounded up and 0; 0 and ~0 for a group of 1
  uint32_t q_sign;          // xor of two bf16 queries: a negative scale is taken as its magnitude and the queries negated, so that scores rise with products
  float scale_log2, decay;
  float *scores;            // kept for the weights: [batch][kv_heads][cols][max_len to a whole block], in units of log2
  int score_rows, join_groups, batch, by_length, col_splits;
  float* wpart;             // of many columns shared out: [col_splits][batch][kv_heads][max_len to a whole block]
  float *part, *part_ml, *weights;  // part: [batch][kv_heads][cols][splits][head_dim], part_ml: ... [splits][2]
  md_f32pair* norm;                 // with weights: [batch][kv_heads][cols], norm_of
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
// column -> query (exact: columns * group < 2^32)
__device__ __forceinline__ int query_of(const Params& p, int col) { return (int)(__umulhi((uint32_t)col, p.per_group) + ((uint32_t)col & p.all)); }

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

// the scores' product: KT tiles of 16 keys x NT of 16 columns, the independent accumulators in turn
template <int HD, int KT, int NT>
__device__ __forceinline__ void scores(const bf16x8 (&a)[KT][HD / 32], const bf16x8 (&qf)[NT][HD / 32], f32x4 (&s)[NT][KT]) {
#pragma unroll
  for (int ct = 0; ct < NT; ++ct)
#pragma unroll
    for (int t = 0; t < KT; ++t) s[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < HD / 32; ++c)
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int ct = 0; ct < NT; ++ct)
        s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a[t][c]), __builtin_bit_cast(b16x8, qf[ct][c]), s[ct][t], 0, 0, 0);
}

__device__ __forceinline__ bf16x8 query_at(const Params& p, const bf16_t* at) {
  return __builtin_bit_cast(bf16x8, *(const u32x4*)at ^ u32x4{p.q_sign, p.q_sign, p.q_sign, p.q_sign});
}

// a column's query as the scores' second operand: coordinates in the order in which a lane's bytes of a key hold them
template <int HD>
__device__ __forceinline__ void load_query(const Params& p, int b, int kvh, int col, int rows, int q, bf16x8 (&qf)[HD / 32]) {
  const int t = query_of(p, col), g = col - t * p.group;
#pragma unroll
  for (int c = 0; c < HD / 32; ++c) {
    qf[c] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (t < rows) qf[c] = query_at(p, p.q + (int64_t)b * p.q_bs + (int64_t)t * p.q_ts + (int64_t)(kvh * p.group + g) * p.q_hs + (c >> 1) * 64 + q * 16 + (c & 1) * 8);
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

// One block's softmax for NT tiles of columns: scores s -> pf, P as the second product's operand; m, l and acc move with it.  `edge`: some column does
// not see all of the block.
template <int NT, int VT>
__device__ __forceinline__ void softmax_block(f32x4 (&s)[NT][2], f16x8 (&pf)[NT], f32x4 (&acc)[NT][VT], float (&m)[NT], float (&l)[NT], const int (&lim)[NT],
                                              bool edge, int key0, int q, float ck, float ev, float back) {
  if (edge) {
#pragma unroll
    for (int ct = 0; ct < NT; ++ct)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + t * 16 + 4 * q + i >= lim[ct]) s[ct][t][i] = -INFINITY;
  }
  float top[NT], shift[NT];  // (whether a weight is too large is asked in the units in which it is made: scores of 2^24 and more are whole numbers, sums with m and ev too)
  bool over = false;
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    float a = s[ct][0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) a = fmaxf(a, s[ct][j >> 2][j & 3]);
    top[ct] = a;
    shift[ct] = ev - m[ct];
    over |= __builtin_fmaf(a, ck, shift[ct]) > SLACK;
  }
  if (__any(over)) {
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const float now = fmaxf(m[ct], over_q_max(__builtin_fmaf(top[ct], ck, ev)) - LIFT), f0 = __builtin_amdgcn_exp2f(m[ct] - now);
      m[ct] = now;
      shift[ct] = ev - now;
      l[ct] *= f0;
#pragma unroll
      for (int t = 0; t < VT; ++t) acc[ct][t] *= f0;
    }
  }
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    float sum = 0.f, e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][j >> 2][j & 3], ck, shift[ct]));
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
}

// A column's maximum and the reciprocal of its sum (0, 0 where it sees no key): a row's weight is 2^(score - maximum) times that.  (A log of the sum taken from the score
// instead rounds at its own size, and the hardware's log2 to one side: weights were 6e-7 too large.)  Where the sum is no number
// the maximum says so alone, so that a weight of 0 stays 0.
__device__ __forceinline__ md_f32pair norm_of(float m, float l) {
  return l == 0.f ? md_f32pair{0.f, 0.f} : (l == l ? md_f32pair{m, 1.f / l} : md_f32pair{l, 1.f});
}

// Writes column `col`'s coordinates at0 .. of a split, or its output; o[n] unnormalised
template <int HD, int N>
__device__ __forceinline__ void store_column(const Params& p, int b, int kvh, int col, int split, int at0, const float (&o)[N], float m, float l, bool first) {
  const int64_t c = ((int64_t)b * p.kv_heads + kvh) * p.cols + col;
  if (p.splits > 1) {
    float* out = p.part + (c * p.splits + split) * HD + at0;
#pragma unroll
    for (int i = 0; i < N; i += 4) *(f32x4*)(out + i) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
    if (first) {
      p.part_ml[(c * p.splits + split) * 2] = m;
      p.part_ml[(c * p.splits + split) * 2 + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int t = query_of(p, col), g = col - t * p.group;
  bf16_t* out = p.o + (int64_t)b * p.o_bs + (int64_t)t * p.o_ts + (int64_t)(kvh * p.group + g) * p.o_hs + at0;
#pragma unroll
  for (int i = 0; i < N; i += 4) *(u32x2*)(out + i) = u32x2{pack_bf16x2(o[i] * inv, o[i + 1] * inv), pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv)};
  if (p.norm && first) p.norm[c] = norm_of(m, l);
}

// The columns of a wave: queries, how many keys each sees, and the most and the least of them (a later query never sees less)
template <int HD, int NT>
__device__ __forceinline__ void load_columns(const Params& p, const Seq& sq, int b, int kvh, int col0, int n_cols, int lane, bf16x8 (&qf)[NT][HD / 32], int (&lim)[NT],
                                             int& most, int& least) {
  least = limit_of(p, sq, sq.pos0 + query_of(p, col0));
  most = col0 < n_cols ? limit_of(p, sq, sq.pos0 + query_of(p, min(col0 + 16 * NT, n_cols) - 1)) : 0;
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    const int col = col0 + ct * 16 + (lane & 15);
    load_query<HD>(p, b, kvh, col, sq.rows, lane >> 4, qf[ct]);
    lim[ct] = col < n_cols ? limit_of(p, sq, sq.pos0 + query_of(p, col)) : 0;
  }
}

// Few columns: the W waves share NT column tiles and take every W-th block, registers only.
template <int HD, int NT, int W>
__global__ __launch_bounds__(64 * W) void decode_kernel(Params p) {
  constexpr int VT = HD / 16;  // tiles of 16 coordinates of the output
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x % p.splits, cg = blockIdx.x / p.splits, kvh = blockIdx.y, b = blockIdx.z;
  const Seq sq = sequence(p, b);
  const int n_cols = sq.rows * p.group, col0 = cg * 16 * NT;
  if (col0 >= n_cols) return;

  bf16x8 qf[NT][HD / 32];
  int lim[NT], most, least;
  load_columns<HD, NT>(p, sq, b, kvh, col0, n_cols, lane, qf, lim, most, least);
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
    scores<HD, 2, NT>(a, qf, s);
    f16x8 pf[NT];
    const float ck = p.scale_log2 * kv8_pow2(f.ke - 127);
    if (p.scores) {
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const int col = col0 + ct * 16 + r;
        float* out = p.scores + (((int64_t)b * p.kv_heads + kvh) * p.cols + col) * p.score_rows + key0 + 4 * q;
        if (col < n_cols) {
          *(f32x4*)out = s[ct][0] * ck;
          *(f32x4*)(out + 16) = s[ct][1] * ck;
        }
      }
    }
    softmax_block<NT, VT>(s, pf, acc, m, l, lim, key0 + BLK > least, key0, q, ck, (float)(f.ve - 127), kv8_pow2(127 - f.ve));
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
  const int first = begin + wave;
  if (first < end) {
    Block<HD> f0, f1;
    load_block<HD>(f0, k, v, ke, ve, first, lane);
    for (int block = first; block < end; block += 2 * W) {
      load_block<HD>(f1, k, v, ke, ve, min(block + W, end - 1), lane);
      step(f0, block);
      load_block<HD>(f0, k, v, ke, ve, min(block + 2 * W, end - 1), lane);
      if (block + W < end) step(f1, block + W);
    }
  }
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) l[ct] = over_q_sum(l[ct]);

  // a lane holds, of column r, coordinates VT (4 q + i) + t at acc[t][i]
  __shared__ float so[W][VT * 4][64];
  __shared__ float sm[W][16], sl[W][16];
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
    if (wave >= 4) continue;
    float f[W], mm = NO_MAX, ll = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) mm = fmaxf(mm, sm[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      f[w] = __builtin_amdgcn_exp2f(sm[w][r] - mm);
      ll = __builtin_fmaf(sl[w][r], f[w], ll);
    }
    const int col = col0 + ct * 16 + r;
    if (col < n_cols) {  // wave i < 4: coordinates VT (4 q + i) ..
      float out[VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        out[t] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) out[t] = __builtin_fmaf(so[w][t * 4 + wave][lane], f[w], out[t]);
      }
      store_column<HD, VT>(p, b, kvh, col, split, VT * (4 * q + wave), out, mm, ll, q == 0 && wave == 0);
    }
  }
}

// The workgroup of rank `rank` among all sequences' groups of PER columns, the ones that reach farthest into their cache first (a batch's sequences differ
// in length, and what starts last should be short).  Group cg of a sequence reaches to row pos0 + (cg + 1) PER / group, in columns: base + (cg + 1) PER.
// Lane i counts sequence i's groups from a bound on; the bound is found by halving.  False: there are not so many groups.
template <int PER>
__device__ __forceinline__ bool longest_first(const Params& p, int rank, int lane, int& b, int& cg) {
  const Seq s = sequence(p, min(lane, p.batch - 1));
  const int n = lane < p.batch ? (s.rows * p.group + PER - 1) / PER : 0, base = s.pos0 * p.group;
  const auto sum = [](int v) { return (int)lane_63(wave_scan_u32((uint32_t)v)); };
  const auto from = [&](int bound) { return max(0, n - max(0, (bound - base + PER - 1) / PER - 1)); };
  if (rank >= sum(n)) return false;
  int hi = n ? base + n * PER : -0x40000000, lo = n ? base + PER : 0x40000000;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    hi = max(hi, __shfl_xor(hi, o, 64));
    lo = min(lo, __shfl_xor(lo, o, 64));
  }
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (sum(mid > base ? from(mid) : n) > rank) lo = mid;
    else hi = mid - 1;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int off = lo - base;
  const bool here = n && off > 0 && off % PER == 0 && off / PER <= n;
  uint64_t who = __ballot(here);
  for (int skip = rank - sum(lo + 1 > base ? from(lo + 1) : n); skip > 0; --skip) who &= who - 1;
  b = __builtin_ctzll(who);
  cg = __builtin_amdgcn_readlane(off, b) / PER - 1;
  return true;
}

// Many columns: every wave has its own NT tiles, and the four waves share the conversion: of the next two blocks, waves 0 and 1 bring the keys, 2 and 3
// the values into LDS as the products' operands (16 bytes per lane, one operand after another: no bank conflicts either way), while all work on
// the two before.  32 columns per wave: 48 and 64 need the registers of a third wave per SIMD, and larger workgroups even out worse over the CUs
// (compared before workgroups went by their reach, 8 x 767 queries, 32 heads of 64: 61 us against 66 and 67; 2 x 2048 queries over 6101 rows, 32 on 8 heads of 128: 359 against
// 364 and 559.  The times now stand at the head of this file.)
template <int HD, int NT>
__global__ __launch_bounds__(256, 3) void prompt_kernel(Params p) {
  constexpr int VT = HD / 16, KF = 2 * (HD / 32), W = HD / 64;
  constexpr int SB = HD == 64 ? 2 : 1;        // blocks of a step: of one block a wave brings a tile of the keys, or 64 coordinates of the values
  constexpr int T = SB, C = SB == 2 ? W : 1;  // tiles of keys and chunks of 64 coordinates of values that a wave brings
  __shared__ u32x4 frag[2][SB][KF + VT][64];  // [turn][block][operand][lane]
  __shared__ float scale[2][SB][2];           // [turn][block]: a key's exponent as a factor, a value's as a number
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  // Workgroup i runs on XCD i % 8, a head's workgroups on one XCD or few; of the columns that see most go first.
  int id = blockIdx.x, kvh, b, cg;
  const int split = id % p.splits;
  id /= p.splits;
  if (p.kv_heads % 8 == 0) {
    const int n = p.kv_heads / 8;
    kvh = (id >> 3) % n * 8 + (id & 7);
    id = (id >> 3) / n;
  } else {
    kvh = id % p.kv_heads;
    id /= p.kv_heads;
  }
  if (p.by_length) {
    if (!longest_first<64 * NT>(p, id, lane, b, cg)) return;
  } else {
    b = id % p.batch;
    cg = p.col_groups - 1 - id / p.batch;
  }
  const Seq sq = sequence(p, b);
  const int n_cols = sq.rows * p.group, wg0 = cg * 64 * NT, col0 = wg0 + wave * 16 * NT;
  if (wg0 >= n_cols) return;

  bf16x8 qf[NT][HD / 32];
  int lim[NT], most, least;
  load_columns<HD, NT>(p, sq, b, kvh, col0, n_cols, lane, qf, lim, most, least);
  f32x4 acc[NT][VT];
  float m[NT], l[NT];
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    m[ct] = NO_MAX;
    l[ct] = 0.f;
#pragma unroll
    for (int t = 0; t < VT; ++t) acc[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // the workgroup's blocks: what its last query sees, or what the prefix does
  const int first_pos = sq.pos0 + wg0 / p.group, last_pos = sq.pos0 + (min(n_cols, wg0 + 64 * NT) - 1) / p.group;
  const int wg_most = max(limit_of(p, sq, first_pos), limit_of(p, sq, last_pos));
  const int blocks = (wg_most + BLK - 1) / BLK, per = (blocks + p.splits - 1) / p.splits;
  const int begin = split * per, end = min(begin + per, blocks);
  const int64_t head = (int64_t)max(sq.slot, 0) * p.slot_stride + (int64_t)kvh * p.ctx * HD;
  const int64_t ehead = (int64_t)max(sq.slot, 0) * p.exp_stride + (int64_t)kvh * (p.ctx / BLK);
  const bool values = wave >= 2;
  const int mine = wave & 1, part = SB == 2 ? 0 : mine, of = SB == 2 ? mine : 0;  // which tile or chunk, of which block
  const uint8_t* codes = (values ? p.v : p.k) + head;
  const uint8_t* exps = (values ? p.ve : p.ke) + ehead;

  uint32_t st[8 * C > 4 * W * T ? 8 * C : 4 * W * T];
  int st_exp = 0;
  const auto fetch = [&](int block0) {
    const int block = min(block0 + of, end - 1);
    const uint8_t* at = codes + (int64_t)block * BLK * HD;
    if (!values) {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const u32x4 w = *(const u32x4*)(at + ((part + t) * 16 + r) * HD + c * 64 + q * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) st[(t * W + c) * 4 + j] = w[j];
        }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) st[j] = *(const uint32_t*)(at + ((j < 4 ? 4 * q + j : 12 + 4 * q + j)) * HD + (HD / 16) * r + 4 * part);
    }
    st_exp = exps[block];
  };
  const auto convert = [&](int turn, int block0) {
    if (!values) {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int c = 0; c < 2 * W; ++c)
          frag[turn][of][(part + t) * 2 * W + c][lane] = __builtin_bit_cast(u32x4, codes_bf16(st[t * 4 * W + 2 * c], st[t * 4 * W + 2 * c + 1]));
      if (lane == 0) scale[turn][of][0] = p.scale_log2 * kv8_pow2(st_exp - 127);
    } else {
      const int key0 = min(block0 + of, end - 1) * BLK;
      if (key0 + BLK > sq.len) {  // rows behind the last may hold anything
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + (j < 4 ? 4 * q + j : 12 + 4 * q + j) >= sq.len) st[j] = 0;
      }
      const uint32_t w0[4] = {st[0], st[1], st[2], st[3]}, w1[4] = {st[4], st[5], st[6], st[7]};
      uint32_t t0[4], t1[4];
      transpose4(w0, t0);
      transpose4(w1, t1);
#pragma unroll
      for (int t = 0; t < 4; ++t) frag[turn][of][KF + 4 * part + t][lane] = __builtin_bit_cast(u32x4, codes_f16(t0[t], t1[t]));
      if (lane == 0) scale[turn][of][1] = (float)(st_exp - 127);
    }
  };

  if (begin < end) {
    fetch(begin);
    convert(0, begin);
    fetch(begin + SB);
    __syncthreads();
    int turn = 0;
    for (int block0 = begin; block0 < end; block0 += SB, turn ^= 1) {
      if (block0 + SB < end) {
        convert(turn ^ 1, block0 + SB);
        fetch(block0 + 2 * SB);
      }
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        const int key0 = (block0 + i) * BLK;
        if (block0 + i >= end || key0 >= most) continue;  // (this wave's queries see none of it)
        const float ck = scale[turn][i][0], ev = scale[turn][i][1];
        bf16x8 a[2][HD / 32];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) a[t][c] = __builtin_bit_cast(bf16x8, frag[turn][i][t * (HD / 32) + c][lane]);
        f32x4 s[NT][2];
        scores<HD, 2, NT>(a, qf, s);
        f16x8 pf[NT];
        softmax_block<NT, VT>(s, pf, acc, m, l, lim, key0 + BLK > least, key0, q, ck, ev, __builtin_amdgcn_exp2f(-ev));
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          const f16x8 va = __builtin_bit_cast(f16x8, frag[turn][i][KF + t][lane]);
#pragma unroll
          for (int ct = 0; ct < NT; ++ct) acc[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[ct], acc[ct][t], 0, 0, 0);
        }
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    l[ct] = over_q_sum(l[ct]);
    const int col = col0 + ct * 16 + r;
    if (col >= n_cols) continue;
    float out[4 * VT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < VT; ++t) out[VT * i + t] = acc[ct][t][i];
    store_column<HD, 4 * VT>(p, b, kvh, col, split, 4 * VT * q, out, m[ct], l[ct], q == 0);
  }
}

// What the workgroups that shared a column's keys have: lane s holds split s's maximum as a factor; the common maximum, the sum
__device__ __forceinline__ float join_factor(const float* __restrict__ ml, int splits, int lane, float& m, float& l) {
  const float ms = lane < splits ? ml[2 * lane] : NO_MAX, ls = lane < splits ? ml[2 * lane + 1] : 0.f;
  m = wave_max(ms);
  const float f = __builtin_amdgcn_exp2f(ms - m);
  l = wave_sum(ls * f);
  return f;
}

// After workgroups that shared keys.  The first join_groups workgroups of a head: one wave per column, its parts added in the splits' order.  The others (few
// columns with kept scores): every row's softmax weights from the scores that the attention kernel left, 1024 rows each.
template <int HD>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr int N = HD / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kvh = blockIdx.y, b = blockIdx.z;
  const int64_t bh = (int64_t)b * p.kv_heads + kvh;
  const Seq sq = sequence(p, b);
  const int n_cols = sq.rows * p.group;
  if ((int)blockIdx.x < p.join_groups) {
    const int col = blockIdx.x * 4 + wave;
    if (col >= n_cols) return;
    const int64_t c0 = bh * p.cols + col;
    float m, l, f, o[N] = {};
    const float* part = p.part + c0 * p.splits * HD + lane * N;
    const auto add = [&](int s, auto many) {  // splits s .. s + U - 1, requested together
      constexpr int U = decltype(many)::value;
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) x[u][i] = part[(int64_t)min(s + u, p.splits - 1) * HD + i];
      if (s == 0) f = join_factor(p.part_ml + c0 * p.splits * 2, p.splits, lane, m, l);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float fu = s + u < p.splits ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s + u)) : 0.f;
        if (s + u < p.splits) {
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = __builtin_fmaf(x[u][i], fu, o[i]);
        }
      }
    };
    if (p.splits <= 8) {
      add(0, std::integral_constant<int, 8>());
    } else {
      for (int s = 0; s < p.splits; s += 16) add(s, std::integral_constant<int, 16>());
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int t = query_of(p, col), g = col - t * p.group;
    bf16_t* out = p.o + (int64_t)b * p.o_bs + (int64_t)t * p.o_ts + (int64_t)(kvh * p.group + g) * p.o_hs + lane * N;
    if constexpr (N == 1) *out = f2bf(o[0] * inv);
    else *(uint32_t*)out = pack_bf16x2(o[0] * inv, o[1] * inv);
    if (p.norm && lane == 0) p.norm[c0] = norm_of(m, l);
    return;
  }
  __shared__ md_f32pair norm[24];  // (kept scores are those of up to 24 columns)
  __shared__ int lims[24];
  const int first = (blockIdx.x - p.join_groups) * 1024;
  if (first >= sq.len) return;
  for (int col = wave; col < n_cols; col += 4) {
    const int64_t c0 = bh * p.cols + col;
    md_f32pair x;
    if (p.splits > 1) {
      float m, l;
      join_factor(p.part_ml + c0 * p.splits * 2, p.splits, lane, m, l);
      x = norm_of(m, l);
    } else {
      x = p.norm[c0];
    }
    if (lane == 0) {
      norm[col] = x;
      lims[col] = limit_of(p, sq, sq.pos0 + query_of(p, col));
    }
  }
  __syncthreads();
  const int key = first + (int)threadIdx.x * 4;
  if (key >= sq.len) return;
  const float* sc = p.scores + bh * p.cols * p.score_rows + key;
  float w[4] = {};
  for (int col = 0; col < n_cols; ++col) {
    const md_f32pair of = norm[col];
    const int lim = lims[col];
    if (key >= lim) continue;  // (its scores may not be there)
    const f32x4 s = *(const f32x4*)(sc + (int64_t)col * p.score_rows);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] += key + i < lim ? __builtin_amdgcn_exp2f(s[i] - of[0]) * of[1] : 0.f;
  }
  float* out = p.weights + ((int64_t)sq.slot * p.kv_heads + kvh) * p.ctx + key;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + i < sq.len) out[i] = p.decay == 0.f ? w[i] : __builtin_fmaf(p.decay, out[i], w[i]);
}

// The weight that every row got, from scores made again.  A wave holds 32 keys as operands (64 would leave registers for two waves per SIMD, and exponentials and
// products of one wave follow each other: 201 us against 228 at that step for 2 x 2048 queries over 6101 rows, 32 on 8 heads of 128); the columns that see them pass by, 64 at a time
// through LDS for the four waves.  Where that makes few workgroups the columns are shared out too (the first keys are seen by all queries, the last by few: whole columns left
// 42 % of the CUs' time empty), and the shares added in their order afterwards.  The scores are the attention kernel's again (the same products in the same order),
// 2^(score - maximum) over the sum is their softmax.
template <int HD>
__global__ __launch_bounds__(256, 4) void weights_kernel(Params p) {
  constexpr int KT = 2, QF = HD / 32, COLS = 64;  // key tiles, operands of a column tile, columns on their way
  __shared__ u32x4 frag[2][COLS / 16 * QF][64];
  __shared__ md_f32pair norms[2][COLS];
  __shared__ int lims[2][COLS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  // (the first keys, which most queries see, first for all heads)
  const int heads = p.kv_heads * p.batch, kvh = blockIdx.x % heads % p.kv_heads, b = blockIdx.x % heads / p.kv_heads, cs = blockIdx.y;
  const Seq sq = sequence(p, b);
  const int wg_key0 = blockIdx.x / heads * 64 * KT, key0 = wg_key0 + wave * 16 * KT;
  if (wg_key0 >= sq.len) return;
  const int64_t head = (int64_t)sq.slot * p.slot_stride + (int64_t)kvh * p.ctx * HD;
  const int64_t ehead = (int64_t)sq.slot * p.exp_stride + (int64_t)kvh * (p.ctx / BLK);
  bf16x8 a[KT][QF];
  float ck[KT], w[KT][4] = {};
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int key = min(key0 + t * 16, p.ctx - 16);  // (what lies past the cache counts for nothing below)
    ck[t] = p.scale_log2 * kv8_pow2((int)p.ke[ehead + key / BLK] - 127);
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const u32x4 x = *(const u32x4*)(p.k + head + (int64_t)(key + r) * HD + c * 64 + q * 16);
      a[t][2 * c] = codes_bf16(x[0], x[1]);
      a[t][2 * c + 1] = codes_bf16(x[2], x[3]);
    }
  }
  const md_f32pair* norm = p.norm + ((int64_t)b * p.kv_heads + kvh) * p.cols;
  const int n_cols = sq.rows * p.group;
  // queries from row wg_key0 on see something of these keys, those of the prefix if they begin within
  const int from = (wg_key0 < p.prefix ? 0 : min(max(wg_key0 - sq.pos0, 0), sq.rows)) * p.group;
  const int share = ((n_cols - from + COLS - 1) / COLS + p.col_splits - 1) / p.col_splits * COLS;  // of the columns, whole steps
  const int begin = min(from + cs * share, n_cols), end = min(begin + share, n_cols);

  // wave w brings column tile w: every lane its 16-byte pieces of one column
  u32x4 st[QF];
  md_f32pair st_norm = {0.f, 0.f};
  int st_lim = 0;
  const bf16_t* queries = p.q + (int64_t)b * p.q_bs + (int64_t)(kvh * p.group) * p.q_hs + q * 16;
  const auto fetch = [&](int c0) {
    const int want = c0 + wave * 16 + r, col = min(want, n_cols - 1), t = query_of(p, col), g = col - t * p.group;  // (one that is none sees no key)
    const bf16_t* at = queries + (int64_t)t * p.q_ts + (int64_t)g * p.q_hs;
#pragma unroll
    for (int c = 0; c < QF; ++c) st[c] = *(const u32x4*)(at + (c >> 1) * 64 + (c & 1) * 8);
    st_norm = norm[col];
    st_lim = want < n_cols ? limit_of(p, sq, sq.pos0 + t) : 0;
  };
  const auto put = [&](int turn) {
#pragma unroll
    for (int c = 0; c < QF; ++c) frag[turn][wave * QF + c][lane] = st[c] ^ u32x4{p.q_sign, p.q_sign, p.q_sign, p.q_sign};
    if (q == 0) {
      norms[turn][wave * 16 + r] = st_norm;
      lims[turn][wave * 16 + r] = st_lim;
    }
  };
  if (begin < end) {
    fetch(begin);
    put(0);
    fetch(begin + COLS);
    __syncthreads();
    int turn = 0;
    for (int c0 = begin; c0 < end; c0 += COLS, turn ^= 1) {
      if (c0 + COLS < end) {
        put(turn ^ 1);
        fetch(c0 + 2 * COLS);
      }
#pragma unroll
      for (int ct = 0; ct < COLS / 16; ++ct) {
        const md_f32pair of = norms[turn][ct * 16 + r];
        const int lim = lims[turn][ct * 16 + r];
        bf16x8 qf[1][QF];
#pragma unroll
        for (int c = 0; c < QF; ++c) qf[0][c] = __builtin_bit_cast(bf16x8, frag[turn][ct * QF + c][lane]);
        f32x4 sc[1][KT], (&s)[KT] = sc[0];
        scores<HD, KT, 1>(a, qf, sc);
        float top = of[0];
        if (__any(lim < key0 + 16 * KT)) {
          const float none = top - top;  // 0, or no number: that is for the rows that the query sees, and for no other
          top = none == none ? top : 0.f;
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[t][j] = key0 + t * 16 + 4 * q + j >= lim ? -INFINITY : s[t][j] + none;
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[t][j] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j], ck[t], -top)), of[1], w[t][j]);
          asm volatile("" : "+v"(w[t][0]), "+v"(w[t][1]), "+v"(w[t][2]), "+v"(w[t][3]));  // (tile by tile: or the compiler begins more of them than there are registers for, 203 -> 267 us)
        }
      }
      __syncthreads();
    }
  }
  // over the 16 columns of a tile; lane 4 t + j of a group of 16 has key 16 t + 4 q + j
  float mine = 0.f;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = w[t][j];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o, 64);
      mine = r == 4 * t + j ? x : mine;
    }
  const int key = key0 + (r >> 2) * 16 + 4 * q + (r & 3);
  if (r < 4 * KT && key < sq.len) {
    if (p.col_splits > 1) {
      p.wpart[(((int64_t)cs * p.batch + b) * p.kv_heads + kvh) * p.score_rows + key] = mine;
    } else {
      float* out = p.weights + ((int64_t)sq.slot * p.kv_heads + kvh) * p.ctx + key;
      *out = p.decay == 0.f ? mine : __builtin_fmaf(p.decay, *out, mine);
    }
  }
}

// The columns' shares of every row's weight together
__global__ __launch_bounds__(256) void weights_sum_kernel(Params p) {
  const int kvh = blockIdx.y, b = blockIdx.z, key = blockIdx.x * 256 + threadIdx.x;
  const Seq sq = sequence(p, b);
  if (key >= sq.len) return;
  float x = 0.f;
  for (int s = 0; s < p.col_splits; ++s) x += p.wpart[(((int64_t)s * p.batch + b) * p.kv_heads + kvh) * p.score_rows + key];
  float* out = p.weights + ((int64_t)sq.slot * p.kv_heads + kvh) * p.ctx + key;
  *out = p.decay == 0.f ? x : __builtin_fmaf(p.decay, *out, x);
}

// How a call is cut.  Up to 32 columns a wave's tiles would stand empty, and its keys are what there is to read: the waves of a workgroup share
// them.  Splits: enough workgroups for 256 CUs of 4 workgroups each, none with less than 8 blocks (decode) or 16.  Where that would be a second launch
// for little work, workgroups of 16 waves (8 where registers allow no more) take all keys of a head: one per CU at most, up to two blocks a wave,
// eight where half of the CUs have one (us, one launch against two: 1 x 32 heads of 64, 800 keys 7.0 / 8.2, 2000 keys 9.5 / 8.3; 8 x 32 heads 7.9 / 10.3
// and 13.3 / 17.1, 12 x 32 heads 14.0 / 13.7).
// Prompts: 32 columns a wave, 16 where more would stand empty (up to 64 columns) or where workgroups are few and short, so that one's latency counts, about
// a microsecond a block (us, 32 / 16 columns: 767 queries of 32 heads of 64 17.0 / 13.0, 2048 of 32 on 8 heads of 128 76 / 64, but 512 queries of 64 on 8 heads
// of 128 over 8192 rows 177 / 210).
// Weights of few columns come from kept scores where these cost less than the keys and their products again: 8 bytes a key and column, there and back, which up to 3 columns for 16
// coordinates is also a workspace of at most 3/8 of the cache's codes (us, kept / made again, 8 x 8 heads of 32768 keys: head size 64 with 4 columns 64 / 106, 12 95 / 104, 16 106 / 104,
// 32 185 / 107; head size 128 with 4 columns 129 / 190, 16 170 / 195, 24 200 / 202, 32 241 / 206).
struct Plan {
  bool decode, kept;  // kept: few columns' scores stay in the workspace for the weights
  int nt, waves, col_groups, splits, cols, score_rows, col_splits;
  size_t part, ml, norm, scores, bytes;
};

Plan plan_of(const md_kv8_cache* c, const md_kv8_attn_args* a) {
  Plan pl;
  pl.cols = a->q_len * (a->n_heads / c->kv_heads);
  pl.decode = pl.cols <= 32;
  const int max_len = a->max_len > 0 ? std::min(a->max_len, c->ctx) : c->ctx, blocks = (max_len + BLK - 1) / BLK;
  if (pl.decode) pl.nt = pl.cols <= 16 ? 1 : 2;
  else pl.nt = pl.cols <= 64 || (blocks <= 128 && (int64_t)((pl.cols + 127) / 128) * c->kv_heads * a->batch <= 512) ? 1 : 2;
  const int per = 16 * pl.nt * (pl.decode ? 1 : 4);
  pl.col_groups = (pl.cols + per - 1) / per;
  const int64_t groups = (int64_t)pl.col_groups * c->kv_heads * a->batch;
  const int wide = pl.nt == 1 && c->head_dim == 64 ? 16 : 8;
  pl.waves = pl.decode && groups <= 256 && blocks >= 16 && blocks <= (groups >= 128 ? 8 : 2) * wide ? wide : 4;
  const int64_t want = ((pl.decode ? 1024 : 512) + groups - 1) / groups, most = std::max(1, blocks / (pl.decode ? 8 : 16));
  pl.splits = pl.waves > 4 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({want, most, 64}));
  const int64_t cols = (int64_t)a->batch * c->kv_heads * pl.cols;
  pl.part = 0;
  pl.ml = pl.splits > 1 ? cols * pl.splits * c->head_dim * 4 : 0;
  pl.norm = pl.ml + (pl.splits > 1 ? cols * pl.splits * 2 * 4 : 0);
  pl.scores = (pl.norm + (a->weights ? cols * 8 : 0) + 15) & ~(size_t)15;
  pl.score_rows = blocks * BLK;
  const int64_t key_groups = (int64_t)((max_len + 127) / 128) * c->kv_heads * a->batch;
  pl.col_splits = (int)std::max<int64_t>(1, std::min<int64_t>({(3000 + key_groups - 1) / key_groups, (pl.cols + 255) / 256, 16}));
  pl.bytes = pl.scores;
  pl.kept = a->weights && pl.decode && pl.cols * 16 <= 3 * c->head_dim;
  if (pl.kept) pl.bytes += (size_t)cols * pl.score_rows * 4;
  if (a->weights && !pl.kept && pl.col_splits > 1) pl.bytes += (size_t)pl.col_splits * a->batch * c->kv_heads * pl.score_rows * 4;
  return pl;
}

bool args_ok(const md_kv8_cache* c, const md_kv8_attn_args* a) {
  if (!kv8_cache_ok(c) || !a || a->batch <= 0 || a->q_len <= 0 || a->n_heads <= 0 || a->n_heads % c->kv_heads != 0 || a->max_len < 0) return false;
  const int64_t cols = (int64_t)a->q_len * (a->n_heads / c->kv_heads);
  return cols <= 0x7fffff && cols * (a->n_heads / c->kv_heads) < (1ll << 32) && a->batch <= 65535 && c->kv_heads <= 65535 && (a->slot || a->batch <= c->slots);
}

// o: elements of its own, and none of them one of q's but for q itself
bool out_ok(const md_kv8_cache* c, const md_kv8_attn_args* a) {
  const StridedRuns q{(uintptr_t)a->q, c->head_dim * 2, {a->batch, a->q_len, a->n_heads}, {a->q_bs * 2, a->q_ts * 2, a->q_hs * 2}};
  const StridedRuns o{(uintptr_t)a->o, c->head_dim * 2, {a->batch, a->q_len, a->n_heads}, {a->o_bs * 2, a->o_ts * 2, a->o_hs * 2}};
  if (!runs_apart_from_each_other(o)) return false;
  if (a->o == (void*)a->q && runs_same_strides(q, o)) return !a->weights;  // (the weights are made from the queries again)
  return !runs_meet(q, o);
}

}  // namespace

extern "C" size_t md_kv8_attention_workspace_bytes(const md_kv8_cache* cache, const md_kv8_attn_args* args) {
  return args_ok(cache, args) ? plan_of(cache, args).bytes : 0;
}

extern "C" md_status md_kv8_attention(const md_kv8_cache* cache, const md_kv8_attn_args* a, void* stream) {
  MD_CHECK_ARG(args_ok(cache, a) && a->q && a->o && a->kv_len && a->prefix_len >= 0);
  MD_CHECK_ARG((((uintptr_t)a->q | (uintptr_t)a->o) & 15) == 0 && (a->q_bs | a->q_ts | a->q_hs | a->o_bs | a->o_ts | a->o_hs) % 8 == 0);
  MD_CHECK_ARG(out_ok(cache, a));
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
  p.per_group = p.group > 1 ? (uint32_t)((1ull << 32) / p.group + 1) : 0;
  p.all = p.group > 1 ? 0 : ~0u;
  p.q_len = a->q_len;
  p.max_len = a->max_len > 0 ? std::min(a->max_len, cache->ctx) : cache->ctx;
  p.prefix = a->prefix_len;
  p.splits = pl.splits, p.col_groups = pl.col_groups, p.cols = pl.cols;
  // (never 0: a masked score is -inf, and -inf * 0 is no number; 1e-25 times any score is as good)
  p.scale_log2 = std::max(fabsf(a->scale) * LOG2E, 1e-25f);
  p.q_sign = a->scale < 0.f ? 0x80008000u : 0u;
  p.decay = a->decay;
  char* ws = (char*)a->workspace;
  p.part = (float*)(ws + pl.part);
  p.part_ml = (float*)(ws + pl.ml);
  p.norm = a->weights ? (md_f32pair*)(ws + pl.norm) : nullptr;
  p.weights = a->weights;
  p.scores = pl.kept ? (float*)(ws + pl.scores) : nullptr;
  p.score_rows = pl.score_rows;
  p.wpart = (float*)(ws + pl.scores);
  p.col_splits = pl.col_splits;
  p.batch = a->batch;
  p.by_length = p.max_len >= 2048 && a->batch > 1 && a->batch <= 64 && ((int64_t)p.max_len + a->q_len + 128) * p.group < 0x3fffffff;
  p.join_groups = pl.splits > 1 ? (pl.cols + 3) / 4 : 0;
  const int64_t groups = (int64_t)pl.col_groups * pl.splits, all = groups * cache->kv_heads * a->batch;
  const int64_t key_groups = (int64_t)((p.max_len + 127) / 128) * cache->kv_heads * a->batch;
  MD_CHECK_ARG((pl.decode || all <= MOST_GROUPS) && (pl.kept || !a->weights || key_groups <= MOST_GROUPS));
  const dim3 grid(groups, cache->kv_heads, a->batch), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (pl.decode) {
#define MD_DECODE(HD, NT, W) hipLaunchKernelGGL((decode_kernel<HD, NT, W>), grid, dim3(64 * W), 0, s, p)
    if (cache->head_dim == 64) {
      if (pl.nt == 1) {
        if (pl.waves > 4) MD_DECODE(64, 1, 16);
        else MD_DECODE(64, 1, 4);
      } else {
        if (pl.waves > 4) MD_DECODE(64, 2, 8);
        else MD_DECODE(64, 2, 4);
      }
    } else {
      if (pl.nt == 1) {
        if (pl.waves > 4) MD_DECODE(128, 1, 8);
        else MD_DECODE(128, 1, 4);
      } else {
        if (pl.waves > 4) MD_DECODE(128, 2, 8);
        else MD_DECODE(128, 2, 4);
      }
    }
#undef MD_DECODE
  } else if (cache->head_dim == 64) {
    if (pl.nt == 1) hipLaunchKernelGGL((prompt_kernel<64, 1>), dim3(all), block, 0, s, p);
    else hipLaunchKernelGGL((prompt_kernel<64, 2>), dim3(all), block, 0, s, p);
  } else {
    if (pl.nt == 1) hipLaunchKernelGGL((prompt_kernel<128, 1>), dim3(all), block, 0, s, p);
    else hipLaunchKernelGGL((prompt_kernel<128, 2>), dim3(all), block, 0, s, p);
  }
  MD_TRY(md_launch_status());
  const int tail = p.join_groups + (p.scores ? (p.max_len + 1023) / 1024 : 0);
  if (tail) {
    const dim3 jg(tail, cache->kv_heads, a->batch);
    if (cache->head_dim == 64) hipLaunchKernelGGL(join_kernel<64>, jg, block, 0, s, p);
    else hipLaunchKernelGGL(join_kernel<128>, jg, block, 0, s, p);
    MD_TRY(md_launch_status());
  }
  if (a->weights && !pl.kept) {
    const dim3 wg(key_groups, pl.col_splits);
    if (cache->head_dim == 64) hipLaunchKernelGGL(weights_kernel<64>, wg, block, 0, s, p);
    else hipLaunchKernelGGL(weights_kernel<128>, wg, block, 0, s, p);
    if (pl.col_splits > 1) hipLaunchKernelGGL(weights_sum_kernel, dim3((p.max_len + 255) / 256, cache->kv_heads, a->batch), block, 0, s, p);
    MD_TRY(md_launch_status());
  }
  return MD_OK;
}

// The 8-bit cache with block scales: rows in (append), rows out (read), and the rows of least weight leave (evict).
//
// A block is 32 rows of one head.  One wave quantises a block: its largest magnitude gives the power of two, every lane holds 8 (append)
// or 16 (evict) neighbouring coordinates of a few rows, and any lane may hold any row, because the block has ONE scale; so every
// memory instruction of the wave covers whole rows, one after another.  All three are bound by memory: 12000 new rows of 32 heads of 64 in 36 us
// (4.1 TB/s) and back in 34 us (4.3 TB/s), 4096 of 32749 rows of 8 x 8 heads of 128 gathered in 33 us (4.0 TB/s).  A single row per sequence is
// latency: 64 sequences in 5.4 us.
#include "block_cache.hpp"
#include "layout.hpp"
#include "wave_ops.hpp"

#include <algorithm>

namespace {

constexpr int BLK = MD_KV8_BLOCK;

struct Cache {
  uint8_t *k, *v, *ke, *ve;
  int64_t slot_stride, exp_stride;
  int slots, ctx, heads;
};

Cache device_cache(const md_kv8_cache* c) {
  return {(uint8_t*)c->k, (uint8_t*)c->v, (uint8_t*)c->k_exp, (uint8_t*)c->v_exp, c->slot_stride, c->exp_stride, c->slots, c->ctx, c->kv_heads};
}

struct Rows {
  const bf16_t* x;
  int64_t bs, ts, hs;
};

// One wave per (sequence, block that the new rows touch, K or V, head); heads next to one another, as a token's heads are in memory.
template <int HD>
__global__ __launch_bounds__(256) void append_kernel(Cache c, Rows k, Rows v, const int32_t* __restrict__ slot, const int32_t* __restrict__ row0,
                                                     const int32_t* __restrict__ n_new, float* __restrict__ weights, int q_len, uint32_t n_blocks,
                                                     uint32_t n_tasks) {
  constexpr int CPR = HD / 8, N = BLK * CPR / 64;  // chunks of 8 coordinates: per row, per lane
  const int lane = threadIdx.x & 63;
  uint32_t task = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (task >= n_tasks) return;
  const int h = (int)(task % (uint32_t)c.heads);
  task /= (uint32_t)c.heads;
  const int which = (int)(task & 1);
  task >>= 1;
  const int nb = (int)(task % n_blocks), b = (int)(task / n_blocks);
  const int sl = slot ? slot[b] : b, r0 = row0[b], n = min(n_new ? n_new[b] : q_len, q_len);
  if (sl < 0 || sl >= c.slots || r0 < 0 || r0 >= c.ctx || n <= 0) return;
  const int end = min(n, c.ctx - r0) + r0;
  const int block = r0 / BLK + nb, base = block * BLK;
  if (base >= end) return;

  const Rows& in = which ? v : k;
  const bf16_t* x = in.x + (int64_t)b * in.bs + (int64_t)h * in.hs;
  uint8_t* codes = (which ? c.v : c.k) + (int64_t)sl * c.slot_stride + ((int64_t)h * c.ctx + base) * HD;
  uint8_t* ep = (which ? c.ve : c.ke) + (int64_t)sl * c.exp_stride + (int64_t)h * (c.ctx / BLK) + block;
  const int was = *ep;
  u32x4 q[N];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int ch = i * 64 + lane, r = base + ch / CPR;
    q[i] = u32x4{0, 0, 0, 0};
    if (r >= r0 && r < end) q[i] = *(const u32x4*)(x + (int64_t)(r - r0) * in.ts + (ch % CPR) * 8);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, fmaxf(kv8_magnitude(lo_bf(q[i][w])), kv8_magnitude(hi_bf(q[i][w]))));
  int e = kv8_exponent(wave_most_f32(top));
  if (base < r0) {  // older rows: their scale stays, or they are rounded to the larger one
    const int old = min(max(was - 127, MD_KV8_MIN_EXP), MD_KV8_MAX_EXP);
    if (e <= old) {
      e = old;
    } else {
      const float f = kv8_pow2(old - e);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ch = i * 64 + lane;
        if (base + ch / CPR >= r0) continue;
        u32x2 w = *(const u32x2*)(codes + ch * 8);
        float a[4], d[4];
        kv8_unpack4(w[0], a);
        kv8_unpack4(w[1], d);
        w[0] = kv8_pack4(a[0], a[1], a[2], a[3], f);
        w[1] = kv8_pack4(d[0], d[1], d[2], d[3], f);
        *(u32x2*)(codes + ch * 8) = w;
      }
    }
  }
  const float inv = kv8_pow2(-e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int ch = i * 64 + lane, r = base + ch / CPR;
    if (r < r0 || r >= end) continue;
    u32x2 w;
    w[0] = kv8_pack4(lo_bf(q[i][0]), hi_bf(q[i][0]), lo_bf(q[i][1]), hi_bf(q[i][1]), inv);
    w[1] = kv8_pack4(lo_bf(q[i][2]), hi_bf(q[i][2]), lo_bf(q[i][3]), hi_bf(q[i][3]), inv);
    *(u32x2*)(codes + ch * 8) = w;
  }
  if (lane == 0) *ep = (uint8_t)(e + 127);
  if (weights && which == 0 && lane < BLK && base + lane >= r0 && base + lane < end)  // (what an evicted row or the slot's last sequence left there)
    weights[((int64_t)sl * c.heads + h) * c.ctx + base + lane] = 0.f;
}

// 16 coordinates per thread: 16 bytes in, 32 out.  A workgroup belongs to one head's keys or values of one sequence, so that all but the row is the same
// for its threads.
template <int HD>
__global__ __launch_bounds__(256) void read_kernel(Cache c, const int32_t* __restrict__ slot, const int32_t* __restrict__ row0,
                                                   const int32_t* __restrict__ kv_len, int rows, uint32_t groups, bf16_t* __restrict__ ko,
                                                   bf16_t* __restrict__ vo) {
  constexpr int CPR = HD / 16;
  uint32_t id = blockIdx.x;
  const uint32_t part = id % groups;
  id /= groups;
  const int h = (int)(id % (uint32_t)c.heads);
  id /= (uint32_t)c.heads;
  const int which = id & 1, b = (int)(id >> 1);
  const int64_t i = (int64_t)part * blockDim.x + threadIdx.x;
  const int r = (int)(i / CPR), ch = (int)(i % CPR);
  if (r >= rows) return;
  const int sl = slot ? slot[b] : b, n = min(kv_len ? kv_len[b] : c.ctx, c.ctx);
  const int64_t row = (int64_t)(row0 ? row0[b] : 0) + r;
  u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (sl >= 0 && sl < c.slots && row >= 0 && row < n) {
    const u32x4 w = *(const u32x4*)((which ? c.v : c.k) + (int64_t)sl * c.slot_stride + ((int64_t)h * c.ctx + row) * HD + ch * 16);
    const float s = kv8_pow2((int)(which ? c.ve : c.ke)[(int64_t)sl * c.exp_stride + (int64_t)h * (c.ctx / BLK) + row / BLK] - 127);
    float f[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kv8_unpack4(w[j], f[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      lo[2 * j] = pack_bf16x2(f[j][0] * s, f[j][1] * s);
      lo[2 * j + 1] = pack_bf16x2(f[j][2] * s, f[j][3] * s);
      hi[2 * j] = pack_bf16x2(f[j + 2][0] * s, f[j + 2][1] * s);
      hi[2 * j + 1] = pack_bf16x2(f[j + 2][2] * s, f[j + 2][3] * s);
    }
  }
  bf16_t* out = (which ? vo : ko) + (((int64_t)b * c.heads + h) * rows * CPR + i) * 16;
  *(u32x4*)out = lo;
  *(u32x4*)(out + 8) = hi;
}

// ---------------------------------------------------------------------------------------------------------------- eviction
// weights as unsigned numbers of the same order; a NaN is the least (1; 0 is no row), a row that has to stay the largest
__device__ __forceinline__ uint32_t rank_key(float w, bool stays) {
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 and 0 are equal)
  const uint32_t key = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return stays ? 0xffffffffu : (w == w ? key : 1u);
}

constexpr int SEL = 1024;   // threads of the selection
constexpr int DIGIT = 11;   // bits of a key that one pass decides: three passes

// sums over the threads before this one, and of all; `part` has 16 places
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t* part, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t s = wave_scan_u32(v);
  if (lane == 63) part[wave] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SEL / 64; ++w) {
    const uint32_t p = part[w];
    before += w < wave ? p : 0;
    all += p;
  }
  total = all;
  __syncthreads();
  return before + s - v;
}

// One workgroup per (head, sequence): the keep-th largest key digit by digit (a histogram in LDS each), then the rows in their order: those above
// it, and as many of its equals, lowest first, as are still wanted.  Up to HELD * 1024 rows are read once and stay in registers, longer caches
// come by portion by portion in every pass.  Of a portion a wave has HELD * 64 rows in a row, a lane every 64th.  COPIES of the
// histogram lie in different banks, so that lanes that count the same digit (the first digit is sign, exponent and two bits: few are in use) mostly
// do so in different places.  Caches of up to 4096 rows take HELD 4, COPIES 2: 801 rows of 32 heads in 8 us against 25 with 32 and 8.
template <int HELD, int COPIES>
__global__ __launch_bounds__(SEL) void select_kernel(const float* __restrict__ weights, const int32_t* __restrict__ slot,
                                                     const int32_t* __restrict__ kv_len, int32_t* __restrict__ kept, int slots, int ctx, int heads, int keep,
                                                     int first, int recent) {
  constexpr int APART = (1 << DIGIT) + 4;
  __shared__ uint32_t hist[APART * COPIES];
  __shared__ uint32_t part[SEL / 64];
  __shared__ uint32_t found[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* out = kept + ((int64_t)b * heads + h) * keep;
  const int sl = slot ? slot[b] : b;
  const int len = sl < 0 || sl >= slots ? 0 : min(max(kv_len[b], 0), ctx);
  if (len <= keep) {
    for (int j = tid; j < keep; j += SEL) out[j] = j < len ? j : -1;
    return;
  }
  const float* w = weights + ((int64_t)sl * heads + h) * ctx;
  uint32_t key[HELD];
  const auto row_of = [&](int j0, int i) { return j0 + wave * (HELD * 64) + i * 64 + lane; };
  const auto load = [&](int j0) {
    float x[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) x[i] = w[min(row_of(j0, i), len - 1)];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int j = row_of(j0, i);
      key[i] = j < len ? rank_key(x[i], j < first || j >= len - recent) : 0u;
    }
  };
  const bool one = len <= HELD * SEL;
  if (one) load(0);
  uint32_t prefix = 0, mask = 0, want = keep;  // the key's leading digits, and how many of those that share them stay
  for (int shift = 32 - DIGIT;; shift = max(shift - DIGIT, 0)) {
    const int copies = mask == 0 ? COPIES : 1;  // (later on few keys are left that share the leading digits)
    for (int j = tid; j < APART * copies; j += SEL) hist[j] = 0;
    __syncthreads();
    for (int j0 = 0; j0 < len; j0 += HELD * SEL) {
      if (!one) load(j0);
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (key[i] != 0 && (key[i] & mask) == prefix) atomicAdd(&hist[((key[i] >> shift) & ((1 << DIGIT) - 1)) + (lane & (copies - 1)) * APART], 1u);
    }
    __syncthreads();
    // this thread's two digits, the larger first: how many keys lie above them
    const int d1 = (1 << DIGIT) - 1 - 2 * tid, d0 = d1 - 1;
    uint32_t n1 = 0, n0 = 0;
    for (int c = 0; c < copies; ++c) {
      n1 += hist[d1 + c * APART];
      n0 += hist[d0 + c * APART];
    }
    uint32_t total;
    const uint32_t above = scan_before(n1 + n0, part, total);
    if (above < want && above + n1 >= want) {
      found[0] = d1;
      found[1] = want - above;
    } else if (above + n1 < want && above + n1 + n0 >= want) {
      found[0] = d0;
      found[1] = want - above - n1;
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (uint32_t)((1 << DIGIT) - 1) << shift;
    want = found[1];
    __syncthreads();
    if (shift == 0) break;
  }
  // `prefix` is the key, `want` of its equals stay.  (The last pass's digit overlaps the one before by a bit, which is then settled.)
  uint32_t n_above = 0, n_equal = 0;
  for (int j0 = 0; j0 < len; j0 += HELD * SEL) {
    if (!one) load(j0);
    // above in the low half, equal in the high one: 32768 at most
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) mine += (key[i] > prefix ? 1u : 0u) + (key[i] == prefix ? 1u << 16 : 0u);
    uint32_t all, before = scan_before(mine, part, all);
    before = __builtin_amdgcn_readfirstlane(before);  // of the wave's first lane: all earlier waves'
    uint32_t na = n_above + (before & 0xffffu), ne = n_equal + (before >> 16);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      asm("" : "+v"(key[i]));  // (the comparisons are made again: 64 masks kept from above would be spilled)
      const bool above = key[i] > prefix, equal = key[i] == prefix;
      const uint64_t a = __ballot(above), e = __ballot(equal);
      const uint32_t eq = ne + __builtin_amdgcn_mbcnt_hi((uint32_t)(e >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)e, 0u));
      const uint32_t place = na + __builtin_amdgcn_mbcnt_hi((uint32_t)(a >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)a, 0u)) + min(eq, want);
      if (above || (equal && eq < want)) out[place] = row_of(j0, i);
      na += __popcll(a);
      ne += __popcll(e);
    }
    n_above += all & 0xffffu;
    n_equal += all >> 16;
  }
}

// One wave per block of 32 kept rows.  Another cache: a wave for every block of every head.  In place: one workgroup per (head, sequence, K or V)
// takes its blocks 16 at a time, all of them read before any is written; a kept row never moves up, so what later blocks read has not been
// written yet.  (With the choice, us into another cache / in place: 801 rows of 32 heads of 64 to 512 13.7 / 13.0; 8 x 8 heads of 32749 rows of 128 to 4096 48 / 69; one
// sequence of those, 16 workgroups in place, 26 / 58.)
template <int HD, bool IN_PLACE>
__global__ __launch_bounds__(IN_PLACE ? 1024 : 256) void gather_kernel(Cache from, Cache to, const float* weights, float* weights_out,
                                                                       const int32_t* __restrict__ slot, const int32_t* kv_len, int32_t* len_out,
                                                                       const int32_t* __restrict__ kept, int keep, int n_blocks, uint32_t n_tasks) {
  constexpr int CPR = HD / 16, N = BLK * CPR / 64, WAVES = IN_PLACE ? 16 : 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t task = IN_PLACE ? blockIdx.x : blockIdx.x * WAVES + wave;
  if (task >= n_tasks) return;
  int nb0 = wave;
  if constexpr (!IN_PLACE) {
    nb0 = (int)(task % (uint32_t)n_blocks);
    task /= (uint32_t)n_blocks;
  }
  const int which = (int)(task & 1);
  task >>= 1;
  const int h = (int)(task % (uint32_t)from.heads), b = (int)(task / (uint32_t)from.heads);
  const int sl = slot ? slot[b] : b;
  const bool there = sl >= 0 && sl < from.slots && sl < to.slots;
  if (which == 0 && h == 0 && nb0 == 0 && lane == 0) len_out[b] = there ? min(min(max(kv_len[b], 0), from.ctx), keep) : 0;
  if (!there) return;
  const int32_t* idx = kept + ((int64_t)b * from.heads + h) * keep;
  const uint8_t* src = (which ? from.v : from.k) + (int64_t)sl * from.slot_stride + (int64_t)h * from.ctx * HD;
  const uint8_t* se = (which ? from.ve : from.ke) + (int64_t)sl * from.exp_stride + (int64_t)h * (from.ctx / BLK);
  uint8_t* dst = (which ? to.v : to.k) + (int64_t)sl * to.slot_stride + (int64_t)h * to.ctx * HD;
  uint8_t* de = (which ? to.ve : to.ke) + (int64_t)sl * to.exp_stride + (int64_t)h * (to.ctx / BLK);
  const bool with_weights = which == 0 && weights_out != nullptr;
  const float* win = weights + ((int64_t)sl * from.heads + h) * from.ctx;
  float* wout = weights_out + (with_weights ? ((int64_t)sl * to.heads + h) * to.ctx : 0);

  for (int first = 0; first < (IN_PLACE ? n_blocks : 1); first += WAVES) {
    const int nb = IN_PLACE ? first + wave : nb0;
    const int r = nb * BLK + (lane & 31);
    const int my = r < keep ? idx[r] : -1;
    const float my_e = my >= 0 ? kv8_pow2(min(max((int)se[my / BLK] - 127, MD_KV8_MIN_EXP), MD_KV8_MAX_EXP)) : 0.f;
    const float my_w = with_weights && my >= 0 ? win[my] : 0.f;
    u32x4 q[N];
    float s[N], top = 0.f;
    bool live[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int ch = i * 64 + lane, row = __shfl(my, ch / CPR, 64);
      s[i] = __shfl(my_e, ch / CPR, 64);
      live[i] = row >= 0;
      q[i] = u32x4{0, 0, 0, 0};
      if (live[i]) q[i] = *(const u32x4*)(src + (int64_t)row * HD + (ch % CPR) * 16);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float m = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float f[4];
        kv8_unpack4(q[i][w], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, kv8_magnitude(f[j]));
      }
      top = fmaxf(top, m * s[i]);
    }
    const int e = kv8_exponent(wave_most_f32(top));
    const float inv = kv8_pow2(-e);
    if constexpr (IN_PLACE) __syncthreads();  // (every load of these blocks has arrived: their values are in use above)
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      any |= live[i];
      if (!live[i]) continue;
      const int ch = i * 64 + lane;
      const float f = s[i] * inv;
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a[4];
        kv8_unpack4(q[i][j], a);
        w[j] = kv8_pack4(a[0], a[1], a[2], a[3], f);
      }
      *(u32x4*)(dst + (int64_t)nb * BLK * HD + ch * 16) = w;
    }
    if (lane == 0 && any) de[nb] = (uint8_t)(e + 127);
    if (with_weights && lane < 32 && my >= 0) wout[r] = my_w;
  }
}

bool apart(const void* a, int64_t an, const void* b, int64_t bn) {
  return (uintptr_t)a + (uintptr_t)an <= (uintptr_t)b || (uintptr_t)b + (uintptr_t)bn <= (uintptr_t)a;
}

// keys, values and their scales, slot by slot (two layers' slots may lie between one another in a slab of all layers)
StridedRuns slots_of(const md_kv8_cache* c, int which) {
  const void* at[4] = {c->k, c->v, c->k_exp, c->v_exp};
  const int64_t rows = which < 2 ? (int64_t)c->ctx * c->head_dim : c->ctx / MD_KV8_BLOCK;
  return {(uintptr_t)at[which], c->kv_heads * rows, {c->slots, 1, 1}, {which < 2 ? c->slot_stride : c->exp_stride, 0, 0}};
}

bool caches_apart(const md_kv8_cache* a, const md_kv8_cache* b) {
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (runs_meet(slots_of(a, i), slots_of(b, j))) return false;
  return true;
}

}  // namespace

extern "C" md_status md_kv8_append(const md_kv8_cache* cache, const void* k, int64_t k_bs, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_bs,
                                   int64_t v_ts, int64_t v_hs, const int32_t* slot, const int32_t* row0, const int32_t* n_new, int32_t batch,
                                   int32_t q_len, void* stream) {
  return md_kv8_append_weighted(cache, k, k_bs, k_ts, k_hs, v, v_bs, v_ts, v_hs, slot, row0, n_new, nullptr, batch, q_len, stream);
}

extern "C" md_status md_kv8_append_weighted(const md_kv8_cache* cache, const void* k, int64_t k_bs, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_bs,
                                            int64_t v_ts, int64_t v_hs, const int32_t* slot, const int32_t* row0, const int32_t* n_new, float* weights,
                                            int32_t batch, int32_t q_len, void* stream) {
  MD_CHECK_ARG(kv8_cache_ok(cache) && k && v && row0 && batch > 0 && q_len > 0 && (slot || batch <= cache->slots));
  MD_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (k_bs | k_ts | k_hs | v_bs | v_ts | v_hs) % 8 == 0);
  const int n_blocks = (int)(((int64_t)std::min(q_len, cache->ctx) + 2 * BLK - 2) / BLK);  // wherever in a block the first row falls
  const int64_t tasks = (int64_t)batch * n_blocks * 2 * cache->kv_heads, groups = (tasks + 3) / 4;
  MD_CHECK_ARG(groups <= MOST_GROUPS);
  const Rows rk{(const bf16_t*)k, k_bs, k_ts, k_hs}, rv{(const bf16_t*)v, v_bs, v_ts, v_hs};
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(append_kernel<64>, dim3(groups), dim3(256), 0, (hipStream_t)stream, device_cache(cache), rk, rv, slot, row0, n_new, weights, q_len, (uint32_t)n_blocks, (uint32_t)tasks);
  else
    hipLaunchKernelGGL(append_kernel<128>, dim3(groups), dim3(256), 0, (hipStream_t)stream, device_cache(cache), rk, rv, slot, row0, n_new, weights, q_len, (uint32_t)n_blocks, (uint32_t)tasks);
  return md_launch_status();
}

extern "C" md_status md_kv8_read(const md_kv8_cache* cache, const int32_t* slot, const int32_t* row0, const int32_t* kv_len, int32_t batch, int32_t rows,
                                 void* k_out, void* v_out, void* stream) {
  MD_CHECK_ARG(kv8_cache_ok(cache) && k_out && v_out && batch > 0 && rows > 0 && (slot || batch <= cache->slots));
  MD_CHECK_ARG((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0);
  const int64_t chunks = (int64_t)rows * (cache->head_dim / 16), threads = chunks <= 128 ? 128 : 256, groups = (chunks + threads - 1) / threads;
  const int64_t all = groups * cache->kv_heads * 2 * batch;
  MD_CHECK_ARG(all <= MOST_GROUPS);
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(read_kernel<64>, dim3(all), dim3(threads), 0, (hipStream_t)stream, device_cache(cache), slot, row0, kv_len, rows, (uint32_t)groups,
                       (bf16_t*)k_out, (bf16_t*)v_out);
  else
    hipLaunchKernelGGL(read_kernel<128>, dim3(all), dim3(threads), 0, (hipStream_t)stream, device_cache(cache), slot, row0, kv_len, rows, (uint32_t)groups,
                       (bf16_t*)k_out, (bf16_t*)v_out);
  return md_launch_status();
}

extern "C" md_status md_kv8_evict(const md_kv8_cache* from, const md_kv8_cache* to, const md_kv8_evict_args* a, void* stream) {
  MD_CHECK_ARG(kv8_cache_ok(from) && kv8_cache_ok(to) && a && a->weights && a->kv_len && a->len_out && a->kept && a->batch > 0);
  MD_CHECK_ARG(from->kv_heads == to->kv_heads && from->head_dim == to->head_dim && a->keep > 0 && a->keep <= to->ctx);
  MD_CHECK_ARG(a->first >= 0 && a->recent >= 0 && (int64_t)a->first + a->recent <= a->keep);
  MD_CHECK_ARG((a->slot || (a->batch <= from->slots && a->batch <= to->slots)) && a->batch <= 65535);
  const bool in_place = from->k == to->k;
  const int64_t wn = (int64_t)from->slots * from->kv_heads * from->ctx * 4, wm = (int64_t)to->slots * to->kv_heads * to->ctx * 4;
  if (in_place) {
    MD_CHECK_ARG(from->v == to->v && from->k_exp == to->k_exp && from->v_exp == to->v_exp && from->slot_stride == to->slot_stride &&
                 from->exp_stride == to->exp_stride && from->slots == to->slots && from->ctx == to->ctx);
    MD_CHECK_ARG(!a->weights_out || a->weights_out == a->weights || apart(a->weights, wn, a->weights_out, wm));
  } else {
    MD_CHECK_ARG(caches_apart(from, to) && (!a->weights_out || apart(a->weights, wn, a->weights_out, wm)));
  }
  const int n_blocks = (a->keep + BLK - 1) / BLK;
  const int64_t heads2 = (int64_t)a->batch * from->kv_heads * 2, tasks = in_place ? heads2 : heads2 * n_blocks, groups = in_place ? tasks : (tasks + 3) / 4;
  MD_CHECK_ARG(groups <= (in_place ? MOST_GROUPS / 4 : MOST_GROUPS));
  hipStream_t s = (hipStream_t)stream;
#define MD_SELECT(HELD, COPIES)                                                                                                                    \
  hipLaunchKernelGGL((select_kernel<HELD, COPIES>), dim3(from->kv_heads, a->batch), dim3(SEL), 0, s, a->weights, a->slot, a->kv_len, a->kept,      \
                     std::min(from->slots, to->slots), from->ctx, from->kv_heads, a->keep, a->first, a->recent)
  if (from->ctx <= 4 * SEL) MD_SELECT(4, 2);
  else MD_SELECT(32, 8);
#undef MD_SELECT
#define MD_GATHER(HD, IP)                                                                                                                        \
  hipLaunchKernelGGL((gather_kernel<HD, IP>), dim3(groups), dim3(IP ? 1024 : 256), 0, s, device_cache(from), device_cache(to), a->weights,       \
                     a->weights_out, a->slot, a->kv_len, a->len_out, a->kept, a->keep, n_blocks, (uint32_t)tasks)
  if (from->head_dim == 64) {
    if (in_place) MD_GATHER(64, true);
    else MD_GATHER(64, false);
  } else {
    if (in_place) MD_GATHER(128, true);
    else MD_GATHER(128, false);
  }
#undef MD_GATHER
  return md_launch_status();
}

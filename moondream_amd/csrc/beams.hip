// Beam search: the best continuations over beams and vocabulary, and states moved behind their parents.
//
//   total(k, t) = score_k + logit_t - log sum_v exp(logit_v)
// Within a beam totals follow the logits, so a beam's candidates are its `beams` largest logits (ties: the lower token): one pass over the
// logits gives them and the sum, and only beams x beams totals are ever compared.
//   part_kernel    one workgroup per (beam, piece of the vocabulary): the piece in registers; each wave's largest logits, its maximum and its sum
//                  of exponentials
//   choose_kernel  one workgroup per input, one wave per beam: sums joined in 64 bits, the pieces' lists merged, totals; then the beams' lists merged
// Four beams of 51200 logits: 6.4 + 5.8 us, two launches' latency; 64 rows of 51200 bf16 logits 13.3 + 6.0 us; 64 rows of 131075 fp32 ones 26 us (1.3 TB/s: the
// vector instructions, some 1500 for a wave's 2048 logits, 600 of them the sum's in 64 bits, follow the loads, as all workgroups run at once) and 13.9 us for 16 beams.
// States move at 6.8 TB/s (16 x 4 beams, 1.6 GB in 235 us).
#include "layout.hpp"
#include "wave_ops.hpp"

#include <algorithm>

namespace {

// Logits of a thread; a workgroup's piece is 256 times as many.  32 keep the choice among the pieces short; where they make fewer workgroups than there
// are CUs, the latency of a thread's work counts: 8.
constexpr int MANY = 32, FEW = 8;
constexpr int MAXB = MD_MAX_BEAMS;
constexpr int LISTED = 7680;  // candidates of an input that choose_kernel has in LDS (30 pieces of 16 beams, 64 of up to 10)
constexpr int ROOM = 128;    // logits of a wave that are put in order together
constexpr int MOST_VOCAB = 0x7fffffff - 256 * MANY;  // (the places of the last piece are counted in 32 bits)
constexpr float F32_MOST = 3.4028234663852886e38f;

// (value, index) as one number: the larger value first, of equal ones the lower index.  0 stands for nothing.
__device__ __forceinline__ uint64_t candidate(float v, uint32_t index) {
  v = v == 0.f ? 0.f : v;  // -0 and 0 are equal
  const uint32_t u = __float_as_uint(v), o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(uint64_t c) {
  const uint32_t o = (uint32_t)(c >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t c) { return ~(uint32_t)c; }

// exp(x), x <= 0, in 64 bits: 2^n (1 + r q(r)), |r| <= log(2) / 2, q the polynomial of degree 8 through (e^r - 1) / r at nine Chebyshev points: 2^-44 off at most, and 1 at 0.
// In fp32 two beams whose sums differ by less than some 2^-24 would be ranked by rounding.  (64 rows of 131075 logits: 25.8 us, 21.0 with fp32's exponential.)
__device__ __forceinline__ double exp_of(double x) {
  constexpr double WHOLE = 6755399441055744.;  // 1.5 * 2^52: a sum with it ends in a whole number
  x = fmax(x, -700.);  // (e^-700 beside 1 is nothing, and 2^n is no subnormal)
  const double t = fma(x, 1.4426950408889634, WHOLE), n = t - WHOLE;
  const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));  // (log(2) in two parts)
  double q = 2.7625104515531025e-06;
  q = fma(q, r, 2.4876166784942655e-05);
  q = fma(q, r, 0.0001984120875246986);
  q = fma(q, r, 0.0013888821672653597);
  q = fma(q, r, 0.00833333335371942);
  q = fma(q, r, 0.041666666890981904);
  q = fma(q, r, 0.166666666666483);
  q = fma(q, r, 0.49999999999797906);
  q = fma(q, r, 1.0);
  const uint64_t e = __builtin_bit_cast(uint64_t, fma(q, r, 1.));
  return __builtin_bit_cast(double, e + (__builtin_bit_cast(uint64_t, t) << 52));  // (n into the exponent)
}

// 16 bytes of a row at any multiple of its elements' size
typedef u32x4 u32x4_anywhere __attribute__((aligned(2)));

// a beam that has continuations of its own
__device__ __forceinline__ bool goes_on(const float* scores, const int32_t* ended, int row) {
  return scores[row] > -INFINITY && (!ended || ended[row] == 0);
}

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit<bf16_t>(bf16_t x) { return bf2f(x); }
template <>
__device__ __forceinline__ float logit<float>(float x) { return x; }

template <typename T, int PER>
__global__ __launch_bounds__(256) void part_kernel(const T* __restrict__ logits, int64_t ld, int vocab, int beams, int suppress_id,
                                                   const float* __restrict__ scores, const int32_t* __restrict__ ended, int pieces,
                                                   uint64_t* __restrict__ best, double* __restrict__ sums) {
  constexpr int E = 16 / sizeof(T), N = PER / E, PIECE = 256 * PER;  // elements of a load, loads of a thread
  __shared__ uint64_t lists[4 * MAXB], found[4][ROOM];
  __shared__ float wmax[4];
  __shared__ double wsum[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, piece = blockIdx.x, row = blockIdx.y;
  if (!goes_on(scores, ended, row)) return;
  if (threadIdx.x < 8) lists[min(4 * beams + (int)threadIdx.x, 4 * MAXB - 1)] = 0;  // (the count runs over whole eights)
  __syncthreads();
  const T* x = logits + (int64_t)row * ld;
  const int base = piece * PIECE;  // (who has which token follows from the token alone, not from where the row lies: equal rows have equal sums)
  float v[PER];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = base + (i * 256 + (int)threadIdx.x) * E;
    if (at + E <= vocab) {
      const u32x4 w = *(const u32x4_anywhere*)(x + at);
      const T* e = (const T*)&w;
#pragma unroll
      for (int j = 0; j < E; ++j) v[i * E + j] = logit<T>(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) v[i * E + j] = at + j < vocab ? logit<T>(x[at + j]) : -INFINITY;
    }
  }
  const auto id_of = [&](int i) { return base + ((i / E) * 256 + (int)threadIdx.x) * E + i % E; };
  if (suppress_id >= 0 && (unsigned)(suppress_id - base) < (unsigned)PIECE) {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = id_of(i) == suppress_id ? -INFINITY : v[i];
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = v[i] == v[i] ? fminf(v[i], F32_MOST) : -INFINITY;
    top = fmaxf(top, v[i]);
  }
  const float m = wave_most_f32(top);
  double sum = 0.;
  if (m > -INFINITY) {
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += exp_of((double)v[i] - (double)m);
  }
  sum = wave_sum_f64(sum);

  // The wave's `beams` largest: at least as many logits reach the beams-th largest of the lanes' maxima, and seldom many more; those that do are
  // collected and put in order by counting.  Where very many do (equal logits), one after another is looked for.
  int above = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), j)) > top ? 1 : 0;
  const float least = -wave_most_f32(above < beams ? -top : -INFINITY);  // (of equal maxima all count as the first)
  int mine_n = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) mine_n += v[i] >= least && v[i] > -INFINITY ? 1 : 0;
  const uint32_t upto = wave_scan_u32((uint32_t)mine_n);
  const int n = (int)lane_63(upto);
  if (mine_n) {
    int place = (int)upto - mine_n;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (v[i] >= least && v[i] > -INFINITY) {
        if (place < ROOM) found[wave][place] = candidate(v[i], id_of(i));
        ++place;
      }
  }
  if (n <= ROOM) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wave's LDS accesses run in order)
    if (lane < beams) lists[wave * beams + lane] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i = lane; i < n; i += 64) {
      const uint64_t c = found[wave][i];
      int ahead = 0;
      for (int j = 0; j < n; j += 8)
#pragma unroll
        for (int u = 0; u < 8; ++u) ahead += found[wave][j + u] > c && j + u < n;  // (ROOM % 8 == 0)
      if (ahead < beams) lists[wave * beams + ahead] = c;
    }
  } else {
    uint64_t taken = ~0ull, mine = 0;
    const auto next = [&]() {  // this thread's largest below what it gave last
      mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint64_t c = candidate(v[i], id_of(i));
        if (v[i] > -INFINITY && c < taken && c > mine) mine = c;
      }
    };
    next();
    for (int k = 0; k < beams; ++k) {
      const uint64_t c = wave_most_u64(mine);
      if (lane == 0) lists[wave * beams + k] = c;
      if (c != 0 && c == mine) {
        taken = c;
        next();
      }
    }
  }
  if (lane == 0) {
    wmax[wave] = m;
    wsum[wave] = sum;
  }
  __syncthreads();
  if (wave == 0) {  // of at most 64 the largest, one per lane, each at the place that counting gives it
    const int n = (4 * beams + 7) & ~7;
    const uint64_t c = lane < n ? lists[lane] : 0;
    int ahead = 0;
    for (int j = 0; j < n; j += 8)  // (n % 8 == 0)
#pragma unroll
      for (int u = 0; u < 8; ++u) ahead += lists[j + u] > c || (lists[j + u] == c && j + u < lane);
    if (lane < n && ahead < beams) best[((int64_t)row * pieces + piece) * beams + ahead] = c;
    if (lane == 0) {
      const float mm = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
      double s = 0.;
      for (int w = 0; w < 4; ++w)
        if (wmax[w] > -INFINITY) s += wsum[w] * exp((double)wmax[w] - (double)mm);
      sums[((int64_t)row * pieces + piece) * 2] = (double)mm;
      sums[((int64_t)row * pieces + piece) * 2 + 1] = s;
    }
  }
}

struct Ranked {
  double rank;
  uint64_t logit;  // candidate(): the logit and its token
};

__global__ __launch_bounds__(64 * MAXB) void choose_kernel(int beams, int pieces, int end_id, const float* scores, const int32_t* ended,
                                                           const float* __restrict__ rank_weight, const uint64_t* __restrict__ best,
                                                           const double* __restrict__ sums, int32_t* __restrict__ tokens, int32_t* __restrict__ parents,
                                                           float* scores_out, int32_t* ended_out) {
  __shared__ uint64_t listed[LISTED];
  __shared__ Ranked cand[MAXB * MAXB];
  __shared__ double totals[MAXB * MAXB];
  const int lane = threadIdx.x & 63, k = threadIdx.x >> 6, b = blockIdx.x, row0 = b * beams, n = beams * beams, row = row0 + k;
  const float score = scores[row], weight = rank_weight ? rank_weight[row] : 1.f;
  if (!goes_on(scores, ended, row)) {  // (an ended beam of a score: itself, and nothing else)
    if (lane < beams) {
      const double rank = (double)score * (double)weight;
      const bool itself = lane == 0 && score > -INFINITY && rank > -INFINITY;
      cand[k * beams + lane] = {itself ? rank : -INFINITY, itself ? candidate(0.f, end_id) : 0};
      totals[k * beams + lane] = itself ? (double)score : -INFINITY;
    }
  } else {
    const uint64_t* list = best + (int64_t)row * pieces * beams;
    uint64_t carry = 0;  // carry: lane j has the j-th largest so far
    double m = -INFINITY, s = 0.;
    for (int i = 0; i < pieces; i += 64) {
      const bool in = i + lane < pieces;
      const double pm = in ? sums[((int64_t)row * pieces + i + lane) * 2] : -INFINITY, ps = in ? sums[((int64_t)row * pieces + i + lane) * 2 + 1] : 0.;
      const double now = fmax(m, (double)wave_most_f32((float)pm));  // (maxima of logits: exact in fp32)
      if (now > -INFINITY) {
        s = (m > -INFINITY ? s * exp(m - now) : 0.) + (pm > -INFINITY ? ps * exp(pm - now) : 0.);  // (this lane's share)
        m = now;
      }
    }
    s = wave_sum_f64(s);
    const double norm = m + log(s);
    // A piece's list is in falling order: lane i goes along piece i's, in LDS.  (As many pieces at a time as have room, 64 at most, the largest so far as one
    // more entry of each lane.)
    const int room = min(64, LISTED / n);
    uint64_t* mine = listed + k * room * beams;
    for (int first = 0; first < pieces; first += room) {
      const int here = min(room, pieces - first);
      for (int i = lane; i < here * beams; i += 64) mine[i] = list[first * beams + i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wave's LDS accesses run in order)
      uint64_t head = lane < here ? mine[lane * beams] : 0, got = 0;
      int at = lane * beams, last = at + beams - 1;
      for (int j = 0; j < beams; ++j) {
        const uint64_t w = wave_most_u64(head > carry ? head : carry);
        if (lane == j) got = w;
        if (carry == w) carry = 0;
        if (head == w && w != 0) head = at < last ? mine[++at] : 0;
      }
      carry = got;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (lane < beams) {
      const double total = carry ? (double)score + ((double)value_of(carry) - norm) : -INFINITY;
      const double rank = total * (double)weight;
      const bool real = total > -INFINITY && rank > -INFINITY;
      cand[k * beams + lane] = {real ? rank : -INFINITY, real ? carry : 0};
      totals[k * beams + lane] = real ? total : -INFINITY;
    }
  }
  __syncthreads();
  // (every input of this input's beams has been read: what follows may overwrite scores and ended)
  // Every beam's list is in falling order: lane i of the first wave goes along beam i's; of equal ranks the lower beam's is taken.
  if (k != 0) return;
  const auto key_of = [](const Ranked& c) {  // doubles as whole numbers of the same order; 0: no candidate
    const uint64_t u = __builtin_bit_cast(uint64_t, c.rank + 0.0);
    return c.logit == 0 ? 0 : (u >> 63) ? ~u : u | (1ull << 63);
  };
  const bool there = lane < beams;
  const int was_ended = there && ended ? ended[row0 + lane] : 0;
  int at = lane * beams;
  const int last = at + beams - 1;
  Ranked me = there ? cand[at] : Ranked{-INFINITY, 0};
  uint64_t key = key_of(me);
  int live = 0;
  for (; live < beams; ++live) {
    const uint64_t w = wave_most_u64(key);
    if (w == 0) break;
    if (lane == __builtin_ctzll(__ballot(key == w))) {
      const int token = (int)index_of(me.logit), to = row0 + live;
      tokens[to] = token;
      parents[to] = lane;
      scores_out[to] = (float)totals[at];
      if (ended_out) ended_out[to] = was_ended != 0 || token == end_id;
      me = at < last ? cand[++at] : Ranked{-INFINITY, 0};
      key = key_of(me);
    }
  }
  if (there && lane >= live) {
    tokens[row0 + lane] = end_id;
    parents[row0 + lane] = lane;
    scores_out[row0 + lane] = -INFINITY;
    if (ended_out) ended_out[row0 + lane] = 1;
  }
}

int per_thread(int64_t rows, int vocab) { return rows * ((vocab + 256 * MANY - 1) / (256 * MANY)) >= 256 ? MANY : FEW; }
size_t pieces_of(int64_t rows, int vocab) {
  const size_t piece = 256 * per_thread(rows, vocab);
  return ((size_t)vocab + piece - 1) / piece;
}

// ------------------------------------------------------------------------------------------------------------- states
constexpr int MAX_PARTS = 32;  // of a launch (88 bytes each in its arguments)

struct Part {
  const char* src;
  char* dst;
  int64_t src_slot, dst_slot, src_outer, dst_outer, src_seg, dst_seg;
  int32_t per_seg, segs;   // words of a run, runs of an outer index
  int32_t first, width;    // the part's first workgroup; bytes of a word
  uint32_t words;
};
struct Parts {
  Part p[MAX_PARTS];
  int n;
};

template <typename W, int B>
__device__ __forceinline__ void move_words(const Part& p, uint32_t first, const int32_t* __restrict__ parents, int beams, int64_t slot0) {
  const uint32_t w = first + threadIdx.x;
  if (w >= p.words) return;
  const uint32_t run = w / (uint32_t)p.per_seg, in = w - run * (uint32_t)p.per_seg, outer = run / (uint32_t)p.segs, seg = run - outer * (uint32_t)p.segs;
  const char* src = p.src + slot0 * p.src_slot + outer * p.src_outer + seg * p.src_seg + (int64_t)in * sizeof(W);
  char* dst = p.dst + slot0 * p.dst_slot + outer * p.dst_outer + seg * p.dst_seg + (int64_t)in * sizeof(W);
  const bool in_place = p.src == p.dst;
  W v[B];
#pragma unroll
  for (int i = 0; i < B; ++i) {
    if (i >= beams) continue;
    const int q = parents[i], from = q >= 0 && q < beams ? q : i;
    if (!in_place || from != i) v[i] = *(const W*)(src + from * p.src_slot);
  }
#pragma unroll
  for (int i = 0; i < B; ++i) {
    if (i >= beams) continue;
    const int q = parents[i], from = q >= 0 && q < beams ? q : i;
    if (!in_place || from != i) *(W*)(dst + i * p.dst_slot) = v[i];
  }
}

// One thread per word of a slot, for all beams of an input: every word is read from all parents before it is written to any child, so in place
// needs no second copy and no order among workgroups.
template <int B>
__global__ __launch_bounds__(256) void reorder_kernel(Parts parts, const int32_t* __restrict__ parents, int beams) {
  int i = 0;
  while (i + 1 < parts.n && (int)blockIdx.x >= parts.p[i + 1].first) ++i;
  const Part& p = parts.p[i];
  const int64_t slot0 = (int64_t)blockIdx.y * beams;
  const uint32_t first = (blockIdx.x - (uint32_t)p.first) * 256;
  if (p.width == 16) move_words<u32x4, B>(p, first, parents + slot0, beams, slot0);
  else if (p.width == 4) move_words<uint32_t, B>(p, first, parents + slot0, beams, slot0);
  else move_words<uint8_t, B>(p, first, parents + slot0, beams, slot0);
}

// bytes that a thread moves at once, and how many such words a slot has
int width_of(const md_state_part& s) {
  const uint64_t all = (uint64_t)s.src | (uint64_t)s.dst | (uint64_t)s.src_slot_stride | (uint64_t)s.dst_slot_stride | (uint64_t)s.src_outer_stride |
                       (uint64_t)s.dst_outer_stride | (uint64_t)s.src_seg_stride | (uint64_t)s.dst_seg_stride | (uint64_t)s.seg_bytes;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
}
int64_t words_of(const md_state_part& s) {
  const int64_t per = s.seg_bytes / width_of(s);
  return per > 0x7fffffff ? per : (double)per * s.segs * s.outer > 4e9 ? (int64_t)4e9 : per * s.segs * s.outer;
}

bool part_ok(const md_state_part& s, int64_t slots) {
  if (!s.src || !s.dst || s.seg_bytes <= 0 || s.outer <= 0 || s.segs <= 0) return false;
  const int64_t strides[6] = {s.src_slot_stride, s.dst_slot_stride, s.src_outer_stride, s.dst_outer_stride, s.src_seg_stride, s.dst_seg_stride};
  for (int64_t x : strides)
    if (x < 0) return false;
  const StridedRuns src{(uintptr_t)s.src, s.seg_bytes, {slots, s.outer, s.segs}, {s.src_slot_stride, s.src_outer_stride, s.src_seg_stride}};
  const StridedRuns dst{(uintptr_t)s.dst, s.seg_bytes, {slots, s.outer, s.segs}, {s.dst_slot_stride, s.dst_outer_stride, s.dst_seg_stride}};
  if (!runs_apart_from_each_other(dst)) return false;  // (two runs would be written to one place)
  if (s.src == s.dst) return s.src_slot_stride == s.dst_slot_stride && s.src_outer_stride == s.dst_outer_stride && s.src_seg_stride == s.dst_seg_stride;
  return !runs_meet(src, dst);
}

}  // namespace

extern "C" size_t md_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab) {
  if (batch <= 0 || beams < 2 || beams > MAXB || vocab <= 0 || vocab > MOST_VOCAB) return 0;
  return (size_t)batch * beams * pieces_of((int64_t)batch * beams, vocab) * (beams * sizeof(uint64_t) + 2 * sizeof(double));
}

extern "C" md_status md_beam_select(const md_beam_args* a, void* stream) {
  MD_CHECK_ARG(a && a->logits && a->scores && a->tokens && a->parents && a->scores_out && a->batch > 0 && a->vocab > 0 && a->vocab <= MOST_VOCAB && a->ld >= a->vocab);
  MD_CHECK_ARG(a->beams >= 2 && a->beams <= MAXB && (a->dtype == MD_DTYPE_BF16 || a->dtype == MD_DTYPE_F32) && (int64_t)a->batch * a->beams <= 65535);
  MD_CHECK_ARG(a->end_id < a->vocab && (a->end_id >= 0 || !a->ended) && ((uintptr_t)a->logits & (a->dtype == MD_DTYPE_F32 ? 3 : 1)) == 0);
  const int rows = a->batch * a->beams, pieces = (int)pieces_of(rows, a->vocab);
  if (!a->workspace || a->workspace_bytes < md_beam_workspace_bytes(a->batch, a->beams, a->vocab)) return MD_ERR_WORKSPACE;
  MD_CHECK_ARG(((uintptr_t)a->workspace & 15) == 0);
  uint64_t* best = (uint64_t*)a->workspace;
  double* sums = (double*)(best + (size_t)rows * pieces * a->beams);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(pieces, rows);
#define MD_PART(T, PER)                                                                                                                            \
  hipLaunchKernelGGL((part_kernel<T, PER>), grid, dim3(256), 0, s, (const T*)a->logits, a->ld, a->vocab, a->beams, a->suppress_id, a->scores,      \
                     a->ended, pieces, best, sums)
  const bool many = per_thread(rows, a->vocab) == MANY;
  if (a->dtype == MD_DTYPE_BF16) {
    if (many) MD_PART(bf16_t, MANY);
    else MD_PART(bf16_t, FEW);
  } else {
    if (many) MD_PART(float, MANY);
    else MD_PART(float, FEW);
  }
#undef MD_PART
  hipLaunchKernelGGL(choose_kernel, dim3(a->batch), dim3(64 * a->beams), 0, s, a->beams, pieces, a->end_id, a->scores, a->ended, a->rank_weight, best, sums,
                     a->tokens, a->parents, a->scores_out, a->ended_out);
  return md_launch_status();
}

extern "C" md_status md_state_reorder(const md_state_part* parts, int32_t n_parts, const int32_t* parents, int32_t batch, int32_t beams, void* stream) {
  MD_CHECK_ARG(parts && n_parts > 0 && parents && batch > 0 && batch <= 65535 && beams > 0 && beams <= MAXB);
  for (int i = 0; i < n_parts; ++i) MD_CHECK_ARG(part_ok(parts[i], (int64_t)batch * beams) && words_of(parts[i]) <= 0x7fffff00);
  for (int i = 0; i < n_parts; ++i)  // (one launch moves many pieces: what one writes no other reads or writes)
    for (int j = 0; j < n_parts; ++j) MD_CHECK_ARG(i == j || (parts[i].dst != parts[j].dst && parts[i].dst != parts[j].src));
  for (int done = 0; done < n_parts;) {
    Parts ps;
    ps.n = 0;
    int64_t groups = 0;
    for (; done < n_parts && ps.n < MAX_PARTS; ++done) {
      const md_state_part& s = parts[done];
      const int width = width_of(s);
      const int64_t per = s.seg_bytes / width, words = words_of(s), mine = (words + 255) / 256;
      if (groups + mine >= 1 << 24) break;  // (a launch has fewer than 2^32 threads)
      ps.p[ps.n++] = {(const char*)s.src, (char*)s.dst, s.src_slot_stride, s.dst_slot_stride, s.src_outer_stride, s.dst_outer_stride, s.src_seg_stride,
                      s.dst_seg_stride, (int32_t)per, s.segs, (int32_t)groups, width, (uint32_t)words};
      groups += mine;
    }
    const dim3 grid((unsigned)groups, batch);
    hipStream_t st = (hipStream_t)stream;
    if (beams <= 4) hipLaunchKernelGGL(reorder_kernel<4>, grid, dim3(256), 0, st, ps, parents, beams);
    else hipLaunchKernelGGL(reorder_kernel<16>, grid, dim3(256), 0, st, ps, parents, beams);
    MD_TRY(md_launch_status());
  }
  return MD_OK;
}

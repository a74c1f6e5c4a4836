// Where strided operands lie, on the host: what an entry point compares before it launches a kernel that reads one of them and writes another.
#pragma once
#include <stdint.h>

#include <algorithm>

// n[0] x n[1] x n[2] runs of `bytes` bytes, stride[i] bytes apart
struct StridedRuns {
  uintptr_t at;
  int64_t bytes, n[3], stride[3];
};

// the same runs counted so that no stride is negative
inline StridedRuns runs_upward(StridedRuns r) {
  for (int i = 0; i < 3; ++i)
    if (r.stride[i] < 0) {
      r.at += (uintptr_t)((r.n[i] - 1) * r.stride[i]);
      r.stride[i] = -r.stride[i];
    }
  return r;
}

inline bool runs_same_strides(const StridedRuns& a, const StridedRuns& b) {
  for (int i = 0; i < 3; ++i)
    if (a.n[i] > 1 && b.n[i] > 1 && a.stride[i] != b.stride[i]) return false;
  return true;
}

// Every run has bytes of its own: each stride is at least what the smaller ones span.  (Runs that interleave in another way count as if they met.)
inline bool runs_apart_from_each_other(const StridedRuns& r0) {
  const StridedRuns r = runs_upward(r0);
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int i, int j) { return r.stride[i] < r.stride[j]; });
  int64_t span = r.bytes;
  for (int i : order) {
    if (r.n[i] <= 1) continue;
    if (r.stride[i] < span) return false;
    span += (r.n[i] - 1) * r.stride[i];
  }
  return true;
}

// Whether a and b have a byte in common.  Exact where the ranges that they lie in are apart, and where they have the same strides: then the runs' distances are
// sums of d[i] * stride[i], -n_b[i] < d[i] < n_a[i], and one of them would have to lie between b.at - a.at - a.bytes and b.at - a.at + b.bytes.  Else true.
inline bool runs_meet(const StridedRuns& a0, const StridedRuns& b0) {
  const StridedRuns a = runs_upward(a0), b = runs_upward(b0);
  int64_t a_span = a.bytes, b_span = b.bytes;
  for (int i = 0; i < 3; ++i) a_span += (a.n[i] - 1) * a.stride[i], b_span += (b.n[i] - 1) * b.stride[i];
  if (a.at + (uintptr_t)a_span <= b.at || b.at + (uintptr_t)b_span <= a.at) return false;
  if (!runs_same_strides(a, b)) return true;
  struct Dim {
    int64_t stride, low, high;
  } dim[3];
  for (int i = 0; i < 3; ++i) dim[i] = {a.n[i] > 1 ? a.stride[i] : b.stride[i], 1 - b.n[i], a.n[i] - 1};
  std::sort(dim, dim + 3, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  struct Search {
    const Dim* dim;
    // a sum over dimensions k .. strictly between `above` and `below`
    bool reaches(int k, int64_t above, int64_t below) const {
      if (k == 3) return above < 0 && 0 < below;
      int64_t least = 0, most = 0;  // of the dimensions after this one
      for (int j = k + 1; j < 3; ++j) least += dim[j].low * dim[j].stride, most += dim[j].high * dim[j].stride;
      const Dim& d = dim[k];
      if (d.stride == 0 || (d.low == 0 && d.high == 0)) return reaches(k + 1, above, below);
      // d * stride + most > above and d * stride + least < below, a step more on either side for the division's rounding
      const int64_t from = std::max(d.low, (above - most) / d.stride - 1), to = std::min(d.high, (below - least) / d.stride + 1);
      if (to - from > 16) return true;  // (strides that do not nest: not worth telling)
      for (int64_t i = from; i <= to; ++i)
        if (reaches(k + 1, above - i * d.stride, below - i * d.stride)) return true;
      return false;
    }
  };
  const int64_t apart = (int64_t)(b.at - a.at);
  return Search{dim}.reaches(0, apart - a.bytes, apart + b.bytes);
}

// Whether tensors of rows share memory: the checks of entries that write some of
// their tensors, without HIP, so that a host program can run them too.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace frisk {

// Sizes n and strides of three dims around rows of one length (elements).
struct Rows {
  const void* p;
  int64_t n[3], s[3];
};

typedef __int128 Wide;  // a size of 2^31 times a stride of 2^40

// Whether the ranges of two tensors, from the first row's start to the last
// one's end (row bytes, element bytes), share memory.
inline bool spans_share(const Rows& a, int64_t row_a, int es_a, const Rows& b, int64_t row_b, int es_b) {
  Wide ea = row_a, eb = row_b;
  for (int i = 0; i < 3; ++i) {
    ea += (Wide)(a.n[i] - 1) * a.s[i] * es_a;
    eb += (Wide)(b.n[i] - 1) * b.s[i] * es_b;
  }
  const Wide pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
  return pa < pb + eb && pb < pa + ea;
}

// Whether rows of one tensor may share memory: they do not if each stride
// holds all that the smaller ones reach (any permuted or sliced tensor).
inline bool rows_overlap(const int64_t (&n)[3], const int64_t (&s)[3], int64_t row) {
  int d[3] = {0, 1, 2};
  std::sort(d, d + 3, [&](int i, int j) { return s[i] < s[j]; });
  Wide below = row;
  for (const int i : d) {
    if (n[i] == 1) continue;
    if (s[i] < below) return true;
    below += (Wide)(n[i] - 1) * s[i];
  }
  return false;
}

// Whether i * strides of a and j * strides of b, `gap` apart, meet within a
// row: the dims d[0 .. k) by falling stride, equal in both.
inline bool rows_meet(int64_t gap, const Rows& a, const Rows& b, const int* d, int k, int64_t row) {
  if (k == 0) return gap < row && gap > -row;
  const int64_t s = a.s[*d];
  const int64_t q = gap >= 0 ? gap / s : -((-gap + s - 1) / s);
  for (const int64_t i : {q, q + 1})  // index in a less index in b
    if (i < a.n[*d] && -i < b.n[*d] && rows_meet(gap - i * s, a, b, d + 1, k - 1, row)) return true;
  return false;
}

// Whether the rows of two tensors may share memory.  Exact for equal strides
// each at least the extent of the dims below it (heads of one buffer); other
// tensors must not reach into each other's range.  A dim of one row, or of one
// row repeated (stride 0), has the other tensor's stride.
inline bool rows_share(Rows a, Rows b, int64_t row, int es) {
  for (int i = 0; i < 3; ++i) {
    if (a.s[i] == 0) a.n[i] = 1;
    if (b.s[i] == 0) b.n[i] = 1;
    if (a.n[i] == 1) a.s[i] = b.s[i];
    else if (b.n[i] == 1) b.s[i] = a.s[i];
  }
  if (!spans_share(a, row * es, es, b, row * es, es)) return false;
  const int64_t bytes = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p);
  int d[3], k = 0;
  for (int i = 0; i < 3; ++i) {
    if (a.n[i] == 1 && b.n[i] == 1) continue;
    if (a.s[i] != b.s[i]) return true;
    d[k++] = i;
  }
  std::sort(d, d + k, [&](int i, int j) { return a.s[i] > a.s[j]; });
  Wide below = row;
  for (int i = k - 1; i >= 0; --i) {
    if (a.s[d[i]] < below) return true;
    below += (Wide)(std::max(a.n[d[i]], b.n[d[i]]) - 1) * a.s[d[i]];
  }
  if (bytes % es) return true;
  return rows_meet(bytes / es, a, b, d, k, row);
}

}  // namespace frisk

// row_sets.hpp -- where strided rows lie and whether they share memory (host;
// tests/cpp/row_sets.cpp compares it with the bytes themselves).
//
// A set of rows is n[0] x n[1] x ... rows of `row` bytes at byte strides nb[0], nb[1],
// ...; dimension 0 is the heads.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace aq {

// The bytes from a set's first to its last.
struct Span {
  uintptr_t lo, hi;
};

inline Span span_of(const void *p, size_t row, const int *n, const size_t *nb, int dims) {
  uintptr_t hi = reinterpret_cast<uintptr_t>(p) + row;
  for (int i = 0; i < dims; ++i) hi += (size_t)(n[i] - 1) * nb[i];
  return {reinterpret_cast<uintptr_t>(p), hi};
}

// Whether a set's rows are shown to share no byte: each stride steps over all that
// the smaller ones span.
inline bool rows_apart(size_t row, const int *n, const size_t *nb, int dims) {
  size_t extent = row;
  bool used[3] = {};
  for (int k = 0; k < dims; ++k) {
    int at = -1;
    for (int i = 0; i < dims; ++i)
      if (!used[i] && (at < 0 || nb[i] < nb[at] || (nb[i] == nb[at] && n[i] < n[at]))) at = i;
    used[at] = true;
    if (n[at] > 1) {
      if (nb[at] < extent) return false;
      extent += (size_t)(n[at] - 1) * nb[at];
    }
  }
  return true;
}

// Whether a row of the one set and a row of the other share a byte, of sets whose dimensions
// have the same strides, largest first: a pair of rows lies `gap` + the sum of d[i] * nb[i]
// apart, where d[i] runs from -back[i] to ahead[i].  What the smaller dimensions reach leaves few
// d[i] to try where each stride steps over them; where it does not, the sets count as sharing.
inline bool rows_meet(int64_t gap, int64_t row, const int64_t *nb, const int64_t *back,
                      const int64_t *ahead, int dims) {
  if (dims == 0) return gap < row && -gap < row;
  int64_t below = 0, above = 0;  // reach of the dimensions behind this one
  for (int i = 1; i < dims; ++i) {
    below += back[i] * nb[i];
    above += ahead[i] * nb[i];
  }
  if (nb[0] == 0) return rows_meet(gap, row, nb + 1, back + 1, ahead + 1, dims - 1);
  // gap + d nb in (-row - above, row + below)
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  int64_t first = floor_div(-row - above - gap, nb[0]) + 1;
  int64_t last = floor_div(row + below - gap - 1, nb[0]);
  if (first < -back[0]) first = -back[0];
  if (last > ahead[0]) last = ahead[0];
  if (last - first > 3) return true;
  for (int64_t d = first; d <= last; ++d)
    if (rows_meet(gap + d * nb[0], row, nb + 1, back + 1, ahead + 1, dims - 1)) return true;
  return false;
}

// Whether two sets are shown to share no byte: their spans are apart, or they have the same
// strides (parts of one tensor) and no two rows meet.  A dimension of one index in one of the
// sets takes the other's stride.
inline bool sets_apart(const void *a, size_t row, const int *na, const size_t *nba, const void *b,
                       const int *nb_, const size_t *nbb, int dims) {
  const Span x = span_of(a, row, na, nba, dims), y = span_of(b, row, nb_, nbb, dims);
  if (x.hi <= y.lo || y.hi <= x.lo) return true;
  int64_t nb[3], back[3], ahead[3];  // by stride, largest first
  int used = 0;
  for (int i = 0; i < dims; ++i) {
    if (na[i] == 1 && nb_[i] == 1) continue;
    if (na[i] > 1 && nb_[i] > 1 && nba[i] != nbb[i]) return false;
    const int64_t stride = (int64_t)(na[i] > 1 ? nba[i] : nbb[i]);
    int at = used++;
    for (; at > 0 && nb[at - 1] < stride; --at) {
      nb[at] = nb[at - 1];
      back[at] = back[at - 1];
      ahead[at] = ahead[at - 1];
    }
    nb[at] = stride;
    back[at] = na[i] - 1;  // of the first set's index, the second's goes ahead
    ahead[at] = nb_[i] - 1;
  }
  const int64_t gap = y.lo >= x.lo ? (int64_t)(y.lo - x.lo) : -(int64_t)(x.lo - y.lo);
  return !rows_meet(gap, (int64_t)row, nb, back, ahead, used);
}

}  // namespace aq

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

// Whether two sets are shown to share no byte: their spans are apart, or they lie side
// by side in rows of the same strides (columns of one tensor).
inline bool sets_apart(const void *a, size_t row, const int *na, const size_t *nba, const void *b,
                const int *nb_, const size_t *nbb, int dims) {
  const Span x = span_of(a, row, na, nba, dims), y = span_of(b, row, nb_, nbb, dims);
  if (x.hi <= y.lo || y.hi <= x.lo) return true;
  // heads are dimension 0; the outer strides must agree and hold both columns
  size_t pitch = 0;
  for (int i = 1; i < dims; ++i) {
    if (na[i] == 1 && nb_[i] == 1) continue;
    if (nba[i] != nbb[i] || na[i] != nb_[i]) return false;
    if (pitch == 0 || nba[i] < pitch) pitch = nba[i];
  }
  if (pitch == 0) return false;
  for (int i = 1; i < dims; ++i)
    if ((na[i] > 1 || nb_[i] > 1) && nba[i] % pitch) return false;
  const size_t wa = (size_t)(na[0] - 1) * nba[0] + row, wb = (size_t)(nb_[0] - 1) * nbb[0] + row;
  const size_t gap = x.lo <= y.lo ? y.lo - x.lo : x.lo - y.lo;
  const size_t off = gap % pitch;  // of the later set's columns behind the earlier's
  const size_t first = x.lo <= y.lo ? wa : wb, second = x.lo <= y.lo ? wb : wa;
  return off >= first && off + second <= pitch;
}

}  // namespace aq
